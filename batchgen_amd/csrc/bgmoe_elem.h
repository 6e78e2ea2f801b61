// Rows of bf16, fp16 or fp32 elements for the kernels that take all three: eight elements at a time, at any address
// that is a multiple of the element's size.
#pragma once
#include "bgmoe_common.h"

struct Bf16 { static constexpr int kBytes = 2; typedef uint16_t raw; };
struct Fp16 { static constexpr int kBytes = 2; typedef uint16_t raw; };
struct Fp32 { static constexpr int kBytes = 4; typedef uint32_t raw; };

// 16-byte accesses at any byte address: the hardware takes them on global memory, the type tells the compiler so (an
// aligned address gets the same instruction, so there is no second path for rows of odd width)
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
__device__ __forceinline__ u32x4 load16(const void* p) { return *reinterpret_cast<const u32x4_any*>(p); }
__device__ __forceinline__ void store16(void* p, u32x4 v) { *reinterpret_cast<u32x4_any*>(p) = v; }
// NT: past the last-level cache (256 MB), for data that does not fit there and is touched once
template <bool NT>
__device__ __forceinline__ u32x4 load16_as(const void* p) {
  if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p));
  else return load16(p);
}
template <bool NT>
__device__ __forceinline__ void store16_as(void* p, u32x4 v) {
  if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any*>(p));
  else store16(p, v);
}

template <typename T> constexpr int kPer16 = 16 / T::kBytes;      // elements in 16 bytes

template <typename T>
__device__ __forceinline__ void unpack16(u32x4 r, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (__is_same(T, Fp32)) {
      v[i] = __uint_as_float(r[i]);
    } else if constexpr (__is_same(T, Bf16)) {
      v[2 * i] = __uint_as_float(r[i] << 16);
      v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
    } else {
      v[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(r[i] & 0xffffu));
      v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(r[i] >> 16));
    }
  }
}
// one rounding to the element type, to nearest even
template <typename T>
__device__ __forceinline__ u32x4 pack16(const float* v) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (__is_same(T, Fp32))
      r[i] = __float_as_uint(v[i]);
    else if constexpr (__is_same(T, Bf16))
      r[i] = pack2_bf16(v[2 * i], v[2 * i + 1]);
    else
      r[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i]) |
             ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i + 1]) << 16);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ float load_one(const void* p) {
  if constexpr (__is_same(T, Fp32)) return *reinterpret_cast<const float*>(p);
  else if constexpr (__is_same(T, Bf16)) return bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(p));
  else return (float)*reinterpret_cast<const _Float16*>(p);
}
template <typename T>
__device__ __forceinline__ void store_one(void* p, float v) {
  if constexpr (__is_same(T, Fp32)) *reinterpret_cast<float*>(p) = v;
  else if constexpr (__is_same(T, Bf16)) *reinterpret_cast<uint16_t*>(p) = (uint16_t)f32_to_bf16_bits(v);
  else *reinterpret_cast<_Float16*>(p) = (_Float16)v;
}
// v as a reader of the stored element sees it
template <typename T>
__device__ __forceinline__ float round_to(float v) {
  if constexpr (__is_same(T, Fp32)) return v;
  else if constexpr (__is_same(T, Bf16)) return bf16_round_f32(v);
  else return (float)(_Float16)v;
}

// eight elements of a row, `left` of them inside it; the others are 0
template <typename T>
__device__ __forceinline__ void load8(const void* row, int64_t c, int left, float (&v)[8]) {
  const uint8_t* p = reinterpret_cast<const uint8_t*>(row) + c * T::kBytes;
  if (left >= 8) {
    unpack16<T>(load16(p), v);
    if constexpr (T::kBytes == 4) unpack16<T>(load16(p + 16), v + 4);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? load_one<T>(p + i * T::kBytes) : 0.0f;
  }
}
// the same, still packed: half the registers for the two-byte types
template <typename T> struct Packed8 { u32x4 v[T::kBytes / 2]; };
template <typename T, bool NT = false>
__device__ __forceinline__ Packed8<T> load8_packed(const void* row, int64_t c, int left) {
  const uint8_t* p = reinterpret_cast<const uint8_t*>(row) + c * T::kBytes;
  Packed8<T> r;
  if (left >= 8) {
    r.v[0] = load16_as<NT>(p);
    if constexpr (T::kBytes == 4) r.v[1] = load16_as<NT>(p + 16);
  } else {
    typename T::raw e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = i < left ? reinterpret_cast<const typename T::raw*>(p)[i] : (typename T::raw)0;
    __builtin_memcpy(&r, e, sizeof(r));
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void unpack8(const Packed8<T>& r, float (&v)[8]) {
  unpack16<T>(r.v[0], v);
  if constexpr (T::kBytes == 4) unpack16<T>(r.v[1], v + 4);
}
template <typename T, bool NT = false>
__device__ __forceinline__ void store8(void* row, int64_t c, int left, const float (&v)[8]) {
  uint8_t* p = reinterpret_cast<uint8_t*>(row) + c * T::kBytes;
  if (left >= 8) {
    store16_as<NT>(p, pack16<T>(v));
    if constexpr (T::kBytes == 4) store16_as<NT>(p + 16, pack16<T>(v + 4));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) store_one<T>(p + i * T::kBytes, v[i]);
  }
}

// ---- one int8 scale per row: scale = max(amax, 1e-30) / 127, q = rint(v / scale), both IEEE fp32 ----------------------
__device__ __forceinline__ float int8_scale(float amax) { return fmaxf(amax, 1e-30f) / 127.0f; }
// Eight values of a row whose scale is `scale`.  While the scale is in (1e-30, 1e30) the quotient comes from one
// reciprocal and a correction step (div_by_scale: the IEEE quotient at a third of its instructions); |v| <= 127 scale, so
// nothing has to be clamped.  Else (rows of tiny or huge values, non-finite rows) by the division, NaN becoming 0.
__device__ __forceinline__ void int8_store8(int8_t* p, int left, const float (&v)[8], float scale) {
  typedef unsigned int u32x2 __attribute__((ext_vector_type(2), aligned(1)));
  int q[8];
  if (scale_div_ok(scale)) {
    const float r = 1.0f / scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = (int)rintf(div_by_scale(v[i], scale, r));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = rintf(v[i] / scale);
      q[i] = f == f ? (int)fminf(fmaxf(f, -127.0f), 127.0f) : 0;
    }
  }
  if (left >= 8) {
    u32x2 o;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      o[j] = ((uint32_t)q[4 * j] & 0xffu) | (((uint32_t)q[4 * j + 1] & 0xffu) << 8) | (((uint32_t)q[4 * j + 2] & 0xffu) << 16) |
             ((uint32_t)q[4 * j + 3] << 24);
    *reinterpret_cast<u32x2*>(p) = o;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = (int8_t)q[i];
  }
}

// ---- launches of more blocks than one grid dimension holds (2^32 threads): a second dimension of whole slices ---------
inline dim3 bgmoe_grid(int64_t blocks) {
  const int64_t slice = 1 << 20;
  return blocks <= slice ? dim3((unsigned)blocks) : dim3((unsigned)slice, (unsigned)((blocks + slice - 1) / slice));
}
constexpr int64_t kBgmoeMaxBlocks = (int64_t)65535 << 20;
__device__ __forceinline__ int64_t linear_block() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

#define BGMOE_BY_TYPE(dtype, call)                           \
  do {                                                       \
    if ((dtype) == BGMOE_DT_BF16) return call(Bf16);         \
    if ((dtype) == BGMOE_DT_FP16) return call(Fp16);         \
    return call(Fp32);                                       \
  } while (0)
