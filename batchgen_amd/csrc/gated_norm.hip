// The seam between two blocks in one pass for gfx950: RMSNorm behind a block, its gate and residual scale, the residual
// sum, RMSNorm in front of the next block, optionally with that row's int8 form; and the gradient of all of it.
//
//   p = b * i1 * w1,   i1 = 1 / sqrt(mean(b^2) + eps)          (no w1: p = b)
//   y = r + s * g * p                                          (g: 1, per channel, per token or per element)
//   n = y * i2 * w2,   i2 = 1 / sqrt(mean(y^2) + eps)
//
// Gradient, with t = dn * w2, yh = y * i2, c = s * g * w1, bh = b * i1 (row means over h):
//   Dy = dy + i2 * (t - yh * mean(t * yh))                     = d residual
//   db = i1 * (c * Dy - bh * mean(c * Dy * bh))
//   dw2 = sum_rows dn * yh,  dw1 = sum_rows s * g * Dy * bh,  dg = s * p * Dy (summed over what g is shared by)
// The second mean contains the first one, but linearly:
//   sum(c Dy bh) = sum(c bh (dy + i2 t)) - i2 * mean(t yh) * sum(c bh yh)
// so one exchange of three sums per row serves both norms.
//
// Both passes are bound by HBM: a row is held in registers between its sums and its outputs, eight elements per thread
// and vector, and every operand is read once.  The gradient recomputes y in fp32 from block and residual (the same
// bytes as reading the stored y, without its rounding).  The sums over rows (w1, w2, a channel gate) are accumulated
// in LDS (rows wider than 8192: in registers) by blocks that walk many rows, written as one fp32 plane per block and
// added in block order by a second launch: the same bits every time, no atomics.
#include "bgmoe_elem.h"

namespace {

constexpr int kMaxH = 16384;
constexpr int kAccBytes = 3 * 8 * 4;          // LDS accumulators of a thread of the gradient pass

struct NormArgs {
  const void *block, *residual, *post, *gate, *pre;
  int gate_mode, param_fp32;           // bits 0 / 1 / 2: post / gate / pre are fp32
  float scale, eps;
  int64_t rows;
  int h;
  void *y, *normed;
  int8_t* q;
  float *q_scale, *inv_post, *inv_pre;
  // gradient
  const float *i_post, *i_pre;
  const void *dy, *dn;
  void *d_block, *d_residual, *d_gate;
  float* planes;                       // [blocks][kinds][h]
  int want_post, want_pre, want_gate;  // which planes (gate: channel form)
};

// eight values of a parameter vector that is of the rows' type or fp32
template <typename T>
__device__ __forceinline__ void load_param8(const void* p, bool fp32, int64_t c, int left, float (&v)[8]) {
  if (fp32) load8<Fp32>(p, c, left, v);
  else load8<T>(p, c, left, v);
}
template <typename T>
__device__ __forceinline__ float load_param1(const void* p, bool fp32, int64_t i) {
  return fp32 ? reinterpret_cast<const float*>(p)[i] : load_one<T>(reinterpret_cast<const uint8_t*>(p) + i * T::kBytes);
}
// s * g of eight columns
template <typename T>
__device__ __forceinline__ void load_gate8(const NormArgs& a, int64_t row, int c, int left, float token, float (&v)[8]) {
  if (a.gate_mode == BGMOE_GATE_CHANNEL || a.gate_mode == BGMOE_GATE_FULL) {
    load_param8<T>(a.gate, (a.param_fp32 & 2) != 0, a.gate_mode == BGMOE_GATE_FULL ? row * a.h + c : c, left, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= a.scale;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = token * a.scale;
  }
}

// N sums over the block; every thread gets them.  `slot` alternates between calls so that one barrier per call is
// enough (the buffer of the previous call may still be read).
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float (*buf)[16][N]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v[i] = v[i] + __shfl_xor(v[i], off, BGMOE_WAVE);
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  if (waves == 1) return;
  if (lane_id() == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) (*buf)[wave][i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float s = 0.0f;
    for (int w = 0; w < waves; ++w) s += (*buf)[w][i];
    v[i] = s;
  }
}
__device__ __forceinline__ float block_max(float v, float* buf) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, BGMOE_WAVE));
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  if (waves == 1) return v;
  if (lane_id() == 0) buf[wave] = v;
  __syncthreads();
  v = buf[0];
  for (int w = 1; w < waves; ++w) v = fmaxf(v, buf[w]);
  return v;
}
// 1 / sqrt(mean + eps), the square root and the quotient rounded to nearest
__device__ __forceinline__ float inv_rms(float sum, int h, float eps) { return 1.0f / sqrtf(sum / (float)h + eps); }

// One block per row, V vectors of eight elements per thread.
template <typename T, int V, bool NT>
__global__ __launch_bounds__(1024) void gated_norm_kernel(NormArgs a) {
  __shared__ float s_sum[2][16][1];
  __shared__ float s_max[16];
  const int64_t row = linear_block();
  if (row >= a.rows) return;
  const int64_t base = row * a.h;
  const int step = blockDim.x * 8;
  float b[V][8], y[V][8];
  const float token = a.gate_mode == BGMOE_GATE_TOKEN ? load_param1<T>(a.gate, (a.param_fp32 & 2) != 0, row) : 1.0f;
#pragma unroll
  for (int u = 0; u < V; ++u) {
    const int c = threadIdx.x * 8 + u * step, left = a.h - c;
    unpack8<T>(load8_packed<T, NT>(a.block, base + c, left), b[u]);
    unpack8<T>(load8_packed<T, NT>(a.residual, base + c, left), y[u]);
  }
  if (a.post) {
    float sum[1] = {0.0f};
#pragma unroll
    for (int u = 0; u < V; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[0] = __builtin_fmaf(b[u][i], b[u][i], sum[0]);
    block_sum<1>(sum, &s_sum[0]);
    const float i1 = inv_rms(sum[0], a.h, a.eps);
    if (a.inv_post && threadIdx.x == 0) a.inv_post[row] = i1;
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int c = threadIdx.x * 8 + u * step, left = a.h - c;
      float w[8];
      load_param8<T>(a.post, (a.param_fp32 & 1) != 0, c, left, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) b[u][i] = b[u][i] * i1 * w[i];
    }
  }
  float sum[1] = {0.0f};
#pragma unroll
  for (int u = 0; u < V; ++u) {
    const int c = threadIdx.x * 8 + u * step, left = a.h - c;
    float g[8];
    load_gate8<T>(a, row, c, left, token, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[u][i] = __builtin_fmaf(g[i], b[u][i], y[u][i]);
    store8<T, NT>(a.y, base + c, left, y[u]);
    if (left < 8)                                        // what lies past the row does not count
#pragma unroll
      for (int i = 0; i < 8; ++i) y[u][i] = i < left ? y[u][i] : 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[0] = __builtin_fmaf(y[u][i], y[u][i], sum[0]);
  }
  if (!a.pre) return;
  block_sum<1>(sum, &s_sum[1]);
  const float i2 = inv_rms(sum[0], a.h, a.eps);
  if (a.inv_pre && threadIdx.x == 0) a.inv_pre[row] = i2;
  float amax = 0.0f, bad = 0.0f;
#pragma unroll
  for (int u = 0; u < V; ++u) {
    const int c = threadIdx.x * 8 + u * step, left = a.h - c;
    float w[8];
    load_param8<T>(a.pre, (a.param_fp32 & 4) != 0, c, left, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[u][i] = y[u][i] * i2 * w[i];
    if (a.normed) store8<T, NT>(a.normed, base + c, left, y[u]);
    if (a.q) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[u][i] = i < left ? round_to<T>(y[u][i]) : 0.0f;   // the cast sees what a reader of `normed` sees
        amax = fmaxf(amax, fabsf(y[u][i]));
        if (y[u][i] != y[u][i]) bad = 1.0f;                // fmaxf drops a NaN
      }
    }
  }
  if (!a.q) return;
  amax = block_max(bad != 0.0f ? __builtin_huge_valf() : amax, s_max);
  const float sc = int8_scale(amax);
  if (threadIdx.x == 0) a.q_scale[row] = sc;
#pragma unroll
  for (int u = 0; u < V; ++u) {
    const int c = threadIdx.x * 8 + u * step, left = a.h - c;
    int8_store8(a.q + base + c, left, y[u], sc);
  }
}

// Rows are walked by gridDim.x blocks; the next row's operands are requested, still packed, before this row's exchange of
// sums, so that a CU always has a row (57 KB at h = 7168) on its way while its VALU (about 40 operations per element)
// works on another.  What the blocks sum over their rows lives in LDS, eight floats per thread and kind (in registers it
// takes the place of that next row, or of a second block per CU).  Order of the planes: post, pre, gate.
// The two-byte types spill four of the 128 registers that a block of 1024 threads leaves (20 bytes of scratch per lane).
// ACC_LDS = false (rows wider than LDS holds, h > 8192): accumulators in registers, which do not fit: 350 to 390 bytes of
// scratch per lane are written and read for every row and bound that form.  4096 x 16384 bf16 667 us (1.2 TB/s), fp32 761
// (2.1), where 4096 x 8192 takes 103 us (3.9 TB/s) and 201 (4.0).
template <typename T, int V, bool ACC_LDS, bool NT>
__global__ __launch_bounds__(1024) void gated_norm_backward_kernel(NormArgs a) {
  extern __shared__ __align__(16) float s_acc[];         // [kind][thread * 8 + i]
  __shared__ float s_sum[2][16][3];
  const int step = blockDim.x * 8;
  const float inv_h = 1.0f / (float)a.h;
  float racc[ACC_LDS ? 1 : 3][V][8];
  auto add = [&](int kind, int u, const float (&v)[8]) {
    if constexpr (ACC_LDS) {
      float4* p = reinterpret_cast<float4*>(s_acc + kind * step + threadIdx.x * 8);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float4 o = p[q];
        o.x += v[4 * q]; o.y += v[4 * q + 1]; o.z += v[4 * q + 2]; o.w += v[4 * q + 3];
        p[q] = o;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) racc[kind][u][i] += v[i];
    }
  };
#pragma unroll
  for (int kind = 0; kind < 3; ++kind) {
    if constexpr (ACC_LDS) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s_acc[kind * step + threadIdx.x * 8 + i] = 0.0f;
    } else {
#pragma unroll
      for (int u = 0; u < V; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) racc[kind][u][i] = 0.0f;
    }
  }
  const bool norm = a.pre != nullptr && a.dn != nullptr;
  struct Row { Packed8<T> b[V], r[V], dy[V], dn[V]; };
  auto request = [&](int64_t row) {
    Row o;
    const int64_t base = row * a.h;
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int c = threadIdx.x * 8 + u * step, left = a.h - c;
      o.b[u] = load8_packed<T, NT>(a.block, base + c, left);
      o.r[u] = load8_packed<T, NT>(a.residual, base + c, left);
      o.dy[u] = a.dy ? load8_packed<T, NT>(a.dy, base + c, left) : Packed8<T>{};
      o.dn[u] = norm ? load8_packed<T, NT>(a.dn, base + c, left) : Packed8<T>{};
    }
    return o;
  };
  constexpr bool kAhead = ACC_LDS && T::kBytes == 2;     // (fp32 rows have twice the bytes in flight without it)
  Row next;
  if (kAhead) next = request(blockIdx.x);
  int slot = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, slot ^= 1) {
    const int64_t base = row * a.h;
    if (!kAhead) next = request(row);
    const float token = a.gate_mode == BGMOE_GATE_TOKEN ? load_param1<T>(a.gate, (a.param_fp32 & 2) != 0, row) : 1.0f;
    const float i1 = a.post ? a.i_post[row] : 1.0f;
    const float i2 = norm ? a.i_pre[row] : 0.0f;         // without a gradient through that norm y plays no part
    // bh: b * i1;  w1 (1 without a norm behind the block);  yh: y * i2;  e: dy + i2 * t;  sg: s g without a token's gate
    float bh[V][8], yh[V][8], e[V][8], sg[V][8], w1[V][8];
    float sum[3] = {0.0f, 0.0f, 0.0f};                   // t yh, c' bh e, c' bh yh  (c' without the token's gate)
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int c = threadIdx.x * 8 + u * step, left = a.h - c;
      float dn[8], w2[8], dw2[8];
      load_gate8<T>(a, row, c, left, 1.0f, sg[u]);
      if (a.post) load_param8<T>(a.post, (a.param_fp32 & 1) != 0, c, left, w1[u]);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) w1[u][i] = 1.0f;
      if (norm) load_param8<T>(a.pre, (a.param_fp32 & 4) != 0, c, left, w2);
      unpack8<T>(next.b[u], bh[u]);
      unpack8<T>(next.r[u], yh[u]);
      unpack8<T>(next.dy[u], e[u]);
      unpack8<T>(next.dn[u], dn);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        bh[u][i] *= i1;
        const float cb = sg[u][i] * (w1[u][i] * bh[u][i]);
        if (norm) {                                        // (past the row's end every operand is 0, and so is yh)
          yh[u][i] = __builtin_fmaf(token, cb, yh[u][i]) * i2;
          const float t = dn[i] * w2[i];
          sum[0] = __builtin_fmaf(t, yh[u][i], sum[0]);
          e[u][i] = __builtin_fmaf(i2, t, e[u][i]);
          dw2[i] = dn[i] * yh[u][i];
          sum[2] = __builtin_fmaf(cb, yh[u][i], sum[2]);
        }
        sum[1] = __builtin_fmaf(cb, e[u][i], sum[1]);
      }
      if (norm && a.want_pre) add(1, u, dw2);
    }
    if (kAhead && row + gridDim.x < a.rows) next = request(row + gridDim.x);
    block_sum<3>(sum, &s_sum[slot]);
    const float m = i2 * (sum[0] * inv_h);               // i2 * mean(t yh)
    const float cdb = sum[1] - m * sum[2];               // sum(c' Dy bh)
    const float mb = token * cdb * inv_h;
    if (a.gate_mode == BGMOE_GATE_TOKEN && a.d_gate && threadIdx.x == 0) {
      if (a.param_fp32 & 2) reinterpret_cast<float*>(a.d_gate)[row] = cdb;
      else store_one<T>(reinterpret_cast<uint8_t*>(a.d_gate) + row * T::kBytes, cdb);
    }
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int c = threadIdx.x * 8 + u * step, left = a.h - c;
      float db[8], dw1[8], gd[8];
      if (a.gate_mode == BGMOE_GATE_TOKEN)
#pragma unroll
        for (int i = 0; i < 8; ++i) sg[u][i] *= token;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (norm) e[u][i] = __builtin_fmaf(-m, yh[u][i], e[u][i]);   // Dy
        const float dp = sg[u][i] * e[u][i];
        dw1[i] = dp * bh[u][i];
        gd[i] = a.scale * e[u][i] * (bh[u][i] * w1[u][i]);
        db[i] = a.post ? i1 * __builtin_fmaf(-mb, bh[u][i], dp * w1[u][i]) : dp;
      }
      if (a.d_block) store8<T, NT>(a.d_block, base + c, left, db);
      if (a.d_residual) store8<T, NT>(a.d_residual, base + c, left, e[u]);
      if (a.gate_mode == BGMOE_GATE_FULL && a.d_gate) {
        if (a.param_fp32 & 2) store8<Fp32>(a.d_gate, base + c, left, gd);
        else store8<T>(a.d_gate, base + c, left, gd);
      }
      if (a.want_post) add(0, u, dw1);
      if (a.want_gate) add(2, u, gd);
    }
  }
  float* plane = a.planes + (int64_t)blockIdx.x * (a.want_post + a.want_pre + a.want_gate) * a.h;
  int64_t o = 0;
#pragma unroll
  for (int kind = 0; kind < 3; ++kind) {
    if (!(kind == 0 ? a.want_post : kind == 1 ? a.want_pre : a.want_gate)) continue;
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int c = threadIdx.x * 8 + u * step, left = a.h - c;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = ACC_LDS ? s_acc[kind * step + threadIdx.x * 8 + i] : racc[ACC_LDS ? 0 : kind][u][i];
      store8<Fp32>(plane, o + c, left, v);
    }
    o += a.h;
  }
}

struct SumArgs {
  const float* planes;
  int blocks, kinds, h;
  void* out[3];
  int fp32[3];
};
// 64 columns per block: 16 waves add every 16th plane each, then their sums are added in wave order
template <typename T>
__global__ __launch_bounds__(1024) void plane_sum_kernel(SumArgs a) {
  __shared__ float s_part[16][64];
  const int wave = threadIdx.x >> 6, lane = lane_id();
  const int64_t col = (int64_t)blockIdx.x * 64 + lane, cols = (int64_t)a.kinds * a.h;
  float s = 0.0f;
  if (col < cols)
#pragma unroll 8
    for (int b = wave; b < a.blocks; b += 16) s += a.planes[(int64_t)b * cols + col];
  s_part[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || col >= cols) return;
  s = 0.0f;
#pragma unroll
  for (int w = 0; w < 16; ++w) s += s_part[w][lane];
  const int kind = (int)(col / a.h);
  const int64_t c = col - (int64_t)kind * a.h;
  if (a.fp32[kind]) reinterpret_cast<float*>(a.out[kind])[c] = s;
  else store_one<T>(reinterpret_cast<uint8_t*>(a.out[kind]) + c * T::kBytes, s);
}

// Threads for rows of h elements in `vecs` vectors of eight.
int threads_for(int h, int vecs) { return ((h + 8 * vecs - 1) / (8 * vecs) + BGMOE_WAVE - 1) / BGMOE_WAVE * BGMOE_WAVE; }
// Forward: two vectors per thread from 1024 rows on (half the waves per row: more rows at work; with the int8 form
// 16384 x 7168 269 us against 340 through the cache, 4096 x 7168 45 against 54 us without it), one below (a shorter chain per row: 16 x
// 7168 5.4 against 5.9 us, 333 x 1001 5.4 against 6.9).
int forward_vecs(int64_t rows, int h) { return h > 8192 || rows >= 1024 ? 2 : 1; }
int backward_vecs(int h) { return h > 8192 ? 2 : 1; }
// Blocks of the gradient pass: what is resident at 128 registers per thread (1024 threads per CU), at most one per row.
// Fewer blocks would write fewer planes, but a row takes a block about 2.2 us: 1024 x 7168 35 us with 256 blocks, 82
// with 64; 4096 x 2048 56 us with 256.  16384 x 7168 bf16: 337 us, 4.2 TB/s.
int64_t backward_blocks(int64_t rows, int h) {
  const int64_t blocks = 256 * (1024 / threads_for(h, backward_vecs(h)));
  return rows < blocks ? rows : blocks;
}

// Whether a pass over `operands` row matrices moves more than the last-level cache holds, which it then bypasses: forward
// of 16384 x 7168 bf16 230 -> 168 us (5.6 TB/s), with the int8 form 269 -> 203; gradient of 16384 x
// 2048 116 -> 96 us.  4096 x 7168, which fits, 45.2 us through it and 47.5 past it.
template <typename T>
bool past_cache(const NormArgs& a, int operands) { return a.rows * a.h * T::kBytes * operands > (256LL << 20); }

template <typename T>
int run_forward(const NormArgs& a, hipStream_t st) {
  const int vecs = forward_vecs(a.rows, a.h), threads = threads_for(a.h, vecs);
  BgmoeProf prof(BGMOE_K_GATED_NORM, st);
  if (vecs == 1) hipLaunchKernelGGL((gated_norm_kernel<T, 1, false>), bgmoe_grid(a.rows), dim3(threads), 0, st, a);
  else if (!past_cache<T>(a, 4)) hipLaunchKernelGGL((gated_norm_kernel<T, 2, false>), bgmoe_grid(a.rows), dim3(threads), 0, st, a);
  else hipLaunchKernelGGL((gated_norm_kernel<T, 2, true>), bgmoe_grid(a.rows), dim3(threads), 0, st, a);
  return bgmoe_check_launch("gated_residual_norm");
}
// the dynamic-LDS opt-in (more than 64 KB), once per device
int ensure_init() {
  static bool done[64] = {};
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) {
    bgmoe_set_error("gated_residual_norm_backward: no current HIP device (or device index >= 64)");
    return BGMOE_ERR_HIP;
  }
  if (done[dev]) return BGMOE_OK;
  const void* fns[6] = {
      (const void*)gated_norm_backward_kernel<Bf16, 1, true, false>, (const void*)gated_norm_backward_kernel<Bf16, 1, true, true>,
      (const void*)gated_norm_backward_kernel<Fp16, 1, true, false>, (const void*)gated_norm_backward_kernel<Fp16, 1, true, true>,
      (const void*)gated_norm_backward_kernel<Fp32, 1, true, false>, (const void*)gated_norm_backward_kernel<Fp32, 1, true, true>};
  for (const void* f : fns) {
    const hipError_t err = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, 1024 * kAccBytes);
    if (err != hipSuccess) {
      bgmoe_set_error("gated_residual_norm_backward: hipFuncSetAttribute(dynamic LDS) failed: %s", hipGetErrorString(err));
      return BGMOE_ERR_HIP;
    }
  }
  done[dev] = true;
  return BGMOE_OK;
}
template <typename T>
int run_backward(const NormArgs& a, const SumArgs& s, hipStream_t st) {
  const int rc = ensure_init();
  if (rc != BGMOE_OK) return rc;
  const int vecs = backward_vecs(a.h), threads = threads_for(a.h, vecs);
  BgmoeProf prof(BGMOE_K_GATED_NORM, st);
  const dim3 grid((unsigned)s.blocks), block(threads);
  if (vecs == 2) hipLaunchKernelGGL((gated_norm_backward_kernel<T, 2, false, false>), grid, block, 0, st, a);
  else if (!past_cache<T>(a, 6)) hipLaunchKernelGGL((gated_norm_backward_kernel<T, 1, true, false>), grid, block, threads * kAccBytes, st, a);
  else hipLaunchKernelGGL((gated_norm_backward_kernel<T, 1, true, true>), grid, block, threads * kAccBytes, st, a);
  if (s.kinds) {
    const int64_t cols = (int64_t)s.kinds * s.h;
    hipLaunchKernelGGL((plane_sum_kernel<T>), dim3((unsigned)((cols + 63) / 64)), dim3(1024), 0, st, s);
  }
  return bgmoe_check_launch("gated_residual_norm_backward");
}

int check_common(const char* what, int dtype, const void* gate, int gate_mode, int64_t rows, int h, const void* block,
                 const void* residual) {
  BGMOE_REQUIRE(dtype >= BGMOE_DT_BF16 && dtype <= BGMOE_DT_FP32, "%s: unknown element type %d", what, dtype);
  BGMOE_REQUIRE(rows >= 0 && rows <= 0x7fffffffLL, "%s: bad row count %lld", what, (long long)rows);
  BGMOE_REQUIRE(h >= 1 && h <= kMaxH, "%s: row width %d outside [1,%d]", what, h, kMaxH);
  BGMOE_REQUIRE(gate_mode >= BGMOE_GATE_NONE && gate_mode <= BGMOE_GATE_FULL, "%s: unknown gate_mode %d", what, gate_mode);
  BGMOE_REQUIRE((gate_mode == BGMOE_GATE_NONE) == (gate == nullptr), "%s: gate and gate_mode do not agree", what);
  BGMOE_REQUIRE(rows == 0 || (block && residual), "%s: null pointer", what);
  return BGMOE_OK;
}

}  // namespace

int bgmoe_internal_init_gated_norm() { return ensure_init(); }

extern "C" int bgmoe_gated_residual_norm(const void* block, const void* residual, int dtype, const void* post_weight,
                                         const void* gate, int gate_mode, float residual_scale, const void* pre_weight,
                                         int param_fp32, int64_t rows, int h, float eps, void* y, void* normed, int8_t* q,
                                         float* q_scale, float* inv_post, float* inv_pre, bgmoe_stream_t stream) {
  const int rc = check_common("gated_residual_norm", dtype, gate, gate_mode, rows, h, block, residual);
  if (rc != BGMOE_OK) return rc;
  if (rows == 0) return BGMOE_OK;
  BGMOE_REQUIRE(y, "gated_residual_norm: null pointer");
  BGMOE_REQUIRE(pre_weight || (!normed && !q), "gated_residual_norm: normed / q without pre_weight");
  BGMOE_REQUIRE(!q == !q_scale, "gated_residual_norm: q and q_scale come together");
  BGMOE_REQUIRE(!pre_weight || normed || q, "gated_residual_norm: pre_weight without an output for its norm");
  NormArgs a{};
  a.block = block; a.residual = residual; a.post = post_weight; a.gate = gate; a.pre = pre_weight;
  a.gate_mode = gate_mode; a.param_fp32 = param_fp32; a.scale = residual_scale; a.eps = eps; a.rows = rows; a.h = h;
  a.y = y; a.normed = normed; a.q = q; a.q_scale = q_scale; a.inv_post = inv_post; a.inv_pre = inv_pre;
#define BGMOE_CALL(T) run_forward<T>(a, bgmoe_stream(stream))
  BGMOE_BY_TYPE(dtype, BGMOE_CALL);
#undef BGMOE_CALL
}

extern "C" size_t bgmoe_gated_residual_norm_backward_workspace_bytes(int64_t rows, int h) {
  if (rows <= 0 || h < 1 || h > kMaxH) return 0;
  return (size_t)backward_blocks(rows, h) * 3 * (size_t)h * sizeof(float);
}

extern "C" int bgmoe_gated_residual_norm_backward(const void* block, const void* residual, int dtype,
                                                  const void* post_weight, const void* gate, int gate_mode,
                                                  float residual_scale, const void* pre_weight, int param_fp32,
                                                  int64_t rows, int h, const float* inv_post, const float* inv_pre,
                                                  const void* d_y, const void* d_normed, void* d_block, void* d_residual,
                                                  void* d_post, void* d_gate, void* d_pre, void* workspace,
                                                  size_t workspace_bytes, bgmoe_stream_t stream) {
  const int rc = check_common("gated_residual_norm_backward", dtype, gate, gate_mode, rows, h, block, residual);
  if (rc != BGMOE_OK) return rc;
  BGMOE_REQUIRE(rows > 0, "gated_residual_norm_backward: no rows (the gradients of the weights are zero)");
  BGMOE_REQUIRE(!d_post || post_weight, "gated_residual_norm_backward: d_post without post_weight");
  BGMOE_REQUIRE(!d_pre || pre_weight, "gated_residual_norm_backward: d_pre without pre_weight");
  BGMOE_REQUIRE(!d_gate || gate, "gated_residual_norm_backward: d_gate without a gate");
  BGMOE_REQUIRE(!d_normed || pre_weight, "gated_residual_norm_backward: d_normed without pre_weight");
  BGMOE_REQUIRE((!post_weight || inv_post) && (!pre_weight || inv_pre),
                "gated_residual_norm_backward: the forward pass's inv_post / inv_pre are needed");
  NormArgs a{};
  a.block = block; a.residual = residual; a.post = post_weight; a.gate = gate; a.pre = pre_weight;
  a.gate_mode = gate_mode; a.param_fp32 = param_fp32; a.scale = residual_scale; a.rows = rows; a.h = h;
  a.i_post = inv_post; a.i_pre = inv_pre; a.dy = d_y; a.dn = d_normed; a.d_block = d_block; a.d_residual = d_residual;
  a.d_gate = d_gate;
  a.want_post = d_post != nullptr; a.want_pre = d_pre != nullptr;
  a.want_gate = d_gate != nullptr && gate_mode == BGMOE_GATE_CHANNEL;
  SumArgs s{};
  s.blocks = (int)backward_blocks(rows, h); s.h = h;
  if (a.want_post) { s.fp32[s.kinds] = param_fp32 & 1; s.out[s.kinds++] = d_post; }
  if (a.want_pre) { s.fp32[s.kinds] = param_fp32 & 4; s.out[s.kinds++] = d_pre; }
  if (a.want_gate) { s.fp32[s.kinds] = param_fp32 & 2; s.out[s.kinds++] = d_gate; }
  if (s.kinds) {
    const size_t need = (size_t)s.blocks * s.kinds * h * sizeof(float);
    if (workspace == nullptr || workspace_bytes < need) {
      bgmoe_set_error("gated_residual_norm_backward: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
      return BGMOE_ERR_WORKSPACE;
    }
    BGMOE_REQUIRE((uintptr_t)workspace % 4 == 0, "gated_residual_norm_backward: workspace must be 4-byte aligned");
  }
  a.planes = (float*)workspace;
  s.planes = a.planes;
#define BGMOE_CALL(T) run_backward<T>(a, s, bgmoe_stream(stream))
  BGMOE_BY_TYPE(dtype, BGMOE_CALL);
#undef BGMOE_CALL
}
