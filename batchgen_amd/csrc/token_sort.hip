// Tokens sorted by expert and brought back with their routing weights, and the gradients of both, for gfx950.
//
//   sort      rows[pos[t,j]] = x[t]                          gradient: dx[t] = sum_j drows[pos[t,j]]  (unsort, no weights)
//   unsort    out[t] = sum_j w[t,j] * y[pos[t,j]]            gradient: dy[pos[t,j]] = w[t,j] * dout[t],
//                                                                      dw[t,j] = <dout[t], y[pos[t,j]]>
//
// pos comes from the stable counting sort of permute.hip; pos = -1 marks a pair without a row here (another rank's
// expert, a padding token).  All four are bound by HBM: a token's row moves once and its k expert rows once per
// direction.  Every kernel therefore walks TOKENS, not pairs: the token side is read (or written) once, from registers
// to k places, and no output has two writers, so there are no atomics and the results are one function of the inputs.
#include "bgmoe_elem.h"

namespace {

constexpr int kMaxK = 32;
constexpr int kRestBlocks = 256;      // blocks that clear rows without a pair

struct Rest {                          // the rows of a sorted buffer that hold no pair
  const int32_t* counts;
  const int32_t* cu;
  int experts;
  int64_t rows, row_bytes;
  uint8_t* out;
};

// one wave clears one row
__device__ __forceinline__ void clear_row(const Rest& r, int64_t row) {
  uint8_t* p = r.out + row * r.row_bytes;
  const int lane = lane_id();
  if (r.row_bytes < 16) {
    if (lane < r.row_bytes) p[lane] = 0;
    return;
  }
  for (int64_t o = lane * 16; o < r.row_bytes; o += 1024) store16(p + min(o, r.row_bytes - 16), u32x4{0u, 0u, 0u, 0u});
}
__device__ __forceinline__ void clear_rest(const Rest& r, int64_t wave, int64_t waves) {
  for (int64_t row = (int64_t)r.cu[r.experts] + wave; row < r.rows; row += waves) clear_row(r, row);
  for (int64_t e = wave; e < r.experts; e += waves) {
    const int64_t end = min((int64_t)r.cu[e + 1], r.rows);
    for (int64_t row = (int64_t)r.cu[e] + r.counts[e]; row < end; ++row) clear_row(r, row);
  }
}

// One wave moves up to 4 KB of one token's row: four 16-byte loads per lane, then the same registers to every row the
// token has.  A row's last 16 bytes are moved by a vector that ends with the row (it may overlap its neighbour, which
// writes the same bytes); rows shorter than 16 bytes go byte by byte.
constexpr int kSegBytes = 4096;
template <bool NT>
__global__ __launch_bounds__(256) void sort_rows_kernel(const uint8_t* __restrict__ x, int64_t stride, int64_t row_bytes,
                                                        int64_t n, int k, int segs, const int32_t* __restrict__ pos,
                                                        uint8_t* __restrict__ out, int64_t job_blocks, int64_t all_blocks,
                                                        Rest rest) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = lane_id();
  const int64_t block = linear_block();
  if (block >= job_blocks) {
    if (block < all_blocks) clear_rest(rest, (block - job_blocks) * 4 + wave, (all_blocks - job_blocks) * 4);
    return;
  }
  const int64_t job = block * 4 + wave;
  const int64_t t = job / segs;
  if (t >= n) return;
  const int64_t seg0 = (job - t * segs) * kSegBytes;
  const int32_t mine = lane < k ? pos[t * k + lane] : -1;
  unsigned long long live = __ballot(mine >= 0 && mine < rest.rows);
  if (live == 0ull) return;
  const uint8_t* src = x + t * stride;
  if (row_bytes < 16) {
    while (live) {
      const int64_t dst = __builtin_amdgcn_readlane(mine, __ffsll((long long)live) - 1);
      live &= live - 1;
      if (lane < row_bytes) out[dst * row_bytes + lane] = src[lane];
    }
    return;
  }
  u32x4 v[4];
  int64_t off[4];
  bool in[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t o = seg0 + i * 1024 + lane * 16;
    in[i] = o < row_bytes;
    off[i] = min(o, row_bytes - 16);
    if (in[i]) v[i] = load16(src + off[i]);
  }
  while (live) {
    const int64_t dst = __builtin_amdgcn_readlane(mine, __ffsll((long long)live) - 1);
    live &= live - 1;
    uint8_t* d = out + dst * row_bytes;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (in[i]) store16_as<NT>(d + off[i], v[i]);
  }
}

// One wave sums one token's rows over 64 x 16 bytes of columns: the loads of up to 8 rows are in flight together, the
// sum is taken in slot order (fused multiply-adds).  The vector that ends with the row may overlap its neighbour:
// both compute the same values.
template <typename T, bool NT>
__global__ __launch_bounds__(256) void unsort_kernel(const uint8_t* __restrict__ rows, const int32_t* __restrict__ pos,
                                                     const float* __restrict__ weights, int64_t n, int k, int h, int segs,
                                                     uint8_t* __restrict__ out) {
  constexpr int W = kPer16<T>;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t job = linear_block() * 4 + wave;
  const int64_t t = job / segs;
  if (t >= n) return;
  const int64_t row_bytes = (int64_t)h * T::kBytes;
  int64_t o = (job - t * segs) * 1024 + lane_id() * 16;
  const int32_t* tp = pos + t * k;
  const float* tw = weights + t * k;
  if (row_bytes < 16) {                                   // a row narrower than a vector: one element per lane
    const int c = lane_id();
    if (c >= h) return;
    float acc = 0.0f;
    for (int j = 0; j < k; ++j)
      if (tp[j] >= 0)
        acc = __builtin_fmaf(load_one<T>(rows + (int64_t)tp[j] * row_bytes + c * T::kBytes), weights ? tw[j] : 1.0f, acc);
    store_one<T>(out + t * row_bytes + c * T::kBytes, acc);
    return;
  }
  if (o >= row_bytes) return;
  o = min(o, row_bytes - 16);
  float acc[W];
#pragma unroll
  for (int i = 0; i < W; ++i) acc[i] = 0.0f;
  for (int j0 = 0; j0 < k; j0 += 8) {
    u32x4 raw[8];
    float wj[8];
    bool on[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int j = j0 + u;
      const int p = j < k ? tp[j] : -1;
      on[u] = p >= 0;
      wj[u] = 1.0f;
      if (on[u]) {
        if (weights) wj[u] = tw[j];
        raw[u] = load16_as<NT>(rows + (int64_t)p * row_bytes + o);
      }
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (on[u]) {
        float v[W];
        unpack16<T>(raw[u], v);
#pragma unroll
        for (int i = 0; i < W; ++i) acc[i] = __builtin_fmaf(v[i], wj[u], acc[i]);
      }
    }
  }
  store16(out + t * row_bytes + o, pack16<T>(acc));
}

// Gradients of unsort: one block per token walks the columns; a thread holds 16 bytes of dout, reads the same columns
// of up to 8 expert rows, adds to their dot products and writes their gradients.  The dot products are summed over
// the wave by shuffles, over the waves in wave order.
template <typename T, int THREADS, bool NT>
__global__ __launch_bounds__(THREADS) void unsort_backward_kernel(const uint8_t* __restrict__ dout, const uint8_t* __restrict__ rows,
                                                             const int32_t* __restrict__ pos,
                                                             const float* __restrict__ weights, int64_t n, int k, int h,
                                                             uint8_t* __restrict__ drows, float* __restrict__ dw, Rest rest) {
  constexpr int W = kPer16<T>;
  __shared__ float s_dot[THREADS / 64][8];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = lane_id();
  const int64_t t = linear_block();
  if (t >= n) {
    if (drows && t < n + kRestBlocks) clear_rest(rest, (t - n) * (THREADS / 64) + wave, (int64_t)kRestBlocks * (THREADS / 64));
    return;
  }
  const int64_t row_bytes = (int64_t)h * T::kBytes;
  const uint8_t* g = dout + t * row_bytes;
  for (int j0 = 0; j0 < k; j0 += 8) {
    float dot[8], wj[8];
    int p[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      dot[u] = 0.0f;
      p[u] = j0 + u < k ? pos[t * k + j0 + u] : -1;
      wj[u] = p[u] >= 0 && weights ? weights[t * k + j0 + u] : 1.0f;
    }
    for (int64_t o = threadIdx.x * 16; o < row_bytes; o += THREADS * 16) {
      const int64_t left = row_bytes - o;
      if (left >= 16) {
        float gv[W];
        unpack16<T>(load16(g + o), gv);
        u32x4 raw[8];
        if (dw) {
#pragma unroll
          for (int u = 0; u < 8; ++u)
            if (p[u] >= 0) raw[u] = load16_as<NT>(rows + (int64_t)p[u] * row_bytes + o);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          if (p[u] < 0) continue;
          if (dw) {
            float v[W];
            unpack16<T>(raw[u], v);
#pragma unroll
            for (int i = 0; i < W; ++i) dot[u] = __builtin_fmaf(v[i], gv[i], dot[u]);
          }
          if (drows) {
            float d[W];
#pragma unroll
            for (int i = 0; i < W; ++i) d[i] = wj[u] * gv[i];
            store16_as<NT>(drows + (int64_t)p[u] * row_bytes + o, pack16<T>(d));
          }
        }
      } else {                                            // the row's last elements, one by one
        for (int64_t c = o; c < row_bytes; c += T::kBytes) {
          const float gc = load_one<T>(g + c);
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            if (p[u] < 0) continue;
            if (dw) dot[u] = __builtin_fmaf(load_one<T>(rows + (int64_t)p[u] * row_bytes + c), gc, dot[u]);
            if (drows) store_one<T>(drows + (int64_t)p[u] * row_bytes + c, wj[u] * gc);
          }
        }
      }
    }
    if (dw) {
#pragma unroll
      for (int u = 0; u < 8; ++u) {
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) dot[u] = dot[u] + __shfl_xor(dot[u], off, BGMOE_WAVE);
        if (lane == 0) s_dot[wave][u] = dot[u];
      }
      __syncthreads();
      if (threadIdx.x < 8 && j0 + (int)threadIdx.x < k) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) sum += s_dot[w][threadIdx.x];
        dw[t * k + j0 + threadIdx.x] = sum;               // a pair without a row added nothing: 0
      }
      __syncthreads();
    }
  }
}

// Expert rows that together exceed the 256 MB last-level cache bypass it: 16384 tokens x 8 x 7168 bf16 (1.9 GB) sort 414 ->
// 362 us (5.8 TB/s), unsort 415 -> 368, its gradients 808 -> 754; rows that fit are better left to it: 4096 x 8 x 2048
// (134 MB) sort 24.2 us (6.2 TB/s) against 27.8, unsort 24.8 against 28.8, gradients 47.0 against 52.9.
// All n * k pairs are counted, which is what the host knows: on a rank that holds a part of the experts the rows that move
// may fit where this bypasses.
bool past_cache(int64_t pairs, int64_t row_bytes) { return pairs * row_bytes > (256LL << 20); }

template <typename T>
int run_unsort(const void* rows, const int32_t* pos, const float* weights, int n, int k, int h, void* out, hipStream_t st) {
  const int64_t row_bytes = (int64_t)h * T::kBytes;
  const int segs = (int)((row_bytes + 1023) / 1024);
  const int64_t blocks = ((int64_t)n * segs + 3) / 4;
  BGMOE_REQUIRE(blocks <= kBgmoeMaxBlocks, "token_unsort: %d tokens of %d columns are too many for one launch", n, h);
  BgmoeProf prof(BGMOE_K_TOKEN_UNSORT, st);
#define BGMOE_LAUNCH(NT)                                                                                                     \
  hipLaunchKernelGGL((unsort_kernel<T, NT>), bgmoe_grid(blocks), dim3(256), 0, st, (const uint8_t*)rows, pos, weights,         \
                     (int64_t)n, k, h, segs, (uint8_t*)out)
  if (past_cache((int64_t)n * k, row_bytes)) BGMOE_LAUNCH(true);
  else BGMOE_LAUNCH(false);
#undef BGMOE_LAUNCH
  return bgmoe_check_launch("token_unsort");
}

template <typename T>
int run_unsort_backward(const void* dout, const void* rows, const int32_t* pos, const float* weights, int n, int k, int h,
                        void* drows, float* dw, const Rest& rest, hipStream_t st) {
  const int64_t blocks = (int64_t)n + (drows ? kRestBlocks : 0), row_bytes = (int64_t)h * T::kBytes;
  BGMOE_REQUIRE(blocks <= kBgmoeMaxBlocks, "token_unsort_backward: %d tokens are too many for one launch", n);
  BgmoeProf prof(BGMOE_K_TOKEN_UNSORT, st);
#define BGMOE_LAUNCH(THREADS, NT)                                                                                            \
  hipLaunchKernelGGL((unsort_backward_kernel<T, THREADS, NT>), bgmoe_grid(blocks), dim3(THREADS), 0, st, (const uint8_t*)dout, \
                     (const uint8_t*)rows, pos, weights, (int64_t)n, k, h, (uint8_t*)drows, dw, rest)
  const bool nt = past_cache((int64_t)n * k, row_bytes);
  if (row_bytes <= 1024) {                                // one wave covers 1 KB of columns at a time
    if (nt) BGMOE_LAUNCH(64, true);
    else BGMOE_LAUNCH(64, false);
  } else {
    if (nt) BGMOE_LAUNCH(256, true);
    else BGMOE_LAUNCH(256, false);
  }
#undef BGMOE_LAUNCH
  return bgmoe_check_launch("token_unsort_backward");
}

}  // namespace

extern "C" int bgmoe_token_sort_rows(const void* x, int64_t x_row_stride, int64_t row_bytes, int n, int k,
                                     const int32_t* topk_pos, const int32_t* counts, const int32_t* cu_seqlens,
                                     int num_local_experts, int64_t rows, int zero_rest, void* out, bgmoe_stream_t stream) {
  BGMOE_REQUIRE(n >= 0 && rows >= 0 && row_bytes >= 0, "token_sort_rows: negative size");
  BGMOE_REQUIRE(k >= 1 && k <= kMaxK, "token_sort_rows: top-k %d outside [1,%d]", k, kMaxK);
  BGMOE_REQUIRE(num_local_experts >= 1, "token_sort_rows: no experts");
  if (row_bytes == 0 || rows == 0) return BGMOE_OK;
  BGMOE_REQUIRE(out && counts && cu_seqlens && (n == 0 || (x && topk_pos)), "token_sort_rows: null pointer");
  const int64_t segs = (row_bytes + kSegBytes - 1) / kSegBytes;
  const int64_t jobs = ((int64_t)n * segs + 3) / 4, blocks = jobs + (zero_rest ? kRestBlocks : 0);
  BGMOE_REQUIRE(segs <= 0x7fffffffLL && blocks <= kBgmoeMaxBlocks,
                "token_sort_rows: %d tokens of %lld bytes are too many for one launch", n, (long long)row_bytes);
  if (blocks == 0) return BGMOE_OK;
  const Rest rest{counts, cu_seqlens, num_local_experts, rows, row_bytes, (uint8_t*)out};
  hipStream_t st = bgmoe_stream(stream);
  BgmoeProf prof(BGMOE_K_TOKEN_SORT, st);
#define BGMOE_LAUNCH(NT)                                                                                                     \
  hipLaunchKernelGGL((sort_rows_kernel<NT>), bgmoe_grid(blocks), dim3(256), 0, st, (const uint8_t*)x, x_row_stride, row_bytes, \
                     (int64_t)n, k, (int)segs, topk_pos, (uint8_t*)out, jobs, blocks, rest)
  if (past_cache((int64_t)n * k, row_bytes)) BGMOE_LAUNCH(true);
  else BGMOE_LAUNCH(false);
#undef BGMOE_LAUNCH
  return bgmoe_check_launch("token_sort_rows");
}

extern "C" int bgmoe_token_unsort(const void* rows, int dtype, const int32_t* topk_pos, const float* weights, int n, int k,
                                  int h, void* out, bgmoe_stream_t stream) {
  BGMOE_REQUIRE(n >= 0 && h >= 0, "token_unsort: negative size");
  BGMOE_REQUIRE(k >= 1 && k <= kMaxK, "token_unsort: top-k %d outside [1,%d]", k, kMaxK);
  BGMOE_REQUIRE(dtype >= BGMOE_DT_BF16 && dtype <= BGMOE_DT_FP32, "token_unsort: unknown element type %d", dtype);
  if (n == 0 || h == 0) return BGMOE_OK;
  BGMOE_REQUIRE(rows && topk_pos && out, "token_unsort: null pointer");
#define BGMOE_CALL(T) run_unsort<T>(rows, topk_pos, weights, n, k, h, out, bgmoe_stream(stream))
  BGMOE_BY_TYPE(dtype, BGMOE_CALL);
#undef BGMOE_CALL
}

extern "C" int bgmoe_token_unsort_backward(const void* d_out, const void* rows, int dtype, const int32_t* topk_pos,
                                           const float* weights, int n, int k, int h, const int32_t* counts,
                                           const int32_t* cu_seqlens, int num_local_experts, int64_t num_rows, void* d_rows,
                                           float* d_weights, bgmoe_stream_t stream) {
  BGMOE_REQUIRE(n >= 0 && h >= 0 && num_rows >= 0, "token_unsort_backward: negative size");
  BGMOE_REQUIRE(k >= 1 && k <= kMaxK, "token_unsort_backward: top-k %d outside [1,%d]", k, kMaxK);
  BGMOE_REQUIRE(dtype >= BGMOE_DT_BF16 && dtype <= BGMOE_DT_FP32, "token_unsort_backward: unknown element type %d", dtype);
  BGMOE_REQUIRE(num_local_experts >= 1, "token_unsort_backward: no experts");
  if (!d_rows && !d_weights) return BGMOE_OK;
  if (n == 0 && num_rows == 0) return BGMOE_OK;
  // rows without elements may have no address; their weights' gradient is 0
  BGMOE_REQUIRE(counts && cu_seqlens && (n == 0 || ((d_out || h == 0) && topk_pos)), "token_unsort_backward: null pointer");
  BGMOE_REQUIRE(n == 0 || !d_weights || rows || h == 0, "token_unsort_backward: the weights' gradient needs the rows");
  const int size = dtype == BGMOE_DT_FP32 ? 4 : 2;
  const Rest rest{counts, cu_seqlens, num_local_experts, num_rows, (int64_t)h * size, (uint8_t*)d_rows};
#define BGMOE_CALL(T) \
  run_unsort_backward<T>(d_out, rows, topk_pos, weights, n, k, h, d_rows, d_weights, rest, bgmoe_stream(stream))
  BGMOE_BY_TYPE(dtype, BGMOE_CALL);
#undef BGMOE_CALL
}
