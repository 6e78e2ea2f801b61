// Products in 8-bit integers for gfx950: out[t][j] = (sum_k x[t][k] w[j][k]) * xs[t] * ws[j], dense or grouped by
// expert, and the row quantiser in front of them.
//
// Both operands are K-major rows, which is what v_mfma_i32_16x16x64_i8 takes: lane l = 16 q + r supplies the 16 bytes
// k = 16 q .. 16 q + 15 of row r.  With the weights as first operand a lane's four results are four consecutive output
// columns of one token.  The accumulators are exact 32-bit integers (|sum| <= k * 128^2 < 2^31 for k <= 131071), so
// no result depends on how K is cut; the scales enter once, in fp32, in the epilogue.
//
// Streaming kernel, for groups of up to 32 rows: a block owns 64 weight rows (4 waves x 16), 16 or 32 tokens and all of K.
// It is bound by the weights' stream from HBM (32 experts x 8 rows, gate + up of 2048 x 7168: 940 MB in 140 us, 6.7 TB/s).
// Weights and tokens go global -> LDS asynchronously in stages of 256 bytes of K (one 1 KB wave load
// covers 4 rows x 256 contiguous bytes) into a ring; a stage's 16-byte chunks are stored at position
// chunk ^ (row & 15), so that the 16 lanes that read one chunk of 16 rows hit 16 different 16-byte slots of the 256
// bytes the LDS serves at once.
#include "bgmoe_async.h"
#include "bgmoe_elem.h"

namespace {

constexpr int kMaxK = 131071;                 // k * 128 * 128 < 2^31
constexpr int kStageK = 256;                  // bytes of K per stage
constexpr int kTile = 16 * kStageK;           // 16 rows of a stage: 4 KB
constexpr int kRingBytes = 80 * 1024;         // two blocks per CU

__device__ const uint4 g_zeros = {0u, 0u, 0u, 0u};     // what chunks past K read

struct Int8Args {
  const int8_t* x;
  int64_t ldx;                                // bytes between rows of x
  const float* xs;
  const int8_t *w0, *w1;                      // w1: the up projection of a fused stage 1, else null
  int64_t w0_group, w1_group;
  const float *ws0, *ws1;
  int64_t ws0_group, ws1_group;
  const float* bias;
  const int32_t *seqlens, *cu;                // null: one group of all m rows
  int64_t m;
  int n, k;
  uint8_t* out;
  int64_t ldo;                                // elements between rows of out
  int out_dtype;
  int past_cache;                             // the streaming kernel's weights bypass the last-level cache
};

// four consecutive columns of one output row
__device__ __forceinline__ void store4(const Int8Args& a, int64_t row, int col, const float (&v)[4]) {
  const int left = a.n - col;
  if (left <= 0) return;
  typedef unsigned int u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
  if (a.out_dtype == BGMOE_DT_FP32) {
    float* p = reinterpret_cast<float*>(a.out) + row * a.ldo + col;
    if (left >= 4) store16(p, u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
    else for (int i = 0; i < left; ++i) p[i] = v[i];
    return;
  }
  uint16_t* p = reinterpret_cast<uint16_t*>(a.out) + row * a.ldo + col;
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    b[i] = a.out_dtype == BGMOE_DT_BF16 ? f32_to_bf16_bits(v[i]) : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[i]);
  if (left >= 4) *reinterpret_cast<u32x2_any*>(p) = u32x2_any{b[0] | (b[1] << 16), b[2] | (b[3] << 16)};
  else for (int i = 0; i < left; ++i) p[i] = (uint16_t)b[i];
}

// rows [row0, row0 + cnt) of group g; counts and offsets that reach outside [0, m] are cut
__device__ __forceinline__ void group_rows(const Int8Args& a, int g, int64_t* row0, int* cnt) {
  if (a.seqlens == nullptr) {
    *row0 = 0;
    *cnt = (int)a.m;
    return;
  }
  const int64_t r = a.cu[g];
  const int64_t end = min(r + (int64_t)a.seqlens[g], a.m);
  *row0 = r;
  *cnt = r >= 0 && end > r ? (int)(end - r) : 0;
}

template <bool FUSED, int MT>
__device__ __forceinline__ void stream_chunk(const Int8Args& a, uint8_t* smem, const int8_t* wbase, int wrow0, int wrows,
                                             const float* ws, const float* ws_up, int64_t row0, int cnt, int n0) {
  constexpr int kStage = (4 + MT) * kTile;             // 64 weight rows, 16 MT tokens
  constexpr int kStages = kRingBytes / kStage;         // 4 or 3
  constexpr int kLoads = 4 + MT;                       // wave loads per stage and wave
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int r = lane & 15, q = lane >> 4;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)smem);
  const int S = (a.k + kStageK - 1) / kStageK;
  const int chunks = a.k >> 4;                          // 16-byte chunks of a row

  // sources: lane l of wave load i covers row 4 i + l/16 of the tile, LDS position l % 16, i.e. source chunk
  // (l % 16) ^ (row & 15)
  const int lr = lane >> 4, lc = lane & 15;
  uint32_t w_off[4], x_off[MT];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 4 * i + lr;
    w_off[i] = (uint32_t)min(row, wrows - 1) * (uint32_t)a.k + (uint32_t)((lc ^ row) * 16);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int row = 4 * (wave * MT + i) + lr;           // token of the chunk
    x_off[i] = (uint32_t)min(row, cnt - 1) * (uint32_t)a.ldx + (uint32_t)((lc ^ (row & 15)) * 16);
  }
  const uint8_t* wsrc = uniform_ptr(reinterpret_cast<const uint8_t*>(wbase) + (int64_t)wrow0 * a.k);
  const uint8_t* xsrc = uniform_ptr(reinterpret_cast<const uint8_t*>(a.x) + row0 * a.ldx);

  auto issue = [&](int s) {
    const uint32_t d = lds0 + (uint32_t)(s % kStages) * kStage;
    const uint32_t dw = d + wave * kTile, dx = d + 4 * kTile + wave * MT * 1024;
    const int ko = s * kStageK;
    if ((s + 1) * 16 <= chunks) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (a.past_cache) async_load16_nt(wsrc + ko, w_off[i], dw + i * 1024);
        else async_load16(wsrc + ko, w_off[i], dw + i * 1024);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) async_load16(xsrc + ko, x_off[i], dx + i * 1024);
    } else {                                            // the last, partial stage: chunks past K read zeros
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = s * 16 + (lc ^ (4 * i + lr)) < chunks;
        async_load16_lane(in ? (const void*)(wsrc + ko + w_off[i]) : (const void*)&g_zeros, dw + i * 1024);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const bool in = s * 16 + (lc ^ ((4 * (wave * MT + i) + lr) & 15)) < chunks;
        async_load16_lane(in ? (const void*)(xsrc + ko + x_off[i]) : (const void*)&g_zeros, dx + i * 1024);
      }
    }
  };

  intx4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = intx4{0, 0, 0, 0};
  for (int s = 0; s < kStages - 1 && s < S; ++s) issue(s);
  for (int s = 0; s < S; ++s) {
    // stages s + 1 .. s + kStages - 2 may still be in flight
    if (S - 1 - s >= kStages - 2) wait_vm<(kStages - 2) * kLoads>();
    else wait_vm<0>();
    lds_exchange_barrier();                             // everybody's share has landed; everybody is done with stage s - 1
    if (s + kStages - 1 < S) issue(s + kStages - 1);
    const uint8_t* b = smem + (s % kStages) * kStage;
    const uint8_t* bw = b + wave * kTile + r * kStageK;
    const uint8_t* bx = b + 4 * kTile + r * kStageK;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int o = ((4 * c + q) ^ r) * 16;
      const intx4 wv = *reinterpret_cast<const intx4*>(bw + o);
#pragma unroll
      for (int t = 0; t < MT; ++t)
        acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv, *reinterpret_cast<const intx4*>(bx + t * kTile + o), acc[t], 0, 0, 0);
    }
  }
  lds_exchange_barrier();                               // the ring is free

  // epilogue: lane (r, q) holds columns 4 q .. 4 q + 3 of this wave's 16 for token r of each 16-token tile
  if constexpr (FUSED) {
    // waves 0, 1: gate rows, waves 2, 3: the up rows of the same columns, handed over through LDS
    float* up = reinterpret_cast<float*>(smem);
    const int col = n0 + (wave & 1) * 16 + 4 * q;
    float sc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) sc[i] = (wave < 2 ? ws : ws_up)[min(col + i, a.n - 1)];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const float xs = a.xs[row0 + min(16 * t + r, cnt - 1)];
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = (float)acc[t][i] * xs * sc[i];
      if (wave >= 2)
#pragma unroll
        for (int i = 0; i < 4; ++i) up[(((wave & 1) * MT + t) * 4 + i) * 64 + lane] = v[i];
      else
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = __float_as_int(v[i]);
    }
    __syncthreads();
    if (wave < 2) {
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[i] = silu_f32(__int_as_float(acc[t][i])) * up[((wave * MT + t) * 4 + i) * 64 + lane];
        const int tok = 16 * t + r;
        if (tok < cnt) store4(a, row0 + tok, col, v);
      }
    }
  } else {
    const int col = n0 + wave * 16 + 4 * q;
    float sc[4], bias[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sc[i] = ws[min(col + i, a.n - 1)];
      bias[i] = a.bias ? a.bias[min(col + i, a.n - 1)] : 0.0f;
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int tok = 16 * t + r;
      if (tok >= cnt) continue;
      const float xs = a.xs[row0 + tok];
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = (float)acc[t][i] * xs * sc[i];
        if (a.bias) v[i] += bias[i];
      }
      store4(a, row0 + tok, col, v);
    }
  }
}

template <bool FUSED>
__global__ __launch_bounds__(256) void int8_stream_kernel(Int8Args a, int max_rows) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int g = blockIdx.y;
  int64_t row0;
  int cnt;
  group_rows(a, g, &row0, &cnt);
  if (cnt == 0 || cnt > max_rows) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * (FUSED ? 32 : 64);
  const bool second = FUSED && wave >= 2;
  const int8_t* wbase = second ? a.w1 + g * a.w1_group : a.w0 + g * a.w0_group;
  const float* ws = a.ws0 + g * a.ws0_group;
  const float* ws_up = FUSED ? a.ws1 + g * a.ws1_group : nullptr;
  // this wave's 16 weight rows; a wave whose rows all lie past n repeats the last row and stores nothing
  const int wrow0 = min(n0 + (FUSED ? wave & 1 : wave) * 16, a.n - 1);
  const int wrows = min(16, a.n - wrow0);
  if (cnt <= 16) stream_chunk<FUSED, 1>(a, smem, wbase, wrow0, wrows, ws, ws_up, row0, cnt, n0);
  else stream_chunk<FUSED, 2>(a, smem, wbase, wrow0, wrows, ws, ws_up, row0, cnt, n0);
}

// ---- tiled kernel: many rows per group ---------------------------------------------------------------------------------
// Macro tile 256 tokens x 256 weight rows (fused: 128 gate + 128 up), 8 waves = 4 (64 weight rows) x 2 (128 tokens); a wave
// holds 4 x 8 tiles of v_mfma_i32_16x16x64_i8, 128 accumulators.  K advances 128 bytes per step through two 64 KB slots.
// Whole 128-byte lines on purpose: a CU takes in 134 GB/s through asynchronous loads whose lanes cover 128-byte pieces of
// rows, 65 GB/s with 64-byte pieces, however many are in flight; a step needs 64 KB in the 0.9 us its MFMAs take.
// A step is two halves of 64 bytes.  While a half is multiplied the operands of the next one are read from LDS, and in
// the second half the step after next is requested; both are spread between the MFMAs, two reads and one load per
// four (all of them behind the barrier: 20% more time per step with 16 CUs at work, since 64 loads keep the CU's address
// unit busy for as long as half the step's MFMAs).  One barrier per step:
//
//   multiply half 0, read half 1 | wait for the next step's loads and this wave's reads, barrier: the next step is there,
//   this slot is free | multiply half 1, read the next step's half 0, request step s + 2 into this slot
//
// A row's eight 16-byte chunks of a step lie at chunk ^ ((row / 2) & 7): the 16 lanes that read one chunk of 16 rows hit
// 16 different 16-byte slots of 256 bytes (no bank conflicts by the counter).
// Bound: the chip's power.  With every CU at work the MFMAs alone run at 3.2 (32x32x32) and 3.6 (16x16x64) PFLOP/s on
// normally distributed bytes, because the clock falls to about 1.6 GHz; this loop runs at 2.7.
// Tile<4, 8> is that macro tile.  Tile<2, 4> is 128 x 128 with 4 waves of 4 x 4 tiles and two 32 KB slots, two blocks per
// CU: half the products per byte requested, four times the tiles, for problems whose large tiles would not fill the
// chip (four slots, i.e. one block per CU with three steps in flight, are no faster with few tiles and slower with many).
template <int WN_, int XT_> struct Tile {
  static constexpr int WN = WN_, XT = XT_;              // waves along the weights; token tiles per wave
  static constexpr int W = 64 * WN_, M = 32 * XT_;      // weight rows and tokens of a macro tile
  static constexpr int kThreads = 128 * WN_;            // WN x 2 waves, each of which loads 32 rows of either operand
  static constexpr int kSlot = (W + M) * 128;
  static constexpr int kRing = 2 * kSlot;
  static_assert(W == 64 * WN_ && M == 64 * WN_, "every wave loads 32 token rows and 32 weight rows");
};
typedef Tile<4, 8> Large;
typedef Tile<2, 4> Small;
constexpr int kTK = 128;
constexpr int kMaxGroups = 1024;
constexpr int kPanel = 8;                     // m-tiles that share their weight tiles in an XCD's L2

// four consecutive per-column values, the last one repeated past n
__device__ __forceinline__ void load_cols(const float* p, int col, int n, float (&v)[4]) {
  if (col + 3 < n) {
    const u32x4 r = load16(p + col);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = p[min(col + i, n - 1)];
  }
}
// Writes a wave's 16 XT tokens x 16 TILES columns: value(i, j, v) gives the lane's four columns of column tile i and token
// tile j.  A row of the patch is one token's columns in 16-byte chunks at chunk ^ (row mod chunks per row).
template <typename T, int TILES, int XT, typename V>
__device__ __forceinline__ void store_tiles(const Int8Args& a, uint8_t* patch, int64_t row0, int rows, int wcol, V value) {
  constexpr int kChunks = TILES * T::kBytes;           // 16-byte chunks per row
  constexpr int kPer = 16 / T::kBytes;                 // columns per chunk
  const int lane = threadIdx.x & 63, fr = lane & 15, fq = lane >> 4;
#pragma unroll
  for (int j = 0; j < XT; ++j) {
    if (16 * j >= rows) break;                         // wave-uniform
    uint8_t* buf = patch + (j & 1) * 4096;             // two patches: the next tile is written while this one leaves
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      float v[4];
      value(i, j, v);
      uint8_t* row = buf + fr * kChunks * 16;
      if constexpr (T::kBytes == 4) {
        const u32x4 w = {__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
        *reinterpret_cast<u32x4*>(row + ((4 * i + fq) ^ (fr & (kChunks - 1))) * 16) = w;
      } else {
        const float w[8] = {v[0], v[1], v[2], v[3], 0.0f, 0.0f, 0.0f, 0.0f};
        const u32x4 packed = pack16<T>(w);
        *reinterpret_cast<uint2*>(row + ((2 * i + (fq >> 1)) ^ (fr & (kChunks - 1))) * 16 + (fq & 1) * 8) =
            make_uint2(packed[0], packed[1]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int t = 0; t < kChunks / 4; ++t) {
      const int idx = t * 64 + lane, row = idx / kChunks, c = idx % kChunks;
      const u32x4 v = *reinterpret_cast<const u32x4*>(buf + row * kChunks * 16 + (c ^ (row & (kChunks - 1))) * 16);
      const int left = a.n - (wcol + c * kPer);
      if (16 * j + row < rows && left > 0) {
        uint8_t* dst = a.out + ((row0 + 16 * j + row) * a.ldo + wcol + c * kPer) * T::kBytes;
        if (left >= kPer) {
          store16(dst, v);
        } else {
          for (int u = 0; u < left; ++u) {
            if constexpr (T::kBytes == 4) reinterpret_cast<uint32_t*>(dst)[u] = v[u];
            else reinterpret_cast<uint16_t*>(dst)[u] = (uint16_t)(v[u >> 1] >> (16 * (u & 1)));
          }
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

template <bool FUSED, typename TL>
__global__ __launch_bounds__(TL::kThreads) void int8_tiled_kernel(Int8Args a, int groups, int min_rows) {
  constexpr int kTM = TL::M, kSlotBytes = TL::kSlot, XT = TL::XT, WN = TL::WN;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int s_tiles[kMaxGroups + 1];
  constexpr int kCols = FUSED ? TL::W / 2 : TL::W;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % WN, wm = wave / WN;
  const int ntn = (a.n + kCols - 1) / kCols;

  // ---- which (group, m-tile, n-tile): block b runs on XCD b % 8 and takes items of that eighth of the list ----
  int total_m;
  if (a.seqlens == nullptr) {
    total_m = (int)((a.m + kTM - 1) / kTM);
  } else {
    if (tid < 64) {                           // one wave scans the groups' tile counts
      int run = 0;
      for (int g0 = 0; g0 < groups; g0 += 64) {
        const int g = g0 + lane;
        int64_t r0;
        int c = 0;
        if (g < groups) group_rows(a, g, &r0, &c);
        const int t = c > min_rows ? (c + kTM - 1) / kTM : 0;
        int inc = t;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
          const int up = __shfl_up(inc, off, BGMOE_WAVE);
          if (lane >= off) inc += up;
        }
        if (g < groups) s_tiles[g + 1] = run + inc;
        run += __shfl(inc, 63, BGMOE_WAVE);
      }
      if (lane == 0) s_tiles[0] = 0;
    }
    __syncthreads();
    total_m = s_tiles[groups];
  }
  const int64_t total = (int64_t)total_m * ntn;
  const int64_t per_x = (total + 7) / 8;
  const int64_t idx = blockIdx.x >> 3;
  const int64_t item = (int64_t)(blockIdx.x & 7) * per_x + idx;
  if (idx >= per_x || item >= total) return;
  int grp = 0, m_tiles = total_m, first = 0;
  if (a.seqlens != nullptr) {
    int lo = 0, hi = groups - 1;              // the last group whose tiles start at or before the item
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((int64_t)s_tiles[mid] * ntn <= item) lo = mid;
      else hi = mid - 1;
    }
    grp = __builtin_amdgcn_readfirstlane(lo);
    first = __builtin_amdgcn_readfirstlane(s_tiles[grp]);
    m_tiles = __builtin_amdgcn_readfirstlane(s_tiles[grp + 1]) - first;
  }
  const int64_t rel = item - (int64_t)first * ntn;
  const int panel = (int)(rel / ((int64_t)kPanel * ntn));
  const int pm = min(kPanel, m_tiles - panel * kPanel);
  const int in_panel = (int)(rel - (int64_t)panel * kPanel * ntn);
  const int nt = in_panel / pm;
  const int m0 = (panel * kPanel + in_panel - nt * pm) * kTM, n0 = nt * kCols;
  int64_t row0;
  int cnt;
  group_rows(a, grp, &row0, &cnt);

  // ---- load sources: a wave load covers 8 rows x 128 bytes; lane = row lane / 8, LDS position lane % 8.  This wave
  // loads token rows and weight rows 32 wave .. 32 wave + 31 of the tile, four loads each ----
  const int lr = lane >> 3;
  const int lc[2] = {(lane & 7) ^ (lane >> 4), (lane & 7) ^ (4 + (lane >> 4))};      // source chunk in even and odd loads
  const uint8_t* xsrc = uniform_ptr(reinterpret_cast<const uint8_t*>(a.x) + (row0 + m0) * a.ldx);
  const bool up = FUSED && wave >= WN;
  const int8_t* wmat = up ? a.w1 + grp * a.w1_group : a.w0 + grp * a.w0_group;
  const int first_row = min(n0 + 32 * (FUSED ? wave % WN : wave), a.n - 1);
  const uint8_t* wsrc = uniform_ptr(reinterpret_cast<const uint8_t*>(wmat) + (int64_t)first_row * a.k);
  uint32_t x_off[4], w_off[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 8 * i + lr;
    x_off[i] = (uint32_t)min(32 * wave + r, cnt - 1 - m0) * (uint32_t)a.ldx + (uint32_t)(lc[i & 1] * 16);
    w_off[i] = (uint32_t)min(r, a.n - 1 - first_row) * (uint32_t)a.k + (uint32_t)(lc[i & 1] * 16);
  }
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)smem);
  const int S = max((a.k + kTK - 1) / kTK, 3);        // a short K is padded with steps of zeros
  const int chunks = a.k >> 4;
  auto issue_one = [&](int s, int i) {        // one of the eight loads of a whole step
    const uint32_t d = lds0 + (uint32_t)(s & 1) * kSlotBytes + 4096 * wave + (i & 3) * 1024;
    if (i < 4) async_load16(xsrc + s * kTK, x_off[i & 3], d);
    else async_load16(wsrc + s * kTK, w_off[i & 3], d + kTM * kTK);
  };
  auto issue = [&](int s) {
    if ((s + 1) * 8 <= chunks) {
#pragma unroll
      for (int i = 0; i < 8; ++i) issue_one(s, i);
      return;
    }
    const uint32_t d = lds0 + (uint32_t)(s & 1) * kSlotBytes + 4096 * wave;
    const int ko = s * kTK;
#pragma unroll
    for (int i = 0; i < 4; ++i) {             // the last, partial step: chunks past K read zeros
      const bool in = s * 8 + lc[i & 1] < chunks;
      async_load16_lane(in ? (const void*)(xsrc + ko + x_off[i]) : (const void*)&g_zeros, d + i * 1024);
      async_load16_lane(in ? (const void*)(wsrc + ko + w_off[i]) : (const void*)&g_zeros, d + kTM * kTK + i * 1024);
    }
  };

  // ---- operands: 16 rows x 64 bytes of K per tile; lane = row lane % 16, chunk 4 half + lane / 16 ----
  const int fr = lane & 15, fq = lane >> 4;
  int f_off[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) f_off[h] = fr * kTK + (((4 * h + fq) ^ ((fr >> 1) & 7)) * 16);
  int a_off[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) a_off[i] = kTM * kTK + 16 * kTK * (FUSED ? 2 * WN * (i >> 1) + 2 * wn + (i & 1) : 4 * wn + i);
  const int b_off = kTM / 2 * kTK * wm;
  // the weights of a half are double-buffered; a token tile's register is refilled as soon as it has been multiplied
  intx4 w0[4], w1[4], x[XT];
  auto read_w = [&](int s, int h, int i) {
    return *reinterpret_cast<const intx4*>(smem + (s & 1) * kSlotBytes + f_off[h] + a_off[i]);
  };
  auto read_x = [&](int s, int h, int j) {
    return *reinterpret_cast<const intx4*>(smem + (s & 1) * kSlotBytes + f_off[h] + b_off + 16 * kTK * j);
  };
  intx4 acc[4][XT];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < XT; ++j) acc[i][j] = intx4{0, 0, 0, 0};
  // multiplies w with x while reading half rh of step rs into wnext and x; load: requests step ls
  auto half = [&](auto load, const intx4 (&w)[4], intx4 (&wnext)[4], int rs, int rh, int ls) {
#pragma unroll
    for (int j = 0; j < XT; ++j) {
      if constexpr (decltype(load)::value)
#pragma unroll
        for (int u = 0; u < 8 / XT; ++u) issue_one(ls, j * (8 / XT) + u);
      if (j < 4) wnext[j] = read_w(rs, rh, j);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i], x[j], acc[i][j], 0, 0, 0);
      x[j] = read_x(rs, rh, j);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  issue(0);
  issue(1);
  wait_vm<8>();
  block_barrier();
  // a wave without a row of either operand inside the problem only loads and keeps the barriers
  const bool live = m0 + kTM / 2 * wm < cnt && n0 + (FUSED ? 32 : 64) * wn < a.n;
  if (!live) {
    for (int s = 0; s + 1 < S; ++s) {
      wait_vm<0>();
      block_barrier();
      if (s + 2 < S) issue(s + 2);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) w0[i] = read_w(0, 0, i);
#pragma unroll
  for (int j = 0; j < XT; ++j) x[j] = read_x(0, 0, j);
  auto next_step = [&] {                      // step s + 1 is there; everybody has read step s
    wait_vm<0>();
    lds_reads_done();
    block_barrier();
  };
  for (int s = 0; s < S - 3; ++s) {
    half(No{}, w0, w1, s, 1, 0);
    next_step();
    half(Yes{}, w1, w0, s + 1, 0, s + 2);     // step s + 2 < S - 1 is whole
  }
  // the last three steps, without a loop (one behind the other would make the compiler move accumulators around)
  half(No{}, w0, w1, S - 3, 1, 0);
  next_step();
  issue(S - 1);
  half(No{}, w1, w0, S - 2, 0, 0);
  half(No{}, w0, w1, S - 2, 1, 0);
  next_step();
  half(No{}, w1, w0, S - 1, 0, 0);
  half(No{}, w0, w1, S - 1, 1, 0);
#pragma unroll
  for (int j = 0; j < XT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w1[i], x[j], acc[i][j], 0, 0, 0);

  // ---- epilogue: a lane holds columns 4 q .. 4 q + 3 of each 16-column tile for token r of each token tile ----
  constexpr int kTiles = FUSED ? 2 : 4;       // 16-column tiles of the output
  const float* ws0 = a.ws0 + grp * a.ws0_group;
  const float* ws1 = FUSED ? a.ws1 + grp * a.ws1_group : nullptr;
  const int wcol = n0 + 16 * kTiles * wn;     // this wave's first column
  const int wrow = m0 + kTM / 2 * wm;         // and first token
  float sc[4][4], bias[kTiles][4], xs[XT];
#pragma unroll
  for (int j = 0; j < XT; ++j) xs[j] = a.xs[row0 + min(wrow + 16 * j + fr, cnt - 1)];
#pragma unroll
  for (int i = 0; i < 4; ++i) load_cols(i < kTiles ? ws0 : ws1, wcol + 16 * (i % kTiles) + 4 * fq, a.n, sc[i]);
  if (a.bias) {
#pragma unroll
    for (int i = 0; i < kTiles; ++i) load_cols(a.bias, wcol + 16 * i + 4 * fq, a.n, bias[i]);
  }
  auto value = [&](int i, int j, float (&v)[4]) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      v[u] = (float)acc[i][j][u] * xs[j] * sc[i][u];
      if constexpr (FUSED) v[u] = silu_f32(v[u]) * ((float)acc[i + 2][j][u] * xs[j] * sc[i + 2][u]);
      else if (a.bias) v[u] += bias[i][u];
    }
  };
  // Stored as they are, a wave's store would touch 16 rows with 32 bytes each: 16 tokens go through a patch of LDS and
  // leave as whole row segments.  The slot of step S - 2 is free (everybody passed the last barrier after reading it).
  uint8_t* patch = smem + (S & 1) * kSlotBytes + wave * 8192;
  if (a.out_dtype == BGMOE_DT_FP32) store_tiles<Fp32, kTiles, XT>(a, patch, row0 + wrow, cnt - wrow, wcol, value);
  else if (a.out_dtype == BGMOE_DT_BF16) store_tiles<Bf16, kTiles, XT>(a, patch, row0 + wrow, cnt - wrow, wcol, value);
  else store_tiles<Fp16, kTiles, XT>(a, patch, row0 + wrow, cnt - wrow, wcol, value);
}

// ---- split kernel: one weight matrix and few rows, the dense decode case ------------------------------------------------
// There are too few (row block, token block) pairs to fill the chip when each walks all of K, so the eight waves of a
// block take an eighth of K each for the same 16 RT weight rows and 16 MT tokens and add their integer sums through
// LDS at the end: no workspace, no second launch.  Operands go straight from global memory to the MFMA registers: lane
// (r, q) reads 32 contiguous bytes of row r per 128-byte step (K is permuted alike for both operands: the first 16
// bytes feed one MFMA, the second 16 the next), so that four lanes cover a line.
template <int RT, int MT>
__global__ __launch_bounds__(512) void int8_split_kernel(Int8Args a) {
  constexpr int kWaves = 8;
  __shared__ __align__(16) int s_sum[kWaves][MT * RT > 4 ? 4 : MT * RT][256];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16 * RT;
  const int64_t t0 = (int64_t)blockIdx.y * 16 * MT;
  const int chunks = a.k >> 4, S = (a.k + 127) / 128, whole = a.k / 128;
  const int s0 = S * wave / kWaves, s1 = S * (wave + 1) / kWaves;
  const uint8_t* wp[RT];
  const uint8_t* xp[MT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
    wp[i] = reinterpret_cast<const uint8_t*>(a.w0) + (int64_t)min(n0 + 16 * i + r, a.n - 1) * a.k + 32 * q;
#pragma unroll
  for (int j = 0; j < MT; ++j)
    xp[j] = reinterpret_cast<const uint8_t*>(a.x) + min(t0 + 16 * j + r, a.m - 1) * a.ldx + 32 * q;
  intx4 acc[RT][MT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = intx4{0, 0, 0, 0};
  auto step = [&](const intx4 (&w)[RT][2], const intx4 (&x)[MT][2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int i = 0; i < RT; ++i) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i][h], x[j][h], acc[i][j], 0, 0, 0);
  };
  constexpr int kUnroll = RT * MT >= 8 ? 2 : 4;
  int s = s0;
  for (; s + kUnroll <= min(s1, whole); s += kUnroll) {
    intx4 w[kUnroll][RT][2], x[kUnroll][MT][2];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < RT; ++i) w[u][i][h] = gload_x4(wp[i] + (s + u) * 128 + 16 * h);
#pragma unroll
        for (int j = 0; j < MT; ++j) x[u][j][h] = gload_x4(xp[j] + (s + u) * 128 + 16 * h);
      }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) step(w[u], x[u]);
  }
  for (; s < s1; ++s) {
    intx4 w[RT][2], x[MT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool in = 8 * s + 2 * q + h < chunks;
#pragma unroll
      for (int i = 0; i < RT; ++i) w[i][h] = in ? gload_x4(wp[i] + s * 128 + 16 * h) : intx4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < MT; ++j) x[j][h] = in ? gload_x4(xp[j] + s * 128 + 16 * h) : intx4{0, 0, 0, 0};
    }
    step(w, x);
  }

  // sums over the waves, up to four 16 x 16 tiles at a time; a thread then holds four columns of one token
  constexpr int kAll = RT * MT, kAtOnce = kAll > 4 ? 4 : kAll;
#pragma unroll
  for (int base = 0; base < kAll; base += kAtOnce) {
    if (base) __syncthreads();
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
      *reinterpret_cast<intx4*>(&s_sum[wave][u][lane * 4]) = acc[(base + u) / MT][(base + u) % MT];
    __syncthreads();
    const int u = threadIdx.x >> 6;
    if (u < kAtOnce) {
      intx4 sum = *reinterpret_cast<const intx4*>(&s_sum[0][u][lane * 4]);
#pragma unroll
      for (int w = 1; w < kWaves; ++w) sum += *reinterpret_cast<const intx4*>(&s_sum[w][u][lane * 4]);
      const int col = n0 + 16 * ((base + u) / MT) + 4 * q;
      const int64_t tok = t0 + 16 * ((base + u) % MT) + r;
      if (tok < a.m && col < a.n) {
        float sc[4], bias[4] = {0.0f, 0.0f, 0.0f, 0.0f}, v[4];
        load_cols(a.ws0, col, a.n, sc);
        if (a.bias) load_cols(a.bias, col, a.n, bias);
        const float xs = a.xs[tok];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = (float)sum[i] * xs * sc[i];
          if (a.bias) v[i] += bias[i];
        }
        store4(a, tok, col, v);
      }
    }
  }
}

// ---- row quantiser: one block per row, the row in registers between its maximum and its cast -----------------------------
template <typename T, int V>
__global__ __launch_bounds__(1024) void int8_quant_kernel(const uint8_t* __restrict__ x, int64_t stride, int64_t rows,
                                                          int k, int8_t* __restrict__ q, float* __restrict__ scale) {
  __shared__ float s_max[16];
  const int64_t row = linear_block();
  if (row >= rows) return;
  const uint8_t* src = x + row * stride * T::kBytes;
  const int step = blockDim.x * 8;
  float v[V > 0 ? V : 1][8];
  float amax = 0.0f;
  bool bad = false;
  auto take = [&](const float (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      amax = fmaxf(amax, fabsf(w[i]));
      bad = bad || w[i] != w[i];                        // fmaxf drops a NaN
    }
  };
  if constexpr (V > 0) {
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int c = threadIdx.x * 8 + u * step;
      load8<T>(src, c, k - c, v[u]);
    }
#pragma unroll
    for (int u = 0; u < V; ++u) take(v[u]);
  } else {                                              // a row longer than the registers hold is read twice
    for (int c = threadIdx.x * 8; c < k; c += step) {
      load8<T>(src, c, k - c, v[0]);
      take(v[0]);
    }
  }
  if (bad) amax = __builtin_huge_valf();
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off, BGMOE_WAVE));
  const int waves = blockDim.x >> 6;
  if (waves > 1) {
    if (lane_id() == 0) s_max[threadIdx.x >> 6] = amax;
    __syncthreads();
    amax = s_max[0];
    for (int w = 1; w < waves; ++w) amax = fmaxf(amax, s_max[w]);
  }
  const float sc = int8_scale(amax);
  if (threadIdx.x == 0) scale[row] = sc;
  int8_t* dst = q + row * k;
  if constexpr (V > 0) {
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int c = threadIdx.x * 8 + u * step;
      int8_store8(dst + c, k - c, v[u], sc);
    }
  } else {
    for (int c = threadIdx.x * 8; c < k; c += step) {
      load8<T>(src, c, k - c, v[0]);
      int8_store8(dst + c, k - c, v[0], sc);
    }
  }
}

template <typename T>
int run_quant(const void* x, int64_t stride, int64_t rows, int k, int8_t* q, float* scale, hipStream_t st) {
  // two vectors per thread: 8192 x 7168 bf16 in 31.5 us (5.6 TB/s), 1 x 7168 in 3.2 us; one vector (896 threads a row)
  // 68 and 4.0 us, four 31.1 and 3.8 us, eight 34.6 and 5.2 us
  const bool held = k <= 16384;
  const int threads = held ? ((k + 15) / 16 + BGMOE_WAVE - 1) / BGMOE_WAVE * BGMOE_WAVE : 1024;
  const dim3 grid = bgmoe_grid(rows), block(threads);
  BgmoeProf prof(BGMOE_K_INT8_QUANT, st);
  if (held) hipLaunchKernelGGL((int8_quant_kernel<T, 2>), grid, block, 0, st, (const uint8_t*)x, stride, rows, k, q, scale);
  else hipLaunchKernelGGL((int8_quant_kernel<T, 0>), grid, block, 0, st, (const uint8_t*)x, stride, rows, k, q, scale);
  return bgmoe_check_launch("int8_quant_rows");
}

int check_sizes(const char* what, int64_t m, int n, int k, int out_dtype) {
  BGMOE_REQUIRE(m >= 0 && m <= 0x7fffffffLL && n >= 0, "%s: bad sizes m=%lld n=%d", what, (long long)m, n);
  BGMOE_REQUIRE(k >= 16 && k <= kMaxK && k % 16 == 0, "%s: k=%d must be a multiple of 16 in [16, %d]", what, k, kMaxK);
  BGMOE_REQUIRE(out_dtype >= BGMOE_DT_BF16 && out_dtype <= BGMOE_DT_FP32, "%s: unknown output type %d", what, out_dtype);
  return BGMOE_OK;
}

// Grouped: groups of up to kStreamRows rows are streamed, larger ones tiled; each kernel skips the other's groups.  Equal
// groups, 32 experts x (gate + up of 2048) x 7168 and 64 experts x 7168 x 2048, streamed | tiled 128 x 128:
// 32 rows 167 | 168, 203 | 197 us; 40 rows 180 | 174, 212 | 200 us; 64 rows 194 | 178, 233 | 217 us (streamed through
// the last-level cache; past it the 32 rows take 158).
constexpr int kStreamRows = 32;
// The tile of the larger groups goes by the average, which is what the host knows.  128 x 128 | 256 x 256:
// 96 rows 195 | 214 us, 128 rows 206 | 220, 192 rows 292 | 250, 512 rows 594 | 458 (32 experts); 128 rows 243 | 267,
// 256 rows 385 | 309 us (64 experts).
constexpr int kSmallTileRows = 160;

template <bool FUSED, typename TL>
int64_t tiled_blocks(const Int8Args& a, int groups) {
  // a bound on the m-tiles of groups above the streaming limit, whatever the counts
  const int64_t m_tiles = a.seqlens ? a.m / TL::M + min((int64_t)groups, a.m / (kStreamRows + 1)) : (a.m + TL::M - 1) / TL::M;
  constexpr int kCols = FUSED ? TL::W / 2 : TL::W;
  return (m_tiles * ((a.n + kCols - 1) / kCols) + 7) / 8 * 8;
}
constexpr int64_t kMaxBlocks = 1 << 22;
constexpr int kMaxN = 1 << 22;

template <bool FUSED, typename TL>
int run_tiled(const char* what, const Int8Args& a, int groups, hipStream_t st) {
  const int64_t blocks = tiled_blocks<FUSED, TL>(a, groups);
  BGMOE_REQUIRE(blocks <= kMaxBlocks, "%s: m=%lld x n=%d is too large for one launch", what, (long long)a.m, a.n);
  hipLaunchKernelGGL((int8_tiled_kernel<FUSED, TL>), dim3((unsigned)blocks), dim3(TL::kThreads), TL::kRing, st, a, groups,
                     kStreamRows);
  return bgmoe_check_launch(what);
}

bool small_tiles(const Int8Args& a, int groups) { return a.m <= (int64_t)kSmallTileRows * groups; }

template <bool FUSED>
int run_stream(const char* what, const Int8Args& a, int groups, hipStream_t st) {
  constexpr int kCols = FUSED ? 32 : 64;
  const dim3 grid((unsigned)((a.n + (int64_t)kCols - 1) / kCols), (unsigned)groups);
  hipLaunchKernelGGL(int8_stream_kernel<FUSED>, grid, dim3(256), kRingBytes, st, a, kStreamRows);
  return bgmoe_check_launch(what);
}

template <bool FUSED>
int run_grouped(const char* what, const Int8Args& a, int groups, hipStream_t st) {
  // Weights that exceed the 256 MB last-level cache are streamed past it: 940 MB, 8 rows per expert, 160 -> 140 us (6.7 TB/s);
  // a stack that fits may still be there from the last call: 16 experts x 4096 x 4096 (268 MB) 44.3 against 48.9 us.
  // The whole stack is counted, which is what the host knows; a step that touches few experts reads less.
  Int8Args s = a;
  s.past_cache = (int64_t)groups * a.n * a.k * (FUSED ? 2 : 1) > (256LL << 20);
  const int rc = run_stream<FUSED>(what, s, groups, st);
  if (rc != BGMOE_OK || a.m <= kStreamRows) return rc;
  return small_tiles(a, groups) ? run_tiled<FUSED, Small>(what, a, groups, st) : run_tiled<FUSED, Large>(what, a, groups, st);
}

template <int RT, int MT>
int run_split(const char* what, const Int8Args& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.n + (int64_t)16 * RT - 1) / (16 * RT)), (unsigned)((a.m + 16 * MT - 1) / (16 * MT)));
  hipLaunchKernelGGL((int8_split_kernel<RT, MT>), grid, dim3(512), 0, st, a);
  return bgmoe_check_launch(what);
}

// Dense: the form with the smallest estimated time.  The estimates (microseconds) are fits to graph-timed runs over
// n x k = 4096 x 7168, 7168 x 2048, 1024 x 1024, 512 x 512 and 36864 x 7168, m = 1 .. 4096:
//   split RT x MT   a launch, a tile's share of the reduction, and the bytes its blocks request at 37 GB/s per CU
//   stream          a stage costs 0.33 (16 tokens) or 0.66 (32) while two blocks share a CU; the weights at 5.9 TB/s
//   tiled 128       0.63 per step until about 300 tiles are at work, then 0.0021 per tile
//   tiled 256       1.15 per step, 1.65 when every CU has a tile
// Measured against one another at 4096 x 7168: m = 1 split 6.5, stream 11.9; m = 64 split 15.2, tiled 128 38; m = 256
// split 30.0, tiled 128 39.9; m = 512 split 57, tiled 128 40.5, tiled 256 67.8; m = 2048 tiled 128 66.0, tiled 256 72.0;
// m = 4096 tiled 128 126, tiled 256 94 us.  At 36864 x 7168, m = 16: stream 44.2, split 52.3 us.
int run_dense(const char* what, const Int8Args& a, hipStream_t st) {
  const double n = a.n, k = a.k, m = (double)a.m, steps = (a.k + kTK - 1) / kTK;
  auto ceil_div = [](int64_t x, int64_t y) { return (double)((x + y - 1) / y); };
  auto split = [&](int rt, int mt) {
    const double blocks = ceil_div(a.n, 16 * rt) * ceil_div(a.m, 16 * mt), rounds = blocks > 256 ? blocks / 256 : 1;
    const double rows = 16 * rt + (m < 16 * mt ? m : 16 * mt), asked = rounds * rows * k / 37e3, hbm = n * k / 4.9e6;
    return 2.6 + 0.11 * rt * mt + (asked > hbm ? asked : hbm);
  };
  const double tiles_s = ceil_div(a.n, 128) * ceil_div(a.m, 128), tiles_l = ceil_div(a.n, 256) * ceil_div(a.m, 256);
  const double stage = 0.33 * ceil_div(a.m, 16) * ceil_div(a.k, kStageK) * ceil_div((int64_t)ceil_div(a.n, 64), 512);
  const double weights = n * k / 5.9e6;
  double best = 6.0 + steps * (tiles_l > 128 ? 1.65 : 1.15) * ceil_div((int64_t)tiles_l, 256);
  int form = 0;
  auto consider = [&](int which, double t) {
    if (t < best) best = t, form = which;
  };
  consider(1, 4.3 + steps * (tiles_s < 300 ? 0.63 : 0.0021 * tiles_s));
  if (a.m <= kStreamRows) consider(2, 3.0 + (stage > weights ? stage : weights));
  if (a.m <= 65535 * 16) {
    consider(11, split(1, 1));
    consider(22, split(2, 2));
    consider(24, split(2, 4));
    consider(44, split(4, 4));
  }
  switch (form) {
    case 11: return run_split<1, 1>(what, a, st);
    case 22: return run_split<2, 2>(what, a, st);
    case 24: return run_split<2, 4>(what, a, st);
    case 44: return run_split<4, 4>(what, a, st);
    case 2: return run_stream<false>(what, a, 1, st);
    case 1: return run_tiled<false, Small>(what, a, 1, st);
    default: return run_tiled<false, Large>(what, a, 1, st);
  }
}

int run_gemm(const char* what, const Int8Args& a, int groups, hipStream_t st) {
  BGMOE_REQUIRE(a.n <= kMaxN, "%s: n=%d is too wide", what, a.n);
  BgmoeProf prof(BGMOE_K_INT8_GEMM, st);
  if (a.seqlens == nullptr) return run_dense(what, a, st);
  return a.w1 ? run_grouped<true>(what, a, groups, st) : run_grouped<false>(what, a, groups, st);
}

}  // namespace

int bgmoe_internal_init_int8_gemm() {
  const struct { const void* fn; int bytes; } fns[] = {{(const void*)int8_stream_kernel<false>, kRingBytes},
                                                       {(const void*)int8_stream_kernel<true>, kRingBytes},
                                                       {(const void*)int8_tiled_kernel<false, Large>, Large::kRing},
                                                       {(const void*)int8_tiled_kernel<true, Large>, Large::kRing},
                                                       {(const void*)int8_tiled_kernel<false, Small>, Small::kRing},
                                                       {(const void*)int8_tiled_kernel<true, Small>, Small::kRing}};
  for (const auto& f : fns) {
    const hipError_t err = hipFuncSetAttribute(f.fn, hipFuncAttributeMaxDynamicSharedMemorySize, f.bytes);
    if (err != hipSuccess) {
      bgmoe_set_error("int8 product: hipFuncSetAttribute(dynamic LDS) failed: %s", hipGetErrorString(err));
      return BGMOE_ERR_HIP;
    }
  }
  return BGMOE_OK;
}

// the dynamic-LDS opt-in holds per device: done once for each before its first launch
static int ensure_init() {
  static bool done[64] = {};
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) {
    bgmoe_set_error("int8 product: no current HIP device (or device index >= 64)");
    return BGMOE_ERR_HIP;
  }
  if (!done[dev]) {
    const int rc = bgmoe_internal_init_int8_gemm();
    if (rc != BGMOE_OK) return rc;
    done[dev] = true;
  }
  return BGMOE_OK;
}

extern "C" int bgmoe_int8_quant_rows(const void* x, int dtype, int64_t x_row_stride, int64_t rows, int k, int8_t* q,
                                     float* scale, bgmoe_stream_t stream) {
  BGMOE_REQUIRE(dtype >= BGMOE_DT_BF16 && dtype <= BGMOE_DT_FP32, "int8_quant_rows: unknown element type %d", dtype);
  BGMOE_REQUIRE(rows >= 0 && rows <= 0x7fffffffLL && k >= 0, "int8_quant_rows: bad sizes rows=%lld k=%d", (long long)rows, k);
  if (rows == 0) return BGMOE_OK;
  BGMOE_REQUIRE(k >= 1 && x && q && scale, "int8_quant_rows: null pointer or empty rows");
#define BGMOE_CALL(T) run_quant<T>(x, x_row_stride, rows, k, q, scale, bgmoe_stream(stream))
  BGMOE_BY_TYPE(dtype, BGMOE_CALL);
#undef BGMOE_CALL
}

extern "C" int bgmoe_int8_gemm(const int8_t* x, int64_t x_row_stride, const float* x_scale, const int8_t* w,
                               const float* w_scale, const float* bias, int64_t m, int n, int k, void* out, int out_dtype,
                               int64_t out_row_stride, bgmoe_stream_t stream) {
  int rc = check_sizes("int8_gemm", m, n, k, out_dtype);
  if (rc != BGMOE_OK) return rc;
  if (m == 0 || n == 0) return BGMOE_OK;
  BGMOE_REQUIRE(x && x_scale && w && w_scale && out, "int8_gemm: null pointer");
  BGMOE_REQUIRE(((uintptr_t)x | (uintptr_t)w | (uintptr_t)x_row_stride) % 16 == 0,
                "int8_gemm: x, w and x_row_stride must be multiples of 16 bytes");
  BGMOE_REQUIRE(x_row_stride >= k && x_row_stride < (1LL << 24), "int8_gemm: x_row_stride %lld outside [k, 2^24)",
                (long long)x_row_stride);
  BGMOE_REQUIRE(out_row_stride >= n, "int8_gemm: out_row_stride %lld is smaller than n=%d", (long long)out_row_stride, n);
  rc = ensure_init();
  if (rc != BGMOE_OK) return rc;
  Int8Args a{};
  a.x = x; a.ldx = x_row_stride; a.xs = x_scale; a.w0 = w; a.ws0 = w_scale; a.bias = bias; a.m = m; a.n = n; a.k = k;
  a.out = (uint8_t*)out; a.ldo = out_row_stride; a.out_dtype = out_dtype;
  return run_gemm("int8_gemm", a, 1, bgmoe_stream(stream));
}

static size_t linear_rows_bytes(int64_t m, int k) { return ((size_t)m * (size_t)k + 15) / 16 * 16; }
static size_t linear_scale_bytes(int64_t m) { return ((size_t)m * 4 + 15) / 16 * 16; }

extern "C" size_t bgmoe_int8_linear_workspace_bytes(int64_t m, int n, int k) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  return linear_rows_bytes(m, k) + linear_scale_bytes(m);
}

extern "C" int bgmoe_int8_linear(const void* x, int x_dtype, int64_t x_row_stride, const int8_t* w, const float* w_scale,
                                 const float* bias, int64_t m, int n, int k, void* out, int out_dtype,
                                 int64_t out_row_stride, void* workspace, size_t workspace_bytes, bgmoe_stream_t stream) {
  int rc = check_sizes("int8_linear", m, n, k, out_dtype);
  if (rc != BGMOE_OK) return rc;
  if (m == 0 || n == 0) return BGMOE_OK;
  BGMOE_REQUIRE(x && w && w_scale && out, "int8_linear: null pointer");
  const size_t need = bgmoe_int8_linear_workspace_bytes(m, n, k);
  if (workspace == nullptr || workspace_bytes < need) {
    bgmoe_set_error("int8_linear: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    return BGMOE_ERR_WORKSPACE;
  }
  BGMOE_REQUIRE((uintptr_t)workspace % 16 == 0, "int8_linear: workspace must be 16-byte aligned");
  uint8_t* ws = (uint8_t*)workspace;
  int8_t* q = (int8_t*)ws;
  float* qs = (float*)(ws + linear_rows_bytes(m, k));
  rc = bgmoe_int8_quant_rows(x, x_dtype, x_row_stride, m, k, q, qs, stream);
  if (rc != BGMOE_OK) return rc;
  return bgmoe_int8_gemm(q, k, qs, w, w_scale, bias, m, n, k, out, out_dtype, out_row_stride,
                         stream);
}

static int grouped(const char* what, Int8Args& a, int groups, int out_dtype, bgmoe_stream_t stream) {
  int rc = check_sizes(what, a.m, a.n, a.k, out_dtype);
  if (rc != BGMOE_OK) return rc;
  BGMOE_REQUIRE(groups >= 1 && groups <= kMaxGroups, "%s: %d groups outside [1, %d]", what, groups, kMaxGroups);
  if (a.m == 0 || a.n == 0) return BGMOE_OK;
  BGMOE_REQUIRE(a.x && a.xs && a.w0 && a.ws0 && a.seqlens && a.cu && a.out, "%s: null pointer", what);
  BGMOE_REQUIRE(((uintptr_t)a.x | (uintptr_t)a.w0 | (uintptr_t)a.w0_group | (uintptr_t)a.w1 | (uintptr_t)a.w1_group) % 16 == 0,
                "%s: x, weights and their group strides must be multiples of 16 bytes", what);
  a.ldx = a.k; a.ldo = a.n; a.out_dtype = out_dtype;
  // before the first of the two launches, so that a refused call has written nothing
  const bool small = small_tiles(a, groups);
  const int64_t blocks = a.w1 ? (small ? tiled_blocks<true, Small>(a, groups) : tiled_blocks<true, Large>(a, groups))
                              : (small ? tiled_blocks<false, Small>(a, groups) : tiled_blocks<false, Large>(a, groups));
  BGMOE_REQUIRE(a.n <= kMaxN && (a.m <= kStreamRows || blocks <= kMaxBlocks), "%s: m=%lld x n=%d is too large for one launch", what,
                (long long)a.m, a.n);
  rc = ensure_init();
  if (rc != BGMOE_OK) return rc;
  return run_gemm(what, a, groups, bgmoe_stream(stream));
}

extern "C" int bgmoe_int8_grouped_gemm(const int8_t* x, const float* x_scale, const int8_t* w, int64_t w_group_stride,
                                       const float* w_scale, int64_t w_scale_group_stride, const int32_t* seqlens,
                                       const int32_t* cu_seqlens, int groups, int64_t m, int n, int k, void* out,
                                       int out_dtype, bgmoe_stream_t stream) {
  Int8Args a{};
  a.x = x; a.xs = x_scale; a.w0 = w; a.w0_group = w_group_stride; a.ws0 = w_scale; a.ws0_group = w_scale_group_stride;
  a.seqlens = seqlens; a.cu = cu_seqlens; a.m = m; a.n = n; a.k = k; a.out = (uint8_t*)out;
  return grouped("int8_grouped_gemm", a, groups, out_dtype, stream);
}

extern "C" int bgmoe_int8_fused_s1(const int8_t* x, const float* x_scale, const int8_t* gate, int64_t gate_group_stride,
                                   const float* gate_scale, int64_t gate_scale_group_stride, const int8_t* up,
                                   int64_t up_group_stride, const float* up_scale, int64_t up_scale_group_stride,
                                   const int32_t* seqlens, const int32_t* cu_seqlens, int groups, int64_t m, int n, int k,
                                   void* out, int out_dtype, bgmoe_stream_t stream) {
  BGMOE_REQUIRE(m == 0 || n == 0 || (up && up_scale), "int8_fused_s1: null pointer");
  Int8Args a{};
  a.x = x; a.xs = x_scale; a.w0 = gate; a.w0_group = gate_group_stride; a.ws0 = gate_scale; a.ws0_group = gate_scale_group_stride;
  a.w1 = up; a.w1_group = up_group_stride; a.ws1 = up_scale; a.ws1_group = up_scale_group_stride;
  a.seqlens = seqlens; a.cu = cu_seqlens; a.m = m; a.n = n; a.k = k; a.out = (uint8_t*)out;
  return grouped("int8_fused_s1", a, groups, out_dtype, stream);
}
