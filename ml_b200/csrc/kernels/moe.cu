// The experts of a mixture: tokens sorted by expert, the experts' products on the tensor cores, the weighted sum of what they give.
//
//   out_n = sum_j w_nj Wd[e] (silu(g) * u),   [g | u] = Wgu[e] x_n,   e = idx_nj (negative: nothing)
//
// A copy of a token is a pair (token n, place j), numbered n k + j.  The plan puts the copies in rows by expert, each expert's rows beginning at a multiple of 32 and
// filled up with empty rows, so that a product's tile and the reductions over tokens end where an expert does:
//   forward    xs = rows of x;  [g | u] = xs Wgu^T, h = silu(g) u (one product, h formed from its accumulators);  y = h Wd^T;  out = weighted sums of y
//   backward   ys = rows of dout;  dh = ys Wd;  dw = h . dh, dgu from w dh, hw = w h;  dxs = dgu Wgu, dx = sums of it;  dWgu = dgu^T xs;  dWd = ys^T hw
// Counts are known on the device only: grids are sized by what there may be at most, and blocks that find nothing leave.
#include "../tc.cuh"
#include "moe_route.cuh"

namespace {

MLB_DEFINE_ERROR_WORD(moe)

constexpr int PAD = 32;            // an expert's rows begin at a multiple of this
constexpr int TILE_TOKENS = 256;   // rows of a tile of the token products

// ------------------------------------------------------------------ the plan
// int32: start[E + 1], count[E], ntiles | tiles[maxT] {expert, first row, rows, 0} | place[N k] | source[R] | hist[blocks][E]
struct PlanShape {
  long rows, tiles, place, source, hist, total;      // R; offsets of the parts in ints
  int max_tiles, blocks, per_block;
};
constexpr int PLAN_THREADS = 256, PLAN_WARPS = PLAN_THREADS / 32;
inline PlanShape plan_shape(long NK, int E) {
  PlanShape p;
  const long used = NK < E ? NK : E;
  p.rows = (NK + (PAD - 1) * used) / PAD * PAD;
  p.max_tiles = (int)(NK / TILE_TOKENS + used);
  p.per_block = NK <= 4096 ? 4096 : (int)std::max(1024L, ((NK + 127) / 128 + PLAN_THREADS - 1) / PLAN_THREADS * PLAN_THREADS);
  p.blocks = (int)((NK + p.per_block - 1) / p.per_block);
  p.tiles = (2L * E + 2 + 3) / 4 * 4;
  p.place = p.tiles + 4L * p.max_tiles;
  p.source = p.place + NK;
  p.hist = p.source + p.rows;
  p.total = p.hist + (p.blocks > 1 ? (long)p.blocks * E : 0);
  return p;
}
struct PlanArgs {
  int *start, *count, *ntiles;
  int4* tiles;
  int *place, *source, *hist;
  const int* idx;
  long NK;
  int E, blocks, per_block;
};

__device__ __forceinline__ int expert_of(const PlanArgs& A, long i) {
  if (i >= A.NK) return -1;
  const int e = A.idx[i];
  if (e >= A.E) {
    mlb_set_error(MLB_ERR_BOUNDS, 0xD1);
    return -1;
  }
  return e;
}
__global__ void __launch_bounds__(PLAN_THREADS) moe_hist_k(const PlanArgs A) {
  mlb_pdl_sync();
  extern __shared__ int cnt[];
  for (int e = threadIdx.x; e < A.E; e += PLAN_THREADS) cnt[e] = 0;
  __syncthreads();
  const long i0 = (long)blockIdx.x * A.per_block;
  for (int i = threadIdx.x; i < A.per_block; i += PLAN_THREADS) {
    const int e = expert_of(A, i0 + i);
    if (e >= 0) atomicAdd(&cnt[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < A.E; e += PLAN_THREADS) A.hist[(long)blockIdx.x * A.E + e] = cnt[e];
}
// Every block adds up all blocks' counts for itself and puts its copies behind those of the blocks before it, in order: the same rows on every run.
__global__ void __launch_bounds__(PLAN_THREADS) moe_place_k(const PlanArgs A) {
  mlb_pdl_sync();
  extern __shared__ int sm[];
  const int E = A.E, tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  int *total = sm, *base = sm + E, *mine = sm + 2 * E;      // mine[PLAN_WARPS][E]
  __shared__ int2 warps[PLAN_WARPS];
  for (int e = tid; e < (2 + PLAN_WARPS) * E; e += PLAN_THREADS) sm[e] = 0;
  __syncthreads();
  // the copies of this block, a run of them to each warp
  const int run = A.per_block / PLAN_WARPS;
  const long i0 = (long)blockIdx.x * A.per_block + (long)w * run;
  for (int i = lane; i < run; i += 32) {
    const int e = expert_of(A, i0 + i);
    if (e >= 0) atomicAdd(&mine[w * E + e], 1);
  }
  if (A.blocks > 1) {
    if (E >= PLAN_THREADS / 2) {
      for (int e = tid; e < E; e += PLAN_THREADS) {
        int all = 0, before = 0;
#pragma unroll 8
        for (int b = 0; b < A.blocks; b++) {
          const int v = A.hist[(long)b * E + e];
          all += v;
          before += b < (int)blockIdx.x ? v : 0;
        }
        total[e] = all, base[e] = before;
      }
    } else {
      const int n = A.blocks * E;
#pragma unroll 4
      for (int i = tid; i < n; i += PLAN_THREADS) {
        const int v = A.hist[i], b = i / E, e = i - b * E;
        if (v) {
          atomicAdd(&total[e], v);
          if (b < (int)blockIdx.x) atomicAdd(&base[e], v);
        }
      }
    }
  }
  __syncthreads();
  if (A.blocks == 1) {
    for (int e = tid; e < E; e += PLAN_THREADS) {
      int all = 0;
      for (int k = 0; k < PLAN_WARPS; k++) all += mine[k * E + e];
      total[e] = all;
    }
    __syncthreads();
  }
  // rows and tiles of the experts before each (a thread has `per` experts, one behind the other)
  const int per = (E + PLAN_THREADS - 1) / PLAN_THREADS, e0 = tid * per, e1 = min(e0 + per, E);
  int2 own = make_int2(0, 0);
  for (int e = e0; e < e1; e++) {
    own.x += (total[e] + PAD - 1) / PAD * PAD;
    own.y += (total[e] + TILE_TOKENS - 1) / TILE_TOKENS;
  }
  int2 sum = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, sum.x, o), b = __shfl_up_sync(0xffffffffu, sum.y, o);
    if (lane >= o) sum.x += a, sum.y += b;
  }
  if (lane == 31) warps[w] = sum;
  __syncthreads();
  for (int k = 0; k < w; k++) sum.x += warps[k].x, sum.y += warps[k].y;
  int row = sum.x - own.x, tile = sum.y - own.y;
  const bool writes = blockIdx.x == 0;
  for (int e = e0; e < e1; e++) {
    const int n = total[e], padded = (n + PAD - 1) / PAD * PAD;
    if (writes) {
      A.start[e] = row, A.count[e] = n;
      for (int t = 0; t < n; t += TILE_TOKENS) A.tiles[tile++] = make_int4(e, row + t, min(TILE_TOKENS, n - t), 0);
      for (int t = n; t < padded; t++) A.source[row + t] = -1;
    }
    int at = row + base[e];
    for (int k = 0; k < PLAN_WARPS; k++) {
      const int v = mine[k * E + e];
      mine[k * E + e] = at;
      at += v;
    }
    row += padded;
  }
  if (writes && tid == PLAN_THREADS - 1) A.start[E] = sum.x, *A.ntiles = sum.y;
  __syncthreads();
  for (int i = lane; i < run; i += 32) {      // (run is a multiple of 32)
    const int e = expert_of(A, i0 + i);
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int first = e >= 0 ? mine[w * E + e] : 0;
    __syncwarp();
    const int rank = __popc(same & ((1u << lane) - 1));
    if (e >= 0) {
      if (rank == 0) mine[w * E + e] = first + __popc(same);
      A.place[i0 + i] = first + rank;
      A.source[first + rank] = (int)(i0 + i);
    } else if (i0 + i < A.NK) {
      A.place[i0 + i] = -1;
    }
    __syncwarp();
  }
}

// ------------------------------------------------------------------ tokens to rows, rows to tokens
// out[r] = x[source[r] / k], empty rows 0; a warp to a row, 16 bytes a lane
__global__ void __launch_bounds__(256) moe_dispatch_k(bf16* __restrict__ out, const bf16* __restrict__ x, const int* __restrict__ source, const int* __restrict__ rows, long ldx, int k,
                                                      int C) {
  mlb_pdl_sync();
  const long r = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (r >= *rows) return;
  const int lane = threadIdx.x & 31, s = source[r];
  uint4* o = reinterpret_cast<uint4*>(out + r * C);
  if (s < 0) {
    for (int c = lane; c < C / 8; c += 32) o[c] = make_uint4(0, 0, 0, 0);
    return;
  }
  const uint4* in = reinterpret_cast<const uint4*>(x + (long)(s / k) * ldx);
#pragma unroll 4
  for (int c = lane; c < C / 8; c += 32) o[c] = __ldg(in + c);
}

template <typename T> __device__ __forceinline__ float as_float(T v) { return (float)v; }
template <> __device__ __forceinline__ float as_float<bf16>(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void add8(float (&s)[8], const uint4& v, float w) {
  const uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    s[2 * i] = fmaf(__uint_as_float(q[i] << 16), w, s[2 * i]);
    s[2 * i + 1] = fmaf(__uint_as_float(q[i] & 0xffff0000u), w, s[2 * i + 1]);
  }
}
// out[n] = sum_j w[n, j] y[place[n, j]] in the order of j, in fp32; without weights plain sums
template <typename W>
__global__ void __launch_bounds__(256) moe_combine_k(bf16* __restrict__ out, const bf16* __restrict__ y, const W* __restrict__ weights, const int* __restrict__ place, long N, int k, int C) {
  mlb_pdl_sync();
  const int vec = C / 8;
  const long at = (long)blockIdx.x * 256 + threadIdx.x;
  if (at >= N * vec) return;
  const long n = at / vec;
  const int c = (int)(at - n * vec);
  float s[8] = {};
#pragma unroll 4
  for (int j = 0; j < k; j++) {
    const int r = place[n * k + j];
    if (r >= 0) add8(s, __ldg(reinterpret_cast<const uint4*>(y + (long)r * C) + c), weights ? as_float(weights[n * k + j]) : 1.f);
  }
  reinterpret_cast<uint4*>(out + n * C)[c] = make_uint4(pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3]), pack_bf16(s[4], s[5]), pack_bf16(s[6], s[7]));
}

// ------------------------------------------------------------------ SwiGLU backward with the weight of a row
// gu and dgu have groups of 16 gate columns and their 16 up columns side by side.  Of a row with weight w and d = dh: s = sigmoid(g), h = g s u;
//   dw = sum h d,  dg = w d u s (1 + g (1 - s)),  du = w d g s,  hw = w h.  Empty rows are written as zeros: the products over rows add them up.
// A row to 128 threads, 8 columns of h a thread: bound by memory (12 bytes a column of h).
template <typename W>
__global__ void __launch_bounds__(128) moe_swiglu_bwd_k(bf16* __restrict__ dgu, bf16* __restrict__ hw, W* __restrict__ dweights, const bf16* __restrict__ dh, const bf16* __restrict__ gu,
                                                        const W* __restrict__ weights, const int* __restrict__ source, const int* __restrict__ rows, int I) {
  mlb_pdl_sync();
  __shared__ float red[32];
  const long r = blockIdx.x;
  if (r >= *rows) return;
  const int s = source[r];
  const float w = s < 0 ? 0.f : as_float(weights[s]);
  float dot = 0.f;
  for (int c = threadIdx.x * 8; c < I; c += 128 * 8) {
    const long at = r * 2 * I + (c >> 4) * 32 + (c & 8);
    uint4 dg4 = make_uint4(0, 0, 0, 0), du4 = dg4, hw4 = dg4;
    if (s >= 0) {
      const uint4 g4 = __ldg(reinterpret_cast<const uint4*>(gu + at)), u4 = __ldg(reinterpret_cast<const uint4*>(gu + at + 16)), d4 = __ldg(reinterpret_cast<const uint4*>(dh + r * I + c));
      const uint32_t gq[4] = {g4.x, g4.y, g4.z, g4.w}, uq[4] = {u4.x, u4.y, u4.z, u4.w}, dq[4] = {d4.x, d4.y, d4.z, d4.w};
      uint32_t a[4], b[4], h4[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float dg[2], du[2], hh[2];
#pragma unroll
        for (int x = 0; x < 2; x++) {
          const float g = __uint_as_float(x ? gq[i] & 0xffff0000u : gq[i] << 16), u = __uint_as_float(x ? uq[i] & 0xffff0000u : uq[i] << 16);
          const float d = __uint_as_float(x ? dq[i] & 0xffff0000u : dq[i] << 16);
          const float sg = 1.f / (1.f + __expf(-g)), silu = g * sg, h = silu * u;
          dot = fmaf(h, d, dot);
          const float wd = w * d;
          dg[x] = wd * u * (sg + silu * (1.f - sg));
          du[x] = wd * silu;
          hh[x] = w * h;
        }
        a[i] = pack_bf16(dg[0], dg[1]), b[i] = pack_bf16(du[0], du[1]), h4[i] = pack_bf16(hh[0], hh[1]);
      }
      dg4 = make_uint4(a[0], a[1], a[2], a[3]), du4 = make_uint4(b[0], b[1], b[2], b[3]), hw4 = make_uint4(h4[0], h4[1], h4[2], h4[3]);
    }
    *reinterpret_cast<uint4*>(dgu + at) = dg4;
    *reinterpret_cast<uint4*>(dgu + at + 16) = du4;
    *reinterpret_cast<uint4*>(hw + r * I + c) = hw4;
  }
  dot = block_sum(dot, red);
  if (threadIdx.x == 0 && s >= 0) dweights[s] = (W)dot;
}
// the gradient of the weight of a copy that goes nowhere
template <typename W>
__global__ void __launch_bounds__(256) moe_no_place_k(W* __restrict__ dweights, const int* __restrict__ place, long NK) {
  mlb_pdl_sync();
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i < NK && place[i] < 0) dweights[i] = (W)0.f;
}

// ------------------------------------------------------------------ products
// CTA pairs share a tile of 256 features x up to 256 tokens (token products) or 256 x 256 features (weight gradients): the leader issues tcgen05.mma.cta_group::2,
// each CTA stages its 128 rows of A and its half of B and drains its own 128 tensor-memory lanes.  The weights are A and the tokens B, whose number
// an instruction takes in steps of 32: an expert's last tile, and that of an expert with few tokens, is no wider than its rows.  Two accumulators, so that a tile's
// epilogue runs under the next one's products.
enum { GATE_UP, DOWN, DOWN_T, GATE_UP_T, D_GATE_UP, D_DOWN };
constexpr int BK = 64, THREADS = 64 + 8 * 32;
struct Smem {
  static constexpr int A_BYTES = 128 * BK * 2, STAGE_BYTES = 2 * A_BYTES, STAGES = 6, STAGING_BYTES = 8 * 4096;
  static constexpr int TOTAL = STAGES * STAGE_BYTES + STAGING_BYTES + 256 + 1024;
};
struct GemmArgs {
  const int* start;      // [E + 1] rows
  const int4* tiles;
  const int* ntiles;
  bf16 *out, *h;         // token products: [R, M]; h [R, M / 2] of GATE_UP, whose out may be null.  Weight gradients: [E, M, N]
  int E, M, N, K;        // weight gradients: M x N each; token products: M features over K
  int tiles_m, tiles_n;
};
// A tile of the token products, or of one expert's weight gradient
struct Item { int e, row0, rows, mt, nt; };
template <int MODE>
struct Items {      // items cid, cid + ncl, ... ; what the next one is read from memory is asked for ahead
  static constexpr bool DW = MODE == D_GATE_UP || MODE == D_DOWN;
  const GemmArgs& g;
  int i, step, n;
  int4 ahead;
  __device__ __forceinline__ Items(const GemmArgs& g_, int cid, int ncl) : g(g_), i(cid), step(ncl) {
    n = DW ? g.E * g.tiles_m * g.tiles_n : *g.ntiles * g.tiles_m;
    fetch();
  }
  __device__ __forceinline__ void fetch() {
    if (i >= n) return;
    if (DW) {
      const int e = i / (g.tiles_m * g.tiles_n);
      ahead.x = e, ahead.y = g.start[e], ahead.z = g.start[e + 1];
    } else {
      ahead = g.tiles[i / g.tiles_m];
    }
  }
  __device__ __forceinline__ bool next(Item& w) {
    if (i >= n) return false;
    w.e = ahead.x, w.row0 = ahead.y;
    if (DW) {
      const int x = i - w.e * g.tiles_m * g.tiles_n;
      w.rows = ahead.z - ahead.y;
      w.mt = x / g.tiles_n, w.nt = x - w.mt * g.tiles_n;
    } else {
      w.rows = ahead.z;
      w.mt = i % g.tiles_m, w.nt = 0;
    }
    i += step;
    fetch();
    return true;
  }
};
__device__ __forceinline__ float swiglu(float g, float u) { return g / (1.f + __expf(-g)) * u; }

template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
moe_gemm_k(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const GemmArgs g) {
  constexpr bool DW = MODE == D_GATE_UP || MODE == D_DOWN, A_MN = MODE != GATE_UP && MODE != DOWN, B_MN = DW;
  using S = Smem;
  constexpr int STAGES = S::STAGES, ACC = 256;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* staging = smem + STAGES * S::STAGE_BYTES;
  uint64_t* full = (uint64_t*)(staging + S::STAGING_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = (uint32_t*)(acc_empty + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = tc::cluster_ctarank();
  const int cid = (int)tc::cluster_id_x(), ncl = (int)tc::cluster_count_x();

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; i++) { tc::mbar_init(&full[i], 1); tc::mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; i++) { tc::mbar_init(&acc_full[i], 1); tc::mbar_init(&acc_empty[i], 16); }
    tc::mbar_fence_init();
    tc::tma_prefetch_desc(&tmA);
    tc::tma_prefetch_desc(&tmB);
  }
  if (warp == 1) tc::tmem_alloc_pair(tmem_slot, 2 * ACC);
  tc::tc_fence_before();
  tc::cluster_sync();
  tc::tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  mlb_pdl_sync();

  if (warp == 0) {
    // ---------------------------------------------------------------- loads (one thread per CTA)
    if (tc::elect_one()) {
      int stage = 0, phase = 0;
      bool ok = true;
      Items<MODE> items(g, cid, ncl);
      Item w;
      while (ok && items.next(w)) {
        const int m0 = w.mt * 256 + (int)rank * 128;
        const int kbs = DW ? (w.rows + BK - 1) / BK : (g.K + BK - 1) / BK;
        const int half = ((w.rows + 31) & ~31) >> 1;      // token products: this CTA's tokens
        for (int kb = 0; kb < kbs; kb++) {
          if (!tc::mbar_wait(&empty[stage], phase ^ 1, 0x71)) { ok = false; break; }
          uint8_t* sA = smem + stage * S::STAGE_BYTES;
          uint8_t* sB = sA + S::A_BYTES;
          const uint32_t bar = tc::mapa_u32(tc::smem_u32(&full[stage]), 0);
          if (rank == 0) tc::mbar_expect_tx(&full[stage], 2 * S::STAGE_BYTES);
          if (MODE == GATE_UP) {      // rows in groups of 16 gate rows and the matching 16 up rows
            tc::tma_load_5d_pair(sA, &tmA, bar, kb * BK, 0, 0, m0 / 32, w.e);
          } else if (MODE == DOWN) {
            tc::tma_load_3d_pair(sA, &tmA, bar, kb * BK, m0, w.e);
          } else if (MODE == DOWN_T) {
            for (int c = 0; c < 2; c++) tc::tma_load_3d_pair(sA + c * 8192, &tmA, bar, m0 + c * 64, kb * BK, w.e);
          } else if (MODE == GATE_UP_T) {      // (K in the same groups)
            for (int c = 0; c < 2; c++) tc::tma_load_5d_pair(sA + c * 8192, &tmA, bar, m0 + c * 64, 0, 0, kb * 2, w.e);
          } else {
            for (int c = 0; c < 2; c++) tc::tma_load_2d_pair(sA + c * 8192, &tmA, bar, m0 + c * 64, w.row0 + kb * BK);
          }
          if (DW) {
            const int n0 = w.nt * 256 + (int)rank * 128;
            for (int c = 0; c < 2; c++) tc::tma_load_2d_pair(sB + c * 8192, &tmB, bar, n0 + c * 64, w.row0 + kb * BK);
          } else {
            tc::tma_load_2d_pair(sB, &tmB, bar, kb * BK, w.row0 + (int)rank * half);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- products (one thread of the leader)
    if (rank == 0 && tc::elect_one()) {
      int stage = 0, phase = 0, it = 0;
      bool ok = true;
      Items<MODE> items(g, cid, ncl);
      Item w;
      while (ok && items.next(w)) {
        const int kbs = DW ? (w.rows + BK - 1) / BK : (g.K + BK - 1) / BK;
        if (kbs == 0) continue;      // an expert without tokens
        const uint32_t idesc = tc::idesc_bf16(256, DW ? 256 : (w.rows + 31) & ~31, A_MN ? 1 : 0, B_MN ? 1 : 0);
        const int acc = it & 1, acc_phase = (it >> 1) & 1;
        it++;
        if (!tc::mbar_wait(&acc_empty[acc], acc_phase ^ 1, 0x72)) { ok = false; break; }
        tc::tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * ACC;
        for (int kb = 0; kb < kbs; kb++) {
          if (!tc::mbar_wait(&full[stage], phase, 0x73)) { ok = false; break; }
          tc::tc_fence_after();
          const uint32_t sA = tc::smem_u32(smem + stage * S::STAGE_BYTES);
          const uint32_t sB = sA + S::A_BYTES;
          const int steps = DW ? min(BK, w.rows - kb * BK) / 16 : BK / 16;      // (the rows behind an expert's are another's)
#pragma unroll
          for (int k = 0; k < BK / 16; k++) {
            if (DW && k >= steps) break;
            const uint64_t da = A_MN ? tc::smem_desc_sw128(sA + k * 2048, 8192, 1024) : tc::smem_desc_sw128(sA + k * 32, 16, 1024);
            const uint64_t db = B_MN ? tc::smem_desc_sw128(sB + k * 2048, 8192, 1024) : tc::smem_desc_sw128(sB + k * 32, 16, 1024);
            tc::mma_bf16_ss_pair(d_tmem, da, db, idesc, (kb > 0 || k > 0) ? 1u : 0u);
          }
          tc::mma_commit_pair(&empty[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (ok) tc::mma_commit_pair(&acc_full[acc]);
      }
    }
  } else {
    // ---------------------------------------------------------------- epilogue (warps 2..9 of each CTA)
    const int lg = warp & 3, half = (warp - 2) >> 2;
    uint8_t* buf = staging + (warp - 2) * 4096;
    const uint32_t sbuf = tc::smem_u32(buf);
    int it = 0;
    bool ok = true;
    Items<MODE> items(g, cid, ncl);
    Item w;
    while (ok && items.next(w)) {
      const int m0 = w.mt * 256 + (int)rank * 128 + lg * 32;
      const bool some = !DW || w.rows > 0;
      const int acc = it & 1, acc_phase = (it >> 1) & 1;
      if (some) {
        it++;
        if (!__all_sync(0xffffffffu, tc::mbar_wait(&acc_full[acc], acc_phase, 0x74))) { ok = false; break; }
        tc::tc_fence_after();
      }
      const uint32_t taddr = tmem_base + ((uint32_t)(lg * 32) << 16) + acc * ACC;
      if constexpr (!DW) {
        const bool live = m0 < g.M;
        const int unit = lane & 3, tok = lane >> 2;
        for (int c = half * 32; c < w.rows; c += 64) {
          uint32_t r[2][16];
          tc::tmem_ld_frag_wait(taddr + c, r);
          if (!live) continue;      // (warp-uniform)
          uint32_t p[2][8];         // p[h][2 j + v]: tokens 8 j + 2 (lane % 4) + {0, 1} of feature 16 h + 8 v + lane / 4
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int q = 0; q < 8; q++) p[h][q] = pack_bf16(__uint_as_float(r[h][2 * q]), __uint_as_float(r[h][2 * q + 1]));
          if (MODE != GATE_UP || g.out != nullptr) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const int t = 8 * j + (lane & 7), u = lane >> 3;
              tc::stmatrix_x4_trans(sbuf + t * 64 + ((u ^ ((t >> 1) & 3)) << 4), p[0][2 * j], p[0][2 * j + 1], p[1][2 * j], p[1][2 * j + 1]);
            }
          }
          if constexpr (MODE == GATE_UP) {      // feature 8 v + lane / 4: h = 0 its gate, h = 1 its up value
            uint32_t x[8];
#pragma unroll
            for (int q = 0; q < 8; q++)
              x[q] = pack_bf16(swiglu(__uint_as_float(p[0][q] << 16), __uint_as_float(p[1][q] << 16)),
                               swiglu(__uint_as_float(p[0][q] & 0xffff0000u), __uint_as_float(p[1][q] & 0xffff0000u)));
#pragma unroll
            for (int j = 0; j < 2; j++) {
              const int t = 16 * j + 8 * (lane >> 4) + (lane & 7), u = (lane >> 3) & 1;
              tc::stmatrix_x4_trans(sbuf + 2048 + t * 32 + ((u ^ ((t >> 2) & 1)) << 4), x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
            }
          }
          __syncwarp();
          if (MODE != GATE_UP || g.out != nullptr) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const int t = 8 * i + tok;
              const uint4 v = *reinterpret_cast<const uint4*>(buf + t * 64 + ((unit ^ ((t >> 1) & 3)) << 4));
              if (c + t < w.rows && m0 + unit * 8 < g.M) *reinterpret_cast<uint4*>(g.out + (size_t)(w.row0 + c + t) * g.M + m0 + unit * 8) = v;
            }
          }
          if constexpr (MODE == GATE_UP) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const int t = 16 * i + (lane >> 1), u = lane & 1;
              const uint4 v = *reinterpret_cast<const uint4*>(buf + 2048 + t * 32 + ((u ^ ((t >> 2) & 1)) << 4));
              if (c + t < w.rows) *reinterpret_cast<uint4*>(g.h + (size_t)(w.row0 + c + t) * (g.M / 2) + m0 / 2 + u * 8) = v;
            }
          }
          __syncwarp();
        }
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive_cluster(tc::mapa_u32(tc::smem_u32(&acc_empty[acc]), 0));
      } else {
        const int n0 = w.nt * 256 + half * 128;
        bf16* out = g.out + (size_t)w.e * g.M * g.N;
#pragma unroll 1
        for (int c = 0; c < 2; c++) {
          uint32_t r[32], r2[32];
          if (some) {
            tc::tmem_ld32x2_wait(taddr + half * 128 + c * 64, r, taddr + half * 128 + c * 64 + 32, r2);
            if (c == 1) {
              tc::tc_fence_before();
              __syncwarp();
              if (lane == 0) tc::mbar_arrive_cluster(tc::mapa_u32(tc::smem_u32(&acc_empty[acc]), 0));
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; i++) r[i] = r2[i] = 0;
          }
          const int col0 = n0 + c * 64;
          if (m0 >= g.M || col0 >= g.N) continue;      // (warp-uniform)
          uint8_t* rowp = buf + lane * 128;
#pragma unroll
          for (int v = 0; v < 8; v++) {
            const uint32_t* s = v < 4 ? &r[v * 8] : &r2[(v - 4) * 8];
            uint4 pk;
            pk.x = pack_bf16(__uint_as_float(s[0]), __uint_as_float(s[1]));
            pk.y = pack_bf16(__uint_as_float(s[2]), __uint_as_float(s[3]));
            pk.z = pack_bf16(__uint_as_float(s[4]), __uint_as_float(s[5]));
            pk.w = pack_bf16(__uint_as_float(s[6]), __uint_as_float(s[7]));
            *reinterpret_cast<uint4*>(rowp + ((v ^ (lane & 7)) << 4)) = pk;
          }
          __syncwarp();
          const int ch = lane & 7, col = col0 + ch * 8;
#pragma unroll
          for (int i = 0; i < 8; i++) {
            const int row = i * 4 + (lane >> 3), m = m0 + row;
            const uint4 v = *reinterpret_cast<const uint4*>(buf + row * 128 + ((ch ^ (row & 7)) << 4));
            // the rows of dWgu come in groups of 16 gate rows and 16 up rows
            const int to = MODE == D_GATE_UP ? (m >> 5) * 16 + (m & 15) + (m & 16 ? g.M / 2 : 0) : m;
            if (m < g.M && col < g.N) *reinterpret_cast<uint4*>(out + (size_t)to * g.N + col) = v;
          }
          __syncwarp();
        }
      }
    }
  }
  tc::tc_fence_before();
  tc::cluster_sync();      // no CTA frees tensor memory or leaves while its peer may still signal or read it
  if (warp == 1) tc::tmem_dealloc_pair(tmem_base, 2 * ACC);
}

template <int MODE>
int launch_gemm(const CUtensorMap& a, const CUtensorMap& b, const GemmArgs& g, long items, cudaStream_t st) {
  auto kern = moe_gemm_k<MODE>;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = mlb_allow_smem(kern, Smem::TOTAL, done);
  if (e != cudaSuccess) return (int)e;
  static const int most = [&] {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(mlb_sm_count() & ~1);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = Smem::TOTAL;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) { cudaGetLastError(); n = mlb_sm_count() / 2; }
    return std::min(n, mlb_sm_count() / 2);
  }();
  if (items <= 0) return 0;
  return (int)mlb_launch_tmem(true, kern, dim3(2 * (unsigned)std::min<long>(items, most)), dim3(THREADS), (size_t)Smem::TOTAL, st, a, b, g);
}

bool map_tokens(CUtensorMap* m, const bf16* base, long rows, int K) {      // [rows, K], K-major
  const uint64_t d[2] = {(uint64_t)K, (uint64_t)rows}, s[1] = {2ull * K};
  const uint32_t b[2] = {64, 128};
  return mlb_make_tmap_nd(m, base, 2, d, s, b);
}
bool map_rows(CUtensorMap* m, const bf16* base, long rows, int cols) {      // the same, its columns M or N and its rows the reduction
  const uint64_t d[2] = {(uint64_t)cols, (uint64_t)rows}, s[1] = {2ull * cols};
  const uint32_t b[2] = {64, 64};
  return mlb_make_tmap_nd(m, base, 2, d, s, b);
}
bool map_down(CUtensorMap* m, const bf16* W, int E, int C, int I, uint32_t rows) {      // Wd [E, C, I]
  const uint64_t d[3] = {(uint64_t)I, (uint64_t)C, (uint64_t)E}, s[2] = {2ull * I, 2ull * C * I};
  const uint32_t b[3] = {64, rows, 1};
  return mlb_make_tmap_nd(m, W, 3, d, s, b);
}
bool map_gate_up(CUtensorMap* m, const bf16* W, int E, int C, int I, uint32_t groups) {      // Wgu [E, 2 I, C] as {column, row of 16, gate or up, group, expert}
  const uint64_t d[5] = {(uint64_t)C, 16, 2, (uint64_t)I / 16, (uint64_t)E}, s[4] = {2ull * C, 2ull * I * C, 32ull * C, 4ull * I * C};
  const uint32_t b[5] = {64, 16, 2, groups, 1};
  return mlb_make_tmap_nd(m, W, 5, d, s, b);
}

struct Sizes { long N, NK; int E, k, C, I; PlanShape p; };
int sizes(Sizes& z, long N, int k, int E, int C, int I) {
  if (N < 0 || k < 1 || E < 1 || E > MAX_E || C < 16 || I < 16 || C % 16 != 0 || I % 16 != 0 || C > (1 << 20) || I > (1 << 20)) return -7;
  if (N * k + 32L * E >= (1L << 31)) return -7;
  z = {N, N * k, E, k, C, I, plan_shape(N * k, E)};
  return 0;
}
PlanArgs plan_args(int* plan, const int* idx, const Sizes& z) {
  return {plan, plan + z.E + 1, plan + 2 * z.E + 1, (int4*)(plan + z.p.tiles), plan + z.p.place, plan + z.p.source, plan + z.p.hist, idx, z.NK, z.E, z.p.blocks, z.p.per_block};
}
bool off16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if ((uintptr_t)p & 15) return true;
  return false;
}
int dispatch(bf16* out, const bf16* x, const PlanArgs& P, const Sizes& z, long ldx, cudaStream_t st) {
  return (int)mlb_launch(moe_dispatch_k, dim3((unsigned)((z.p.rows + 7) / 8)), dim3(256), 0, st, out, x, (const int*)P.source, (const int*)(P.start + z.E), ldx, z.k, z.C);
}
template <typename W>
int combine(bf16* out, const bf16* y, const W* w, const PlanArgs& P, const Sizes& z, cudaStream_t st) {
  return (int)mlb_launch(moe_combine_k<W>, dim3((unsigned)((z.N * (z.C / 8) + 255) / 256)), dim3(256), 0, st, out, y, w, (const int*)P.place, z.N, z.k, z.C);
}

}  // namespace

#define MLB_TRY(x) do { const int rc_ = (x); if (rc_ != 0) return rc_; } while (0)

// ints of a plan, rows of its buffers; -7: sizes out of range
MLB_API long mlb_moe_plan_ints(long N, int k, int E) {
  Sizes z;
  if (sizes(z, N, k, E, 16, 16) != 0) return -7;
  return z.p.total;
}
MLB_API long mlb_moe_plan_rows(long N, int k, int E) {
  Sizes z;
  if (sizes(z, N, k, E, 16, 16) != 0) return -7;
  return z.p.rows;
}
MLB_API int mlb_moe_plan(int* plan, const int* idx, long N, int k, int E, cudaStream_t st) {
  Sizes z;
  MLB_TRY(sizes(z, N, k, E, 16, 16));
  if (off16({plan})) return -7;
  if (z.NK == 0) return 0;
  const PlanArgs P = plan_args(plan, idx, z);
  if (z.p.blocks > 1) MLB_TRY((int)mlb_launch(moe_hist_k, dim3(z.p.blocks), dim3(PLAN_THREADS), (size_t)4 * E, st, P));
  return (int)mlb_launch(moe_place_k, dim3(z.p.blocks), dim3(PLAN_THREADS), (size_t)4 * E * (2 + PLAN_WARPS), st, P);
}
// xs [R, C], gu [R, 2 I] (null: not kept), h [R, I], y [R, C] are workspace, the first two what backward needs
MLB_API int mlb_moe_fwd(void* out, void* xs, void* gu, void* h, void* y, const void* x, const void* weights, const void* gate_up, const void* down, const int* plan, long N, long ldx, int k,
                        int E, int C, int I, int wbits, cudaStream_t st) {
  Sizes z;
  MLB_TRY(sizes(z, N, k, E, C, I));
  if (off16({out, xs, gu, h, y, x, gate_up, down, plan}) || ldx % 8 != 0 || (wbits != 16 && wbits != 32)) return -7;
  if (z.NK == 0) return 0;
  const PlanArgs P = plan_args(const_cast<int*>(plan), nullptr, z);
  alignas(64) CUtensorMap a, b;
  MLB_TRY(dispatch((bf16*)xs, (const bf16*)x, P, z, ldx, st));
  GemmArgs g = {P.start, P.tiles, P.ntiles, (bf16*)gu, (bf16*)h, E, 2 * I, 0, C, (2 * I + 255) / 256, 1};
  if (!map_gate_up(&a, (const bf16*)gate_up, E, C, I, 4) || !map_tokens(&b, (const bf16*)xs, z.p.rows, C)) return -2;
  MLB_TRY(launch_gemm<GATE_UP>(a, b, g, (long)z.p.max_tiles * g.tiles_m, st));
  g = {P.start, P.tiles, P.ntiles, (bf16*)y, nullptr, E, C, 0, I, (C + 255) / 256, 1};
  if (!map_down(&a, (const bf16*)down, E, C, I, 128) || !map_tokens(&b, (const bf16*)h, z.p.rows, I)) return -2;
  MLB_TRY(launch_gemm<DOWN>(a, b, g, (long)z.p.max_tiles * g.tiles_m, st));
  return wbits == 16 ? combine((bf16*)out, (const bf16*)y, (const bf16*)weights, P, z, st) : combine((bf16*)out, (const bf16*)y, (const float*)weights, P, z, st);
}
// ys [R, C], dh [R, I], dgu [R, 2 I], hw [R, I], dxs [R, C]: workspace.  dx, dgate_up and ddown that are null are not formed
MLB_API int mlb_moe_bwd(void* dx, void* dweights, void* dgate_up, void* ddown, void* ys, void* dh, void* dgu, void* hw, void* dxs, const void* dout, const void* xs, const void* gu,
                        const void* weights, const void* gate_up, const void* down, const int* plan, long N, long ldo, int k, int E, int C, int I, int wbits, cudaStream_t st) {
  Sizes z;
  MLB_TRY(sizes(z, N, k, E, C, I));
  if (off16({dx, dgate_up, ddown, ys, dh, dgu, hw, dxs, dout, xs, gu, gate_up, down, plan}) || ldo % 8 != 0 || (wbits != 16 && wbits != 32)) return -7;
  if (z.NK == 0) return 0;
  const PlanArgs P = plan_args(const_cast<int*>(plan), nullptr, z);
  const int* rows = P.start + E;
  alignas(64) CUtensorMap a, b;
  MLB_TRY(dispatch((bf16*)ys, (const bf16*)dout, P, z, ldo, st));
  GemmArgs g = {P.start, P.tiles, P.ntiles, (bf16*)dh, nullptr, E, I, 0, C, (I + 255) / 256, 1};
  if (!map_down(&a, (const bf16*)down, E, C, I, 64) || !map_tokens(&b, (const bf16*)ys, z.p.rows, C)) return -2;
  MLB_TRY(launch_gemm<DOWN_T>(a, b, g, (long)z.p.max_tiles * g.tiles_m, st));
  const dim3 every((unsigned)z.p.rows), copies((unsigned)((z.NK + 255) / 256));
  if (wbits == 16) {
    MLB_TRY((int)mlb_launch(moe_swiglu_bwd_k<bf16>, every, dim3(128), 0, st, (bf16*)dgu, (bf16*)hw, (bf16*)dweights, (const bf16*)dh, (const bf16*)gu, (const bf16*)weights, (const int*)P.source, rows, I));
    MLB_TRY((int)mlb_launch(moe_no_place_k<bf16>, copies, dim3(256), 0, st, (bf16*)dweights, (const int*)P.place, z.NK));
  } else {
    MLB_TRY((int)mlb_launch(moe_swiglu_bwd_k<float>, every, dim3(128), 0, st, (bf16*)dgu, (bf16*)hw, (float*)dweights, (const bf16*)dh, (const bf16*)gu, (const float*)weights, (const int*)P.source, rows, I));
    MLB_TRY((int)mlb_launch(moe_no_place_k<float>, copies, dim3(256), 0, st, (float*)dweights, (const int*)P.place, z.NK));
  }
  if (dx != nullptr) {
    g = {P.start, P.tiles, P.ntiles, (bf16*)dxs, nullptr, E, C, 0, 2 * I, (C + 255) / 256, 1};
    if (!map_gate_up(&a, (const bf16*)gate_up, E, C, I, 2) || !map_tokens(&b, (const bf16*)dgu, z.p.rows, 2 * I)) return -2;
    MLB_TRY(launch_gemm<GATE_UP_T>(a, b, g, (long)z.p.max_tiles * g.tiles_m, st));
    MLB_TRY(combine((bf16*)dx, (const bf16*)dxs, (const float*)nullptr, P, z, st));
  }
  if (dgate_up != nullptr) {
    g = {P.start, P.tiles, P.ntiles, (bf16*)dgate_up, nullptr, E, 2 * I, C, 0, (2 * I + 255) / 256, (C + 255) / 256};
    if (!map_rows(&a, (const bf16*)dgu, z.p.rows, 2 * I) || !map_rows(&b, (const bf16*)xs, z.p.rows, C)) return -2;
    MLB_TRY(launch_gemm<D_GATE_UP>(a, b, g, (long)E * g.tiles_m * g.tiles_n, st));
  }
  if (ddown != nullptr) {
    g = {P.start, P.tiles, P.ntiles, (bf16*)ddown, nullptr, E, C, I, 0, (C + 255) / 256, (I + 255) / 256};
    if (!map_rows(&a, (const bf16*)ys, z.p.rows, C) || !map_rows(&b, (const bf16*)hw, z.p.rows, I)) return -2;
    MLB_TRY(launch_gemm<D_DOWN>(a, b, g, (long)E * g.tiles_m * g.tiles_n, st));
  }
  return 0;
}
