// The experts of a mixture: tokens sorted by expert, the experts' products on the tensor cores, the weighted sum of what they give.
//
//   out_n = sum_j w_nj Wd[e] (silu(g) * u),   [g | u] = Wgu[e] x_n,   e = idx_nj (negative: nothing)
//
// A copy of a token is a pair (token n, place j), numbered n k + j.  The plan puts the copies in rows by expert, each expert's rows beginning at a multiple of 32 and
// filled up with empty rows, so that a product's tile and the reductions over tokens end where an expert does:
//   forward    xs = rows of x;  [g | u] = xs Wgu^T, h = silu(g) u (one product, h formed from its accumulators);  y = h Wd^T;  out = weighted sums of y
//   backward   ys = rows of w dout, dw = dout . y;  dh = ys Wd and from it dgu;  dxs = dgu Wgu, dx = sums of it;  dWgu = dgu^T xs;  dWd = ys^T h
// Of the forward pass xs, [g | u], h and y are kept: with h and y the gradient of a weight and that of Wd need neither SwiGLU again nor a second set of rows.
// Rounded to bf16 on the way, all sums being fp32: h, ys and dgu, which the tensor cores take in no wider form that is as fast; [g | u], from whose rounded values backward forms
// the gradient again; y and dxs, which in fp32 would be 50 MB more to write and to read each at 16384 x 2 copies of 768 (some 15 us).  Outputs are 0.0029, gradients 0.0039 of their norm from
// 64 bits, of which the last rounding is 0.0017.
// Counts are known on the device only: grids are sized by what there may be at most, and blocks that find nothing leave.
#include "../tc.cuh"
#include "moe_route.cuh"

namespace {

MLB_DEFINE_ERROR_WORD(moe)

constexpr int PAD = 32;            // an expert's rows begin at a multiple of this
constexpr int TILE_TOKENS = 256;   // rows of a tile of the token products

// ------------------------------------------------------------------ the plan
// int32: start[E + 1], order[E], ntiles | tiles[maxT] {expert, first row, rows, 0} | place[N k] | source[R] | hist[blocks][E]
struct PlanShape {
  long rows, tiles, place, source, hist, total;      // R; offsets of the parts in ints
  int max_tiles, blocks, per_block;
};
// PLAN_BATCH: copies that a lane asks for at a time.  One block takes up to 2048 copies, with a run of 32 to 256 of them to each of its 8 warps, which put theirs in rows one 32 behind the other; of
// more than 1024 it has 32 warps (32 copies to 8 experts: 4.7 us with 32 warps, 3.1 with 8; 1024 of 64: 6.6 and 5.7; 1806 of 64, by themselves: 8.7 and 10.4), unless there are more lists of
// counts than shared memory takes.
constexpr int PLAN_BATCH = 8;
inline int plan_warps(int E, long NK) { return E <= 256 && NK > 1024 && NK <= 2048 ? 32 : 8; }
inline PlanShape plan_shape(long NK, int E) {
  PlanShape p;
  const long used = NK < E ? NK : E, step = NK <= 2048 ? 32 * plan_warps(E, NK) : 1024;
  p.rows = (NK + (PAD - 1) * used) / PAD * PAD;
  p.max_tiles = (int)(NK / TILE_TOKENS + used);
  p.per_block = (int)std::max(step, ((NK <= 2048 ? NK : (NK + 127) / 128) + step - 1) / step * step);
  p.blocks = (int)((NK + p.per_block - 1) / p.per_block);
  p.tiles = (2L * E + 2 + 3) / 4 * 4;
  p.place = p.tiles + 4L * p.max_tiles;
  p.source = p.place + NK;
  p.hist = p.source + p.rows;
  p.total = p.hist + (p.blocks > 1 ? (long)p.blocks * E : 0);
  return p;
}
struct PlanArgs {
  int *start, *order, *ntiles;
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
__global__ void __launch_bounds__(256) moe_hist_k(const PlanArgs A) {
  mlb_pdl_sync();
  extern __shared__ int cnt[];
  for (int e = threadIdx.x; e < A.E; e += (int)blockDim.x) cnt[e] = 0;
  __syncthreads();
  const long i0 = (long)blockIdx.x * A.per_block;
  for (int i = threadIdx.x; i < A.per_block; i += (int)blockDim.x) {
    const int e = expert_of(A, i0 + i);
    if (e >= 0) atomicAdd(&cnt[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < A.E; e += (int)blockDim.x) A.hist[(long)blockIdx.x * A.E + e] = cnt[e];
}
// Every block adds up all blocks' counts for itself and puts its copies behind those of the blocks before it, in order: the same rows on every run.
__global__ void __launch_bounds__(1024) moe_place_k(const PlanArgs A) {
  mlb_pdl_sync();
  extern __shared__ int sm[];
  const int E = A.E, tid = threadIdx.x, lane = tid & 31, w = tid >> 5, threads = blockDim.x, nw = threads >> 5;
  int *total = sm, *base = sm + E, *mine = sm + 2 * E;      // mine[nw][E]
  __shared__ int2 warps[32];
  for (int e = tid; e < (2 + nw) * E; e += (int)blockDim.x) sm[e] = 0;
  __syncthreads();
  // the copies of this block, a run of them to each warp
  const int run = A.per_block / nw;
  const long i0 = (long)blockIdx.x * A.per_block + (long)w * run;
  for (int i = lane; i < run; i += 32 * PLAN_BATCH) {
    int e[PLAN_BATCH];
#pragma unroll
    for (int j = 0; j < PLAN_BATCH; j++) e[j] = i + 32 * j < run ? expert_of(A, i0 + i + 32 * j) : -1;
#pragma unroll
    for (int j = 0; j < PLAN_BATCH; j++)
      if (e[j] >= 0) atomicAdd(&mine[w * E + e[j]], 1);
  }
  if (A.blocks > 1) {
    if (E >= 128) {
      for (int e = tid; e < E; e += (int)blockDim.x) {
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
      for (int i = tid; i < n; i += (int)blockDim.x) {
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
    for (int e = tid; e < E; e += (int)blockDim.x) {
      int all = 0;
      for (int k = 0; k < nw; k++) all += mine[k * E + e];
      total[e] = all;
    }
    __syncthreads();
  }
  // rows and tiles of the experts before each (a thread has `per` experts, one behind the other)
  const int per = (E + threads - 1) / threads, e0 = tid * per, e1 = min(e0 + per, E);
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
      A.start[e] = row;
      int before = 0;      // experts with more rows: those come first in the weight gradients
      for (int x = 0; x < E; x++) before += total[x] > n || (total[x] == n && x < e);
      A.order[before] = e;
      for (int t = 0; t < n; t += TILE_TOKENS) A.tiles[tile++] = make_int4(e, row + t, min(TILE_TOKENS, n - t), 0);
      for (int t = n; t < padded; t++) A.source[row + t] = -1;
    }
    int at = row + base[e];
    for (int k = 0; k < nw; k++) {
      const int v = mine[k * E + e];
      mine[k * E + e] = at;
      at += v;
    }
    row += padded;
  }
  if (writes && tid == threads - 1) A.start[E] = sum.x, *A.ntiles = sum.y;
  __syncthreads();
  for (int i = lane; i < run; i += 32 * PLAN_BATCH) {      // (run is a multiple of 32)
    int es[PLAN_BATCH];
#pragma unroll
    for (int j = 0; j < PLAN_BATCH; j++) es[j] = i + 32 * j < run ? expert_of(A, i0 + i + 32 * j) : -1;
#pragma unroll
    for (int j = 0; j < PLAN_BATCH; j++) {
      if (i - lane + 32 * j >= run) break;      // (the warp's)
      const long at = i0 + i + 32 * j;
      const int e = es[j];
      const unsigned same = __match_any_sync(0xffffffffu, e);
      const int first = e >= 0 ? mine[w * E + e] : 0;
      __syncwarp();
      const int rank = __popc(same & ((1u << lane) - 1));
      if (e >= 0) {
        if (rank == 0) mine[w * E + e] = first + __popc(same);
        A.place[at] = first + rank;
        A.source[first + rank] = (int)at;
      } else if (at < A.NK) {
        A.place[at] = -1;
      }
      __syncwarp();
    }
  }
}

// ------------------------------------------------------------------ tokens to rows, rows to tokens
template <typename T> __device__ __forceinline__ float as_float(T v) { return (float)v; }
template <> __device__ __forceinline__ float as_float<bf16>(bf16 v) { return __bfloat162float(v); }
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

__device__ __forceinline__ void add8(float (&s)[8], const uint4& v, float w) {
  const uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    s[2 * i] = fmaf(__uint_as_float(q[i] << 16), w, s[2 * i]);
    s[2 * i + 1] = fmaf(__uint_as_float(q[i] & 0xffff0000u), w, s[2 * i + 1]);
  }
}
// backward: out[r] = w dout of its token, rounded once, and the weight's gradient dout . y; a warp to a copy.  What fills up the experts' rows is written as zeros
// (the weight gradients add it up) by the blocks behind the copies', a copy that goes nowhere has the gradient 0.
template <typename W>
__global__ void __launch_bounds__(256) moe_dispatch_bwd_k(bf16* __restrict__ out, W* __restrict__ dweights, const bf16* __restrict__ dout, const bf16* __restrict__ y,
                                                          const W* __restrict__ weights, const int* __restrict__ place, const int* __restrict__ source, const int* __restrict__ rows,
                                                          long ldo, int NK, int k, int C, int copy_blocks) {
  mlb_pdl_sync();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if ((int)blockIdx.x >= copy_blocks) {      // 32 rows to a warp, of which few are empty
    const long r0 = ((long)(blockIdx.x - copy_blocks) * 8 + warp) * 32;
    for (unsigned empty = __ballot_sync(0xffffffffu, r0 < *rows && source[r0 + lane] < 0); empty; empty &= empty - 1) {
      uint4* o = reinterpret_cast<uint4*>(out + (r0 + __ffs(empty) - 1) * C);
      for (int c = lane; c < C / 8; c += 32) o[c] = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const int i = blockIdx.x * 8 + warp;
  if (i >= NK) return;
  const int r = place[i];
  float dot = 0.f;
  if (r >= 0) {
    const float w = as_float(weights[i]);
    const uint4 *in = reinterpret_cast<const uint4*>(dout + (long)(i / k) * ldo), *yr = reinterpret_cast<const uint4*>(y + (long)r * C);
    uint4* o = reinterpret_cast<uint4*>(out + (long)r * C);
#pragma unroll 2
    for (int c = lane; c < C / 8; c += 32) {
      const uint4 a = __ldg(in + c), b = __ldg(yr + c);
      const uint32_t aq[4] = {a.x, a.y, a.z, a.w}, bq[4] = {b.x, b.y, b.z, b.w};
      uint32_t q[4];
#pragma unroll
      for (int v = 0; v < 4; v++) {
        const float lo = __uint_as_float(aq[v] << 16), hi = __uint_as_float(aq[v] & 0xffff0000u);
        dot = fmaf(lo, __uint_as_float(bq[v] << 16), dot);
        dot = fmaf(hi, __uint_as_float(bq[v] & 0xffff0000u), dot);
        q[v] = pack_bf16(w * lo, w * hi);
      }
      o[c] = make_uint4(q[0], q[1], q[2], q[3]);
    }
    dot = warp_sum(dot);
  }
  if (lane == 0) dweights[i] = (W)dot;
}
// out[n] = sum_j w[n, j] y[place[n, j]] in the order of j, in fp32; without weights plain sums.  A warp to a token, or, of few
// tokens, to 256 columns of one (301 tokens of 6 x 2048 columns: 11.4 us with whole tokens, 6.1 so); a lane has SPAN times eight columns on their way.  16384 tokens of 2 x 768: 16.8 us, of 11.5
// for the bytes.
template <typename W, int SPAN>
__global__ void __launch_bounds__(256) moe_combine_k(bf16* __restrict__ out, const bf16* __restrict__ y, const W* __restrict__ weights, const int* __restrict__ place, long N, int k, int C) {
  mlb_pdl_sync();
  const long n = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (n >= N) return;
  const int lane = threadIdx.x & 31, vec = C / 8;
  for (int c0 = blockIdx.y * 32 + lane; c0 < vec; c0 += 32 * SPAN * gridDim.y) {
    float s[SPAN][8] = {};
#pragma unroll 2
    for (int j = 0; j < k; j++) {
      const int r = place[n * k + j];
      if (r < 0) continue;
      const float w = weights ? as_float(weights[n * k + j]) : 1.f;
      const uint4* row = reinterpret_cast<const uint4*>(y + (long)r * C) + c0;
      uint4 v[SPAN];
#pragma unroll
      for (int i = 0; i < SPAN; i++)
        if (c0 + 32 * i < vec) v[i] = __ldg(row + 32 * i);
#pragma unroll
      for (int i = 0; i < SPAN; i++)
        if (c0 + 32 * i < vec) add8(s[i], v[i], w);
    }
    uint4* o = reinterpret_cast<uint4*>(out + n * C) + c0;
#pragma unroll
    for (int i = 0; i < SPAN; i++)
      if (c0 + 32 * i < vec) o[32 * i] = make_uint4(pack_bf16(s[i][0], s[i][1]), pack_bf16(s[i][2], s[i][3]), pack_bf16(s[i][4], s[i][5]), pack_bf16(s[i][6], s[i][7]));
  }
}

// ------------------------------------------------------------------ products
// CTA pairs share a tile of 256 features x up to 256 tokens (token products) or 256 x 256 features (weight gradients): the leader issues tcgen05.mma.cta_group::2,
// each CTA stages its 128 rows of A and its half of B and drains its own 128 tensor-memory lanes.  The weights are A and the tokens B, whose number
// an instruction takes in steps of 32: an expert's last tile, and that of an expert with few tokens, is no wider than its rows.  Two accumulators, so that a tile's
// epilogue runs under the next one's products.
//   GATE_UP  [g | u] = xs Wgu^T and h = silu(g) u;  H  the same, of which only h is kept
//   DOWN     y = h Wd^T
//   DOWN_T   dh = ys Wd, and from it dgu
//   BACK     dWgu, dWd and dxs = dgu Wgu, one launch: tiles of all three behind one another, so that only one last wave leaves SMs idle
// us (PFLOP/s) with 16384 tokens to 2 of 8 experts of 2048 behind 768 columns, and with 4096 to 6 of 64 of 1376 behind 2048, whose rows are 1 to 2900:
//   GATE_UP  152 (1.36)   248 (1.12)      a tile's operands are 62 bytes a clock and SM from the L2, all that it gives; what is stored and few rows to a tile come on top
//   DOWN      82 (1.26)   134 (1.03)
//   DOWN_T   110 (0.94)   154 (0.90)      memory: 573 MB in the first, 5.2 TB/s
//   BACK     356 (1.45)   668 (1.04)      1.08 GB of weight gradients in the second
enum { GATE_UP, DOWN, DOWN_T, BACK, H };
constexpr int BK = 64;
// An epilogue warp has 32 features, of CHUNK tokens at a time.  GATE_UP, DOWN and BACK: four warps have the same tokens and put what leaves side by side, rows of 128 bytes in boxes of
// 4 KB (two, and one of h), two places in turn; by itself a warp would have rows of 64 bytes, and of 32 of h, which the L2 takes as slowly as whole ones (GATE_UP, 16384 tokens to
// 2 of 8 experts of 2048 behind 768 columns: 159 us, 126 with nothing stored, 149 so).  A weight gradient's rows: 4 KB a warp.  DOWN_T: two places a warp for [g | u], which arrive, become
// their gradients where they stand and leave; what comes next is asked for before the arithmetic (132 us behind it, 116 so; with five stages of operands instead of four 110).
template <int MODE>
struct Smem {
  static constexpr int EPI = MODE == DOWN_T ? 16 : 8, THREADS = 64 + 32 * EPI;      // epilogue warps
  static constexpr int CHUNK = MODE == DOWN_T ? 16 : 32;
  static constexpr int A_BYTES = 128 * BK * 2, STAGE_BYTES = 2 * A_BYTES, STAGES = MODE == DOWN_T || MODE == GATE_UP ? 5 : 6;
  static constexpr int PLACES = 2, PLACE = 128 * CHUNK, WARP_BYTES = MODE == DOWN_T ? PLACES * PLACE : MODE == GATE_UP ? 2 * 2048 + 2 * 1024 : MODE == H ? 2 * 1024 : 4096;
  static constexpr int TOTAL = STAGES * STAGE_BYTES + EPI * WARP_BYTES + 512 + 1024;
  static_assert(WARP_BYTES % 1024 == 0 && TOTAL <= 232448, "shared memory of an SM");
};
struct GemmArgs {
  const int *start, *order;      // rows of the experts [E + 1]; the experts, those with the most rows first
  const int4* tiles;
  const int* ntiles;
  bf16 *out, *h;         // [R, M]; GATE_UP, H (which has no out): h [R, M / 2].  DOWN_T: dgu [R, 2 M].  BACK: dxs
  int E, M, K, tiles_m;  // token products: M features over K
  // BACK
  int C, I, per_gate_up, per_down;      // tiles of one expert (0: not asked for)
};
enum { TOKENS, D_GATE_UP, D_DOWN };
struct Item { int type, e, row0, rows, mt, nt; };
template <int MODE>
struct Items {      // items cid, cid + ncl, ... ; what the next one is read from memory is asked for ahead
  const GemmArgs& g;
  int i, step, n, grads;
  int4 ahead;
  __device__ __forceinline__ Items(const GemmArgs& g_, int cid, int ncl) : g(g_), i(cid), step(ncl) {
    grads = MODE == BACK ? g.E * (g.per_gate_up + g.per_down) : 0;
    n = grads + (g.tiles_m > 0 ? *g.ntiles * g.tiles_m : 0);
    fetch();
  }
  __device__ __forceinline__ void fetch() {
    if (i >= n) return;
    if (MODE == BACK && i < grads) {
      const int e = g.order[i / (g.per_gate_up + g.per_down)];
      ahead.x = e, ahead.y = g.start[e], ahead.z = g.start[e + 1];
    } else {
      ahead = g.tiles[(i - grads) / g.tiles_m];
    }
  }
  __device__ __forceinline__ bool next(Item& w) {
    if (i >= n) return false;
    w.e = ahead.x, w.row0 = ahead.y;
    if (MODE == BACK && i < grads) {
      const int x = i % (g.per_gate_up + g.per_down);
      w.type = x < g.per_gate_up ? D_GATE_UP : D_DOWN;
      w.rows = ahead.z - ahead.y;
      const int y = x < g.per_gate_up ? x : x - g.per_gate_up, nt = ((x < g.per_gate_up ? g.C : g.I) + 255) / 256;
      w.mt = y / nt, w.nt = y - w.mt * nt;
    } else {
      w.type = TOKENS;
      w.rows = ahead.z;
      w.mt = (i - grads) % g.tiles_m, w.nt = 0;
    }
    i += step;
    fetch();
    return true;
  }
};
// One warp's 32 x 64 accumulators (lane = row) as bf16 to its 4 KB buffer, from where they leave
__device__ __forceinline__ void put_rows(uint8_t* buf, int lane, const uint32_t (&r)[32], const uint32_t (&r2)[32]) {
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
}
// Unit u (8 features) of token t in rows of 128 bytes, swizzled as TMA has them
__device__ __forceinline__ int wide_at(int t, int u) { return t * 128 + ((u ^ (t & 7)) << 4); }

// Two fp32 values an instruction
typedef uint64_t Two;
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void parts(Two x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ Two two_bf16(uint32_t q) { return two(__uint_as_float(q << 16), __uint_as_float(q & 0xffff0000u)); }
__device__ __forceinline__ uint32_t pack_two(Two x) {
  float a, b;
  parts(x, a, b);
  return pack_bf16(a, b);
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ Two sigmoid2(Two g) {
  float a, b;
  parts(mul2(g, two(-1.44269504f, -1.44269504f)), a, b);
  return two(rcp(1.f + ex2(a)), rcp(1.f + ex2(b)));
}
__device__ __forceinline__ Two swiglu2(Two g, Two u) { return mul2(mul2(g, sigmoid2(g)), u); }

// SwiGLU's gradient, one feature of two tokens.  With s = sigmoid(g) and d = dh:  dg = d u s (1 + g (1 - s)),  du = d g s
__device__ __forceinline__ void swiglu_bwd2(uint32_t& gq, uint32_t& uq, Two d) {
  const Two g = two_bf16(gq), u = two_bf16(uq), s = sigmoid2(g), silu = mul2(g, s);
  gq = pack_two(mul2(mul2(d, u), fma2(silu, fma2(s, two(-1.f, -1.f), two(1.f, 1.f)), s)));
  uq = pack_two(mul2(d, silu));
}

template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Smem<MODE>::THREADS, 1)
moe_gemm_k(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmB16, const __grid_constant__ CUtensorMap tmA1,
           const __grid_constant__ CUtensorMap tmB1, const __grid_constant__ CUtensorMap tmA2, const __grid_constant__ CUtensorMap tmB2, const __grid_constant__ CUtensorMap tmOut,
           const __grid_constant__ CUtensorMap tmOut1, const __grid_constant__ CUtensorMap tmOut2, const GemmArgs g) {
  using S = Smem<MODE>;
  constexpr int STAGES = S::STAGES, ACC = 256, CHUNK = S::CHUNK, PASS = CHUNK * S::EPI / 4;
  constexpr bool A_MN = MODE == DOWN_T || MODE == BACK;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* staging = smem + STAGES * S::STAGE_BYTES;
  uint64_t* full = (uint64_t*)(staging + S::EPI * S::WARP_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* place_full = acc_empty + 2;      // [EPI][PLACES]
  uint32_t* tmem_slot = (uint32_t*)(place_full + (MODE == DOWN_T ? S::EPI * S::PLACES : 0));
  volatile uint32_t* late = tmem_slot + 1;      // the accumulators of some epilogue warp did not come: no tokens' tile is stored

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = tc::cluster_ctarank();
  const int cid = (int)tc::cluster_id_x(), ncl = (int)tc::cluster_count_x();

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; i++) { tc::mbar_init(&full[i], 1); tc::mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; i++) { tc::mbar_init(&acc_full[i], 1); tc::mbar_init(&acc_empty[i], 2 * S::EPI); }
    *late = 0;
    if (MODE == DOWN_T)
      for (int i = 0; i < S::EPI * S::PLACES; i++) tc::mbar_init(&place_full[i], 1);
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
        const bool grad = MODE == BACK && w.type != TOKENS;
        const int m0 = w.mt * 256 + (int)rank * 128;
        const int kbs = ((grad ? w.rows : g.K) + BK - 1) / BK;
        const int half = ((w.rows + 31) & ~31) >> 1;      // token products: this CTA's tokens
        const uint32_t bytes = 2 * (S::A_BYTES + (grad ? S::A_BYTES : half * 128));
        for (int kb = 0; kb < kbs; kb++) {
          if (!tc::mbar_wait(&empty[stage], phase ^ 1, 0x71)) { ok = false; break; }
          uint8_t* sA = smem + stage * S::STAGE_BYTES;
          uint8_t* sB = sA + S::A_BYTES;
          const uint32_t bar = tc::mapa_u32(tc::smem_u32(&full[stage]), 0);
          if (rank == 0) tc::mbar_expect_tx(&full[stage], bytes);
          if (grad) {
            const int y = w.row0 + kb * BK, n0 = w.nt * 256 + (int)rank * 128;
            const CUtensorMap *a = w.type == D_GATE_UP ? &tmA1 : &tmA2, *b = w.type == D_GATE_UP ? &tmB1 : &tmB2;
            for (int c = 0; c < 2; c++) tc::tma_load_2d_pair(sA + c * 8192, a, bar, m0 + c * 64, y);
            for (int c = 0; c < 2; c++) tc::tma_load_2d_pair(sB + c * 8192, b, bar, n0 + c * 64, y);
          } else {
            if (MODE == GATE_UP || MODE == H) {      // rows in groups of 16 gate rows and the matching 16 up rows
              tc::tma_load_5d_pair(sA, &tmA, bar, kb * BK, 0, 0, m0 / 32, w.e);
            } else if (MODE == DOWN) {
              tc::tma_load_3d_pair(sA, &tmA, bar, kb * BK, m0, w.e);
            } else if (MODE == DOWN_T) {
              for (int c = 0; c < 2; c++) tc::tma_load_3d_pair(sA + c * 8192, &tmA, bar, m0 + c * 64, kb * BK, w.e);
            } else {                    // (K in the same groups)
              for (int c = 0; c < 2; c++) tc::tma_load_5d_pair(sA + c * 8192, &tmA, bar, m0 + c * 64, 0, 0, kb * 2, w.e);
            }
            const int y = w.row0 + (int)rank * half;
            if (half == 128) tc::tma_load_2d_pair(sB, &tmB, bar, kb * BK, y);
            else
              for (int c = 0; c < half; c += 16) tc::tma_load_2d_pair(sB + c * 128, &tmB16, bar, kb * BK, y + c);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (rank == 0)      // what was asked for last has arrived (both CTAs' part) when the kernel ends, whoever has given up on it
        for (int i = 0; i < STAGES; i++) tc::mbar_wait(&full[i], i < stage ? phase : phase ^ 1, 0x7A);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- products (one thread of the leader)
    if (rank == 0 && tc::elect_one()) {
      int stage = 0, phase = 0, it = 0;
      bool ok = true;
      Items<MODE> items(g, cid, ncl);
      Item w;
      while (ok && items.next(w)) {
        const bool grad = MODE == BACK && w.type != TOKENS;
        const int kbs = ((grad ? w.rows : g.K) + BK - 1) / BK;
        if (kbs == 0) continue;      // an expert without tokens
        const uint32_t idesc = tc::idesc_bf16(256, grad ? 256 : (w.rows + 31) & ~31, A_MN ? 1 : 0, grad ? 1 : 0);
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
          const int steps = grad ? min(BK, w.rows - kb * BK) / 16 : BK / 16;      // (the rows behind an expert's are another's)
#pragma unroll
          for (int k = 0; k < BK / 16; k++) {
            if (MODE == BACK && k >= steps) break;
            const uint64_t da = A_MN ? tc::smem_desc_sw128(sA + k * 2048, 8192, 1024) : tc::smem_desc_sw128(sA + k * 32, 16, 1024);
            const uint64_t db = grad ? tc::smem_desc_sw128(sB + k * 2048, 8192, 1024) : tc::smem_desc_sw128(sB + k * 32, 16, 1024);
            tc::mma_bf16_ss_pair(d_tmem, da, db, idesc, (kb > 0 || k > 0) ? 1u : 0u);
          }
          tc::mma_commit_pair(&empty[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (ok) tc::mma_commit_pair(&acc_full[acc]);
      }
    }
  } else {
    // ---------------------------------------------------------------- epilogue (warps 2 .. of each CTA): lanes 32 lg .., every EPI / 4-th chunk or half.  Where four warps meet at
    // barriers none of them leaves by itself: after a wait that ran out they go on without waiting, and nothing is stored.
    const int lg = warp & 3, half = (warp - 2) >> 2;
    uint8_t* buf = staging + (warp - 2) * S::WARP_BYTES;
    int it = 0, n = 0;      // items that had products; chunks of 32 tokens
    bool ok = true;
    Items<MODE> items(g, cid, ncl);
    Item w;
    // DOWN_T: the products behind a chunk's gradients are asked for a chunk ahead
    Items<MODE> ahead_items(g, cid, ncl);
    Item ahead = {};
    int ahead_c = 0, ahead_n = 0;
    auto meet = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory"); };      // the four warps that have the same tokens
    auto first_row = [&](const Item& x) { return x.mt * 256 + (int)rank * 128 + lg * 32; };
    auto advance = [&]() {      // the next chunk of this warp; rows 0: there is none
      ahead_c += PASS;
      while (ahead_c >= ((ahead.rows + 31) & ~31) || first_row(ahead) >= g.M) {
        if (!ahead_items.next(ahead)) { ahead.rows = 0; return; }
        ahead_c = half * CHUNK;
      }
    };
    auto ask = [&]() {
      if (ahead.rows == 0) return;
      if (lane == 0) {
        uint64_t* bar = &place_full[(warp - 2) * S::PLACES + ahead_n % S::PLACES];
        tc::mbar_expect_tx(bar, S::PLACE);
        tc::tma_load_2d(buf + ahead_n % S::PLACES * S::PLACE, &tmA1, bar, 2 * first_row(ahead), ahead.row0 + ahead_c);
      }
      ahead_n++;
      advance();
    };
    if constexpr (MODE == DOWN_T) {
      advance();
      for (int i = 1; i < S::PLACES; i++) ask();
    }
    while ((MODE != DOWN_T || ok) && items.next(w)) {
      const bool grad = MODE == BACK && w.type != TOKENS;
      const int m0 = first_row(w);
      const bool some = !grad || w.rows > 0;
      const int acc = it & 1, acc_phase = (it >> 1) & 1;
      const bool live = m0 < g.M;
      if (some) {
        it++;
        if (ok && !__all_sync(0xffffffffu, tc::mbar_wait(&acc_full[acc], acc_phase, 0x74))) ok = false, *late = 1;
        if (MODE == DOWN_T && !ok) break;
        tc::tc_fence_after();
      }
      const uint32_t taddr = tmem_base + ((uint32_t)(lg * 32) << 16) + acc * ACC;
      if (!grad) {
        const int last = (w.rows + 31) & ~31;      // (what fills up an expert's rows belongs to it)
        for (int c = half * CHUNK; c < last; c += PASS) {
          if (MODE == DOWN_T ? !live : m0 - lg * 32 >= g.M) break;      // (the four warps')
          uint8_t* place = MODE == DOWN_T ? buf + n % S::PLACES * S::PLACE : staging + half * (4 * S::WARP_BYTES) + (n & 1) * (2 * S::WARP_BYTES);
          const uint32_t splace = tc::smem_u32(place);
          uint32_t r[2][CHUNK / 2];
          if constexpr (MODE == DOWN_T) {
            if (lane == 0) tc::tma_wait_group_read<0>();      // the chunk before has left its place: the next one may arrive there
            __syncwarp();
            ask();
          }
          tc::tmem_ld_frag_wait(taddr + c, r);
          if constexpr (MODE != DOWN_T) {
            // what left two chunks ago has been read, its place is free; before the first chunk so have weight gradients' rows, which had all places
            if (lane == 0) {
              if (MODE == BACK && n == 0) tc::tma_wait_group_read<0>();
              else if (lg == 0) tc::tma_wait_group_read<1>();
            }
            __syncwarp();
            meet();
          }
          // r[h][4 j + 2 v + x]: token 8 j + 2 (lane % 4) + x of feature 16 h + 8 v + lane / 4
          if (MODE != DOWN_T && MODE != H) {
#pragma unroll
            for (int j = 0; j < CHUNK / 8; j++) {
              uint32_t p[4];
#pragma unroll
              for (int q = 0; q < 4; q++) p[q] = pack_bf16(__uint_as_float(r[q >> 1][4 * j + 2 * (q & 1)]), __uint_as_float(r[q >> 1][4 * j + 2 * (q & 1) + 1]));
              const int t = 8 * j + (lane & 7), u = lane >> 3;
              tc::stmatrix_x4_trans(splace + (lg >> 1) * 4096 + wide_at(t, (lg & 1) * 4 + u), p[0], p[1], p[2], p[3]);
            }
          }
          uint8_t* hs = place + (MODE == GATE_UP ? 8192 : 0);
          if constexpr (MODE == GATE_UP || MODE == H) {      // feature 8 v + lane / 4: h = 0 its gate, h = 1 its up value
            uint32_t x[8];
#pragma unroll
            for (int q = 0; q < 8; q++)
              x[q] = pack_two(swiglu2(two(__uint_as_float(r[0][2 * q]), __uint_as_float(r[0][2 * q + 1])), two(__uint_as_float(r[1][2 * q]), __uint_as_float(r[1][2 * q + 1]))));
#pragma unroll
            for (int j = 0; j < 2; j++) {
              const int t = 16 * j + 8 * (lane >> 4) + (lane & 7), u = (lane >> 3) & 1;
              tc::stmatrix_x4_trans(tc::smem_u32(hs) + wide_at(t, lg * 2 + u), x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
            }
          } else if constexpr (MODE == DOWN_T) {
            if (!__all_sync(0xffffffffu, tc::mbar_wait(&place_full[(warp - 2) * S::PLACES + n % S::PLACES], (n / S::PLACES) & 1, 0x75))) { ok = false; break; }
            const int t = 8 * (lane >> 4) + (lane & 7), v = (lane >> 3) & 1;      // rows of [16 gate | 16 up | 16 gate | 16 up]; matrices of 8 tokens x 8 features, which is how the accumulators lie
            uint32_t gate[2][4], up[2][4];
#pragma unroll
            for (int h = 0; h < 2; h++) tc::ldmatrix_x4_trans(splace + wide_at(t, 4 * h + v), gate[h]), tc::ldmatrix_x4_trans(splace + wide_at(t, 4 * h + 2 + v), up[h]);
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
              for (int q = 0; q < 4; q++) {
                swiglu_bwd2(gate[h][q], up[h][q], two(__uint_as_float(r[h][2 * q]), __uint_as_float(r[h][2 * q + 1])));
                const int left = w.rows - (c + 8 * (q >> 1) + 2 * (lane & 3));      // (rows that fill up an expert's: zeros, whatever stands in them)
                const uint32_t keep = left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
                gate[h][q] &= keep, up[h][q] &= keep;
              }
              tc::stmatrix_x4_trans(splace + wide_at(t, 4 * h + v), gate[h][0], gate[h][1], gate[h][2], gate[h][3]);
              tc::stmatrix_x4_trans(splace + wide_at(t, 4 * h + 2 + v), up[h][0], up[h][1], up[h][2], up[h][3]);
            }
            tc::fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              tc::tma_store_2d(&tmOut, place, 2 * m0, w.row0 + c);
              tc::tma_commit_group();
            }
          }
          if constexpr (MODE != DOWN_T) {
            tc::fence_async_smem();
            meet();
            if (lg == 0 && lane == 0 && !*late) {
              if (MODE != H)
                for (int i = 0; i < 2 && m0 + 64 * i < g.M; i++) tc::tma_store_2d(&tmOut, place + 4096 * i, m0 + 64 * i, w.row0 + c);
              if (MODE == GATE_UP || MODE == H) tc::tma_store_2d(&tmB1, hs, m0 / 2, w.row0 + c);
              tc::tma_commit_group();
            }
          }
          n++;
        }
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive_cluster(tc::mapa_u32(tc::smem_u32(&acc_empty[acc]), 0));
      } else if constexpr (MODE == BACK) {
        const bool gu = w.type == D_GATE_UP;
        const int M = gu ? 2 * g.I : g.C, N = gu ? g.C : g.I;
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
          const int col0 = w.nt * 256 + half * 128 + c * 64;
          if (m0 >= M || col0 >= N) continue;      // (warp-uniform)
          if (lane == 0) tc::tma_wait_group_read<0>();
          __syncwarp();
          put_rows(buf, lane, r, r2);
          tc::fence_async_smem();
          __syncwarp();
          if (ok && lane == 0) {
            if (gu) tc::tma_store_5d(&tmOut1, buf, col0, 0, 0, m0 >> 5, w.e);      // (rows of 16 of the gate and 16 of the up projection)
            else tc::tma_store_3d(&tmOut2, buf, col0, m0, w.e);
            tc::tma_commit_group();
          }
        }
      }
    }
    if constexpr (MODE == DOWN_T) {
      for (; n < ahead_n; n++) tc::mbar_wait(&place_full[(warp - 2) * S::PLACES + n % S::PLACES], (n / S::PLACES) & 1, 0x7B);      // (of a warp that has given up: what is on its way, the late one once more)
      __syncwarp();
    }
    if (lane == 0) tc::tma_wait_group<0>();
  }
  tc::tc_fence_before();
  tc::cluster_sync();      // no CTA frees tensor memory or leaves while its peer may still signal or read it
  if (warp == 1) tc::tmem_dealloc_pair(tmem_base, 2 * ACC);
}

// ------------------------------------------------------------------ few tokens
// A step of a few tokens reads the weights of the experts that they chose, once, and that is all its time.  Warps read boxes of 16 rows x 64 columns of the weights, each into shared memory
// of its own: three stages of four boxes, 192 KB an SM on their way.  The products are m16n8k16 instructions whose 16 rows are weights and whose 8 columns are tokens (which eight
// elements of the reduction an instruction has is the same for both operands: 16 neighbouring bytes a lane serve two instructions).  Two launches: h of all copies, then
// the tokens' weighted sums.  An expert's copies are found by each block for itself: 256 at most.  Up to eight tokens, the instruction's columns, as one more brings a second turn at an expert's weights
// where all go to few.  Eight tokens so, and nine by the other form, us in a graph: 6 of 64 experts of 1376 behind 2048 columns 103.9, 124.2; 2 of 8 of 5504 behind 2048 99.2, 100.5, of
// 2048 behind 768 22.9, 28.8; 2 of 2 of 5504 behind 2048 36.4, 50.6; 1 of 4 of 11008 behind 4096 109.4, 117.1.
// A warp whose wait has run out stores nothing, waits for what is on its way and leaves, meeting those that it shares barriers with until the end: 1.2 per cent of the time, the code around the
// loops' waits (one token to 6 of 64 experts 25.3 -> 25.5, eight 102.8 -> 104.0; asking for nothing more and going on was no faster).
constexpr int FEW_TOKENS = 8, FEW_COPIES = 256, FEW_WARPS = 8, FEW_THREADS = 32 * FEW_WARPS, FEW_BOX = 2048, FEW_BOXES = 4, FEW_STAGES = 3;
constexpr int FEW_SMEM = FEW_WARPS * FEW_STAGES * FEW_BOXES * FEW_BOX + 1024;
struct FewArgs {
  bf16 *out, *h;        // h [N k, I]
  const bf16* x;
  const void* weights;
  const int* idx;
  long ldx;
  int N, k, E, C, I, wbits;
  int ways;             // h: warps that share a unit
};
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The copies by expert: list[first[a] ..] are those of of[a].  More copies than an instruction's columns (a token may name an expert twice) are dealt with as if another expert had them.
struct FewLists {
  __align__(16) int expert[FEW_COPIES];
  int list[FEW_COPIES], nth[FEW_COPIES], first[FEW_COPIES + 1], of[FEW_COPIES], sums[FEW_WARPS];
};
__device__ __forceinline__ int few_lists(FewLists& L, const FewArgs& A, bool reports) {      // by 256 threads; how many experts
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, NK = A.N * A.k;
  int e = tid < NK ? __ldcg(A.idx + tid) : -1;
  if (e >= A.E) {
    if (reports && blockIdx.x == 0) mlb_set_error(MLB_ERR_BOUNDS, 0xD1);
    e = -1;
  }
  L.expert[tid] = e < 0 ? 0x7fffffff : e, L.list[tid] = -1;
  __syncthreads();
  if (e >= 0) {      // a copy's place is the number of those before it
    int less = 0, equal = 0;
#pragma unroll 4
    for (int i = 0; i < NK; i += 4) {
      const int4 x = *reinterpret_cast<const int4*>(L.expert + i);
      less += (x.x < e) + (x.y < e) + (x.z < e) + (x.w < e);
      equal += (x.x == e && i < tid) + (x.y == e && i + 1 < tid) + (x.z == e && i + 2 < tid) + (x.w == e && i + 3 < tid);
    }
    L.nth[tid] = equal;
    L.list[less + equal] = tid;
  }
  __syncthreads();
  const int here = L.list[tid];
  const bool begins = here >= 0 && L.nth[here] % 8 == 0;
  const unsigned b = __ballot_sync(0xffffffffu, begins);
  if (lane == 0) L.sums[w] = __popc(b);
  const int held = __syncthreads_count(here >= 0);
  int experts = 0, before = __popc(b & ((1u << lane) - 1));
#pragma unroll
  for (int i = 0; i < FEW_WARPS; i++) {
    before += i < w ? L.sums[i] : 0;
    experts += L.sums[i];
  }
  if (begins) L.first[before] = tid, L.of[before] = L.expert[here];
  if (tid == 0) L.first[experts] = held;
  __syncthreads();
  return experts;
}
// Eight tokens' part of one step (the reduction's columns 256 s ...): `col` is this lane's token's row
__device__ __forceinline__ void few_tokens(uint4 (&v)[FEW_BOXES][2], const bf16* col, int s, int K, int t) {
#pragma unroll
  for (int x = 0; x < 2 * FEW_BOXES; x++) {
    const int k = (s * FEW_BOXES + x / 2) * 64 + x % 2 * 32 + t * 8;
    v[x / 2][x % 2] = k < K ? *reinterpret_cast<const uint4*>(col + k) : make_uint4(0, 0, 0, 0);
  }
}
// d += the products of one step, `some` boxes (two sums: neighbouring instructions do not wait for one another)
__device__ __forceinline__ void few_products(float (&d)[2][4], const uint8_t* stage, const uint4 (&v)[FEW_BOXES][2], int some, int r, int t) {
#pragma unroll
  for (int x = 0; x < FEW_BOXES; x++) {
    if (x >= some) break;
    const uint8_t* box = stage + x * FEW_BOX + r * 128;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const int at = ((t + 4 * j) ^ r) << 4;
      const uint4 p = *reinterpret_cast<const uint4*>(box + at), q = *reinterpret_cast<const uint4*>(box + 1024 + at);
      mma_16816(d[0], p.x, q.x, p.y, q.y, v[x][j].x, v[x][j].y);
      mma_16816(d[1], p.z, q.z, p.w, q.w, v[x][j].z, v[x][j].w);
    }
  }
}
// h: a unit is 8 rows of the gate and 8 of the up projection of an expert; one, two, four or eight warps share it, each with some steps of its reduction
__global__ void __launch_bounds__(FEW_THREADS, 1) moe_few_h_k(const __grid_constant__ CUtensorMap tmW, const FewArgs A) {
  mlb_pdl_sync();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ FewLists L;
  __shared__ uint64_t full[FEW_WARPS][FEW_STAGES];
  __shared__ float4 part[2][FEW_WARPS][32];
  __shared__ volatile int late;      // a wait of some warp ran out: what it shares units of is not stored
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if (threadIdx.x == 0) late = 0;
  if (lane == 0) {
    for (int i = 0; i < FEW_STAGES; i++) tc::mbar_init(&full[w][i], 1);
    tc::mbar_fence_init();
    if (w == 0) tc::tma_prefetch_desc(&tmW);
  }
  const int experts = few_lists(L, A, true);
  const int K = A.C, groups = A.I / 8, units = experts * groups, boxes = (K + 63) / 64, steps = (boxes + FEW_BOXES - 1) / FEW_BOXES;
  // the units of this warp and those beside it; of each it has the steps `part_of`, part_of + ways, ...
  const int r = lane >> 2, t = lane & 3, ways = A.ways, part_of = w % ways, begin = blockIdx.x + w / ways * gridDim.x, every = gridDim.x * (FEW_WARPS / ways);
  uint8_t* ring = smem + w * (FEW_STAGES * FEW_BOXES * FEW_BOX);
  int next_unit = begin, next_s = part_of, asked = 0, n = 0, turn = 0;      // the step that is asked for next; how many have been, and have been dealt with
  auto ask = [&]() {
    if (next_unit >= units || part_of >= steps) return;
    if (lane == 0) {
      const int a = next_unit / groups, g = next_unit - a * groups, stage = asked % FEW_STAGES, some = min(FEW_BOXES, boxes - next_s * FEW_BOXES);
      uint64_t* bar = &full[w][stage];
      tc::mbar_expect_tx(bar, some * FEW_BOX);
      for (int j = 0; j < some; j++) tc::tma_load_5d(ring + (stage * FEW_BOXES + j) * FEW_BOX, &tmW, bar, (next_s * FEW_BOXES + j) * 64, 0, 0, g, L.of[a]);
    }
    asked++;
    if ((next_s += ways) >= steps) next_s = part_of, next_unit += every;
  };
  for (int i = 0; i < FEW_STAGES; i++) ask();
  uint4 ahead[FEW_BOXES][2] = {};      // the tokens' part of the next step, asked for while this one goes on
  auto tokens = [&](int unit, int s) {
    const int a = unit / groups, f0 = L.first[a], c = L.list[f0 + min(r, L.first[a + 1] - f0 - 1)];      // (columns behind the last copy: its row, nothing of theirs is used)
    few_tokens(ahead, A.x + (size_t)(c / A.k) * A.ldx, s, K, t);
  };
  if (begin < units && part_of < steps) tokens(begin, part_of);
  for (int unit = begin; unit < units; unit += every, turn ^= 1) {
    const int a = unit / groups, g = unit - a * groups, f0 = L.first[a], copies = L.first[a + 1] - f0;
    float d[2][4] = {};
#pragma unroll 1
    for (int s = part_of; s < steps; s += ways, n++) {
      uint4 v[FEW_BOXES][2];
#pragma unroll
      for (int x = 0; x < 2 * FEW_BOXES; x++) v[x / 2][x % 2] = ahead[x / 2][x % 2];
      if (s + ways < steps) tokens(unit, s + ways);
      else if (unit + every < units) tokens(unit + every, part_of);
      const int stage = n % FEW_STAGES;
      if (!__all_sync(0xffffffffu, tc::mbar_wait(&full[w][stage], (n / FEW_STAGES) & 1, 0x76))) {
        // nothing more is asked for or stored; what is on its way is waited for, the late one once more, and so are the warps that share units with this one
        late = 1;
        for (int x = n; x < asked; x++) tc::mbar_wait(&full[w][x % FEW_STAGES], (x / FEW_STAGES) & 1, 0x77);
        __syncwarp();
        for (; ways > 1 && unit < units; unit += every) asm volatile("bar.sync %0, %1;" ::"r"(1 + w / ways), "r"(32 * ways) : "memory");
        return;
      }
      few_products(d, ring + stage * FEW_BOXES * FEW_BOX, v, boxes - s * FEW_BOXES, r, t);
      __syncwarp();
      ask();
    }
    // d[..][2 h + x]: row 8 h + lane / 4, column 2 (lane % 4) + x.  The first half of the rows is the gate's, the second the up projection's.
    float4 sum = make_float4(d[0][0] + d[1][0], d[0][1] + d[1][1], d[0][2] + d[1][2], d[0][3] + d[1][3]);
    if (ways > 1) {      // (two places in turn: whoever writes to one again has met the others behind their reading of it)
      part[turn][w][lane] = sum;
      asm volatile("bar.sync %0, %1;" ::"r"(1 + w / ways), "r"(32 * ways) : "memory");
      if (part_of != 0 || late) continue;
      for (int j = 1; j < ways; j++) {
        const float4 x = part[turn][w + j][lane];
        sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
      }
    }
#pragma unroll
    for (int x = 0; x < 2; x++) {
      if (2 * t + x >= copies) continue;
      const float p = x ? sum.y : sum.x, q = x ? sum.w : sum.z;
      A.h[(size_t)L.list[f0 + 2 * t + x] * A.I + g * 8 + r] = __float2bfloat16(p * rcp(1.f + ex2(-1.44269504f * p)) * q);
    }
  }
}
// out: a cluster of SPLIT blocks has 16 columns of all tokens, and its warps share the steps of all experts' reductions, a run of neighbouring ones each.  Sums of products are
// sums of their parts, so a warp adds what it has of an expert, times the weight, to sums of its own, in fp32; those of all warps are added in their order.
template <int SPLIT>
__global__ void __cluster_dims__(SPLIT, 1, 1) __launch_bounds__(FEW_THREADS, 1) moe_few_out_k(const __grid_constant__ CUtensorMap tmW, const FewArgs A) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ FewLists L;
  __shared__ uint64_t full[FEW_WARPS][FEW_STAGES];
  __shared__ float weight[FEW_COPIES], part[FEW_WARPS][8][16], sums[FEW_WARPS][FEW_TOKENS][16], from[SPLIT][FEW_TOKENS * 16];
  __shared__ volatile int late;      // a wait of some warp of the cluster ran out: nothing more is stored (asked in its first block)
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, rank = SPLIT > 1 ? (int)tc::cluster_ctarank() : 0;
  if (tid == 0) late = 0;
  // The kernel before is that for h, which has waited for all before it: idx and the weights stand, and only h has to be waited for.  (Past the L1, of which nothing is known so early.)
  if (tid < A.N * A.k) weight[tid] = A.wbits == 32 ? __ldcg((const float*)A.weights + tid) : __uint_as_float((uint32_t)__ldcg((const unsigned short*)A.weights + tid) << 16);
  if (lane == 0) {
    for (int i = 0; i < FEW_STAGES; i++) tc::mbar_init(&full[w][i], 1);
    tc::mbar_fence_init();
    if (w == 0) tc::tma_prefetch_desc(&tmW);
  }
  const int experts = few_lists(L, A, false);
  const int K = A.I, groups = A.C / 16, boxes = (K + 63) / 64, steps = (boxes + FEW_BOXES - 1) / FEW_BOXES, all = experts * steps;
  const int share = (all + FEW_WARPS * SPLIT - 1) / (FEW_WARPS * SPLIT), begin = min((rank * FEW_WARPS + w) * share, all), end = min(begin + share, all), every = gridDim.x / SPLIT;
  const int r = lane >> 2, t = lane & 3;
  uint8_t* ring = smem + w * (FEW_STAGES * FEW_BOXES * FEW_BOX);
  int next_g = blockIdx.x / SPLIT, next = begin, asked = 0, n = 0;
  auto ask = [&]() {
    if (next_g >= groups || begin >= end) return;
    if (lane == 0) {
      const int a = next / steps, box = (next - a * steps) * FEW_BOXES, stage = asked % FEW_STAGES, some = min(FEW_BOXES, boxes - box);
      uint64_t* bar = &full[w][stage];
      tc::mbar_expect_tx(bar, some * FEW_BOX);
      for (int j = 0; j < some; j++) tc::tma_load_3d(ring + (stage * FEW_BOXES + j) * FEW_BOX, &tmW, bar, (box + j) * 64, next_g * 16, L.of[a]);
    }
    asked++;
    if (++next >= end) next = begin, next_g += every;
  };
  for (int i = 0; i < FEW_STAGES; i++) ask();
  if (SPLIT > 1) tc::cluster_sync();      // (the first block of the cluster is there to be written to)
  mlb_pdl_sync();
  uint4 ahead[FEW_BOXES][2] = {};
  auto tokens = [&](int i) {
    const int a = i / steps, f0 = L.first[a], c = L.list[f0 + min(r, L.first[a + 1] - f0 - 1)];      // (columns behind the last copy: its row, nothing of theirs is used)
    few_tokens(ahead, A.h + (size_t)c * A.I, i - a * steps, K, t);
  };
  if (begin < end) tokens(begin);
  for (int g = blockIdx.x / SPLIT; g < groups; g += every) {
    for (int i = lane; i < FEW_TOKENS * 16; i += 32) (&sums[w][0][0])[i] = 0.f;
    float d[2][4] = {};
    int a = begin / steps, s = begin - a * steps;
#pragma unroll 1
    for (int i = begin; i < end; i++, n++) {
      uint4 v[FEW_BOXES][2];
#pragma unroll
      for (int x = 0; x < 2 * FEW_BOXES; x++) v[x / 2][x % 2] = ahead[x / 2][x % 2];
      tokens(i + 1 < end ? i + 1 : begin);
      const int stage = n % FEW_STAGES;
      if (!__all_sync(0xffffffffu, tc::mbar_wait(&full[w][stage], (n / FEW_STAGES) & 1, 0x78))) {
        // nothing more is asked for or stored; what is on its way is waited for, the late one once more, and so are the other warps
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc::mapa_u32(tc::smem_u32((const void*)&late), 0)), "r"(1) : "memory");
        for (int x = n; x < asked; x++) tc::mbar_wait(&full[w][x % FEW_STAGES], (x / FEW_STAGES) & 1, 0x79);
        __syncwarp();
        for (; g < groups; g += every) {
          __syncthreads();
          if (SPLIT > 1) tc::cluster_sync();
          else __syncthreads();
        }
        return;
      }
      few_products(d, ring + stage * FEW_BOXES * FEW_BOX, v, boxes - s * FEW_BOXES, r, t);
      __syncwarp();
      ask();
      if (++s < steps && i + 1 < end) continue;
      // the expert's copies are done, as far as this warp has them.  d[..][2 h + x]: row 8 h + lane / 4, column 2 (lane % 4) + x
#pragma unroll
      for (int q = 0; q < 4; q++) {
        part[w][2 * t + (q & 1)][r + 4 * (q & 2)] = d[0][q] + d[1][q];
        d[0][q] = d[1][q] = 0.f;
      }
      __syncwarp();
      const int f0 = L.first[a], copies = L.first[a + 1] - f0, row = lane & 15;
      for (int c = 0; c < copies; c++) {      // even tokens to one half of the warp, odd ones to the other: a token that names an expert twice meets itself in order
        const int copy = L.list[f0 + c], token = copy / A.k;
        if ((token & 1) == lane >> 4) sums[w][token][row] = fmaf(weight[copy], part[w][c][row], sums[w][token][row]);
      }
      __syncwarp();
      s = 0, a++;
    }
    __syncthreads();
    float sum = 0.f;
    if (tid < FEW_TOKENS * 16) {
#pragma unroll
      for (int i = 0; i < FEW_WARPS; i++) sum += (&sums[i][0][0])[tid];
      if (SPLIT > 1 && rank != 0) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(tc::mapa_u32(tc::smem_u32(&from[rank][tid]), 0)), "f"(sum) : "memory");
    }
    if (SPLIT > 1) tc::cluster_sync();      // (where blocks share columns each has one turn: `from` is not written again)
    else __syncthreads();
    if (rank == 0 && tid < 16 * A.N && !late) {
#pragma unroll
      for (int i = 1; i < SPLIT; i++) sum += from[i][tid];
      A.out[(size_t)(tid / 16) * A.C + g * 16 + tid % 16] = __float2bfloat16(sum);
    }
  }
}
int launch_few_h(const CUtensorMap& m, FewArgs g, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = mlb_allow_smem(moe_few_h_k, FEW_SMEM, done);
  if (e != cudaSuccess) return (int)e;
  const int units = std::min(g.N * g.k, g.E) * (g.I / 8), steps = (g.C + 255) / 256;
  // The number of warps to a unit with which the last round of units leaves least idle, two at least of long reductions, eight only where one round is all.  One token, whole call, us, with
  // 1, 2 and 4: 6 of 64 experts of 1376 behind 2048 columns 26.7, 26.6, 26.7 (takes 2); 8 of 128 of 768 behind 2048 23.5, 24.0, 21.9 (4); 2 of 8 of 5504 behind 2048 37.3, 32.8, 31.6 (4), of
  // 2048 behind 768 11.0, 10.3, 11.0 (2).
  const long warps = (long)FEW_WARPS * mlb_sm_count();
  auto rounds = [&](int ways) { return (units * (long)ways + warps - 1) / warps; };
  g.ways = steps >= 8 ? 2 : 1;
  for (int ways = 2 * g.ways; ways <= std::min(steps, FEW_WARPS) && (ways < FEW_WARPS || units * (long)ways <= warps); ways *= 2)
    if (g.ways * rounds(ways) < ways * rounds(g.ways)) g.ways = ways;
  return (int)mlb_launch(moe_few_h_k, dim3(std::min(units, mlb_sm_count())), dim3(FEW_THREADS), (size_t)FEW_SMEM, st, m, g);
}
template <int SPLIT>
int launch_few_out(const CUtensorMap& m, const FewArgs& g, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};
  const cudaError_t e = mlb_allow_smem(moe_few_out_k<SPLIT>, FEW_SMEM, done);
  if (e != cudaSuccess) return (int)e;
  return (int)mlb_launch(moe_few_out_k<SPLIT>, dim3(SPLIT > 1 ? SPLIT * (g.C / 16) : std::min(g.C / 16, mlb_sm_count())), dim3(FEW_THREADS), (size_t)FEW_SMEM, st, m, g);
}

struct Maps { CUtensorMap a, b, b16, a1, b1, a2, b2, out, out1, out2; };
template <int MODE>
int launch_gemm(const Maps& m, const GemmArgs& g, long items, cudaStream_t st) {
  auto kern = moe_gemm_k<MODE>;
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = mlb_allow_smem(kern, Smem<MODE>::TOTAL, done);
  if (e != cudaSuccess) return (int)e;
  static const int most = [&] {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(mlb_sm_count() & ~1);
    cfg.blockDim = dim3(Smem<MODE>::THREADS);
    cfg.dynamicSmemBytes = Smem<MODE>::TOTAL;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) { cudaGetLastError(); n = mlb_sm_count() / 2; }
    return std::min(n, mlb_sm_count() / 2);
  }();
  if (items <= 0) return 0;
  return (int)mlb_launch_tmem(true, kern, dim3(2 * (unsigned)std::min<long>(items, most)), dim3(Smem<MODE>::THREADS), (size_t)Smem<MODE>::TOTAL, st, m.a, m.b, m.b16, m.a1, m.b1, m.a2, m.b2, m.out, m.out1, m.out2, g);
}

bool map_tokens(Maps& m, const bf16* base, long rows, int K) {      // [rows, K], K-major
  const uint64_t d[2] = {(uint64_t)K, (uint64_t)rows}, s[1] = {2ull * K};
  const uint32_t b[2] = {64, 128}, b16[2] = {64, 16};
  return mlb_make_tmap_nd(&m.b, base, 2, d, s, b) && mlb_make_tmap_nd(&m.b16, base, 2, d, s, b16);
}
// the same for what leaves an epilogue warp or arrives there: 64 columns of some tokens
bool map_chunk(CUtensorMap* m, const bf16* base, long rows, int cols, uint32_t tokens = 32) {
  const uint64_t d[2] = {(uint64_t)cols, (uint64_t)rows}, s[1] = {2ull * cols};
  const uint32_t b[2] = {64, tokens};
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
int dispatch_bwd(bf16* out, W* dw, const bf16* dout, const bf16* y, const W* weights, const PlanArgs& P, const Sizes& z, long ldo, cudaStream_t st) {
  const long copies = (z.NK + 7) / 8, empty = (z.p.rows + 255) / 256;
  return (int)mlb_launch(moe_dispatch_bwd_k<W>, dim3((unsigned)(copies + empty)), dim3(256), 0, st, out, dw, dout, y, weights, (const int*)P.place, (const int*)P.source,
                         (const int*)(P.start + z.E), ldo, (int)z.NK, z.k, z.C, (int)copies);
}
template <typename W>
int combine(bf16* out, const bf16* y, const W* w, const PlanArgs& P, const Sizes& z, cudaStream_t st) {
  const long slices = (z.C + 255) / 256, blocks = (z.N + 7) / 8;
  if (blocks * slices <= 8L * mlb_sm_count() && slices < 65536)
    return (int)mlb_launch(moe_combine_k<W, 1>, dim3((unsigned)blocks, (unsigned)slices), dim3(256), 0, st, out, y, w, (const int*)P.place, z.N, z.k, z.C);
  return (int)mlb_launch(moe_combine_k<W, 4>, dim3((unsigned)blocks), dim3(256), 0, st, out, y, w, (const int*)P.place, z.N, z.k, z.C);
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
  if (z.p.blocks > 1) MLB_TRY((int)mlb_launch(moe_hist_k, dim3(z.p.blocks), dim3(256), (size_t)4 * E, st, P));
  return (int)mlb_launch(moe_place_k, dim3(z.p.blocks), dim3(32 * plan_warps(E, z.NK)), (size_t)4 * E * (2 + plan_warps(E, z.NK)), st, P);
}
// xs [R, C], gu [R, 2 I] (null: not kept), h [R, I] and y [R, C] are workspace, and what backward needs
MLB_API int mlb_moe_fwd(void* out, void* xs, void* gu, void* h, void* y, const void* x, const void* weights, const void* gate_up, const void* down, const int* plan, long N, long ldx, int k,
                        int E, int C, int I, int wbits, cudaStream_t st) {
  Sizes z;
  MLB_TRY(sizes(z, N, k, E, C, I));
  if (off16({out, xs, gu, h, y, x, gate_up, down, plan}) || ldx % 8 != 0 || (wbits != 16 && wbits != 32)) return -7;
  if (z.NK == 0) return 0;
  const PlanArgs P = plan_args(const_cast<int*>(plan), nullptr, z);
  alignas(64) Maps m = {};
  MLB_TRY(dispatch((bf16*)xs, (const bf16*)x, P, z, ldx, st));
  GemmArgs g = {};
  g.start = P.start, g.order = P.order, g.tiles = P.tiles, g.ntiles = P.ntiles, g.E = E;
  g.out = (bf16*)gu, g.h = (bf16*)h, g.M = 2 * I, g.K = C, g.tiles_m = (2 * I + 255) / 256;
  if (!map_gate_up(&m.a, (const bf16*)gate_up, E, C, I, 4) || !map_tokens(m, (const bf16*)xs, z.p.rows, C) || !map_chunk(&m.b1, g.h, z.p.rows, I) ||
      (g.out != nullptr && !map_chunk(&m.out, g.out, z.p.rows, 2 * I)))
    return -2;
  MLB_TRY(gu != nullptr ? launch_gemm<GATE_UP>(m, g, (long)z.p.max_tiles * g.tiles_m, st) : launch_gemm<H>(m, g, (long)z.p.max_tiles * g.tiles_m, st));
  g.out = (bf16*)y, g.h = nullptr, g.M = C, g.K = I, g.tiles_m = (C + 255) / 256;
  if (!map_down(&m.a, (const bf16*)down, E, C, I, 128) || !map_tokens(m, (const bf16*)h, z.p.rows, I) || !map_chunk(&m.out, g.out, z.p.rows, C)) return -2;
  MLB_TRY(launch_gemm<DOWN>(m, g, (long)z.p.max_tiles * g.tiles_m, st));
  return wbits == 16 ? combine((bf16*)out, (const bf16*)y, (const bf16*)weights, P, z, st) : combine((bf16*)out, (const bf16*)y, (const float*)weights, P, z, st);
}
// ys [R, C], dgu [R, 2 I], dxs [R, C]: workspace.  dx, dgate_up and ddown that are null are not formed
MLB_API int mlb_moe_bwd(void* dx, void* dweights, void* dgate_up, void* ddown, void* ys, void* dgu, void* dxs, const void* dout, const void* xs, const void* gu, const void* h,
                        const void* y, const void* weights, const void* gate_up, const void* down, const int* plan, long N, long ldo, int k, int E, int C, int I, int wbits, cudaStream_t st) {
  Sizes z;
  MLB_TRY(sizes(z, N, k, E, C, I));
  if (off16({dx, dgate_up, ddown, ys, dgu, dxs, dout, xs, gu, h, y, gate_up, down, plan}) || ldo % 8 != 0 || (wbits != 16 && wbits != 32)) return -7;
  if (z.NK == 0) return 0;
  const PlanArgs P = plan_args(const_cast<int*>(plan), nullptr, z);
  const long R = z.p.rows;
  alignas(64) Maps m = {};
  MLB_TRY(wbits == 16 ? dispatch_bwd((bf16*)ys, (bf16*)dweights, (const bf16*)dout, (const bf16*)y, (const bf16*)weights, P, z, ldo, st)
                      : dispatch_bwd((bf16*)ys, (float*)dweights, (const bf16*)dout, (const bf16*)y, (const float*)weights, P, z, ldo, st));
  if (dx == nullptr && dgate_up == nullptr && ddown == nullptr) return 0;
  GemmArgs g = {};
  g.start = P.start, g.order = P.order, g.tiles = P.tiles, g.ntiles = P.ntiles, g.E = E;
  g.out = (bf16*)dgu, g.M = I, g.K = C, g.tiles_m = (I + 255) / 256;
  if (dx != nullptr || dgate_up != nullptr) {
    constexpr int chunk = Smem<DOWN_T>::CHUNK;
    if (!map_down(&m.a, (const bf16*)down, E, C, I, 64) || !map_tokens(m, (const bf16*)ys, R, C) || !map_chunk(&m.a1, (const bf16*)gu, R, 2 * I, chunk) ||
        !map_chunk(&m.out, g.out, R, 2 * I, chunk))
      return -2;
    MLB_TRY(launch_gemm<DOWN_T>(m, g, (long)z.p.max_tiles * g.tiles_m, st));
  }
  g.out = (bf16*)dxs, g.M = C, g.K = 2 * I, g.tiles_m = dx != nullptr ? (C + 255) / 256 : 0;
  g.C = C, g.I = I;
  g.per_gate_up = dgate_up != nullptr ? ((2 * I + 255) / 256) * ((C + 255) / 256) : 0;
  g.per_down = ddown != nullptr ? ((C + 255) / 256) * ((I + 255) / 256) : 0;
  if (!map_gate_up(&m.a, (const bf16*)gate_up, E, C, I, 2) || !map_tokens(m, (const bf16*)dgu, R, 2 * I) || !map_rows(&m.a1, (const bf16*)dgu, R, 2 * I) ||
      !map_rows(&m.b1, (const bf16*)xs, R, C) || !map_rows(&m.a2, (const bf16*)ys, R, C) || !map_rows(&m.b2, (const bf16*)h, R, I) || (dx != nullptr && !map_chunk(&m.out, g.out, R, C)) ||
      (dgate_up != nullptr && !map_gate_up(&m.out1, (const bf16*)dgate_up, E, C, I, 1)) || (ddown != nullptr && !map_down(&m.out2, (const bf16*)ddown, E, C, I, 32)))
    return -2;
  MLB_TRY(launch_gemm<BACK>(m, g, (long)E * (g.per_gate_up + g.per_down) + (long)z.p.max_tiles * g.tiles_m, st));
  return dx != nullptr ? combine((bf16*)dx, (const bf16*)dxs, (const float*)nullptr, P, z, st) : 0;
}
// floats of the workspace of the form for few tokens; 0: the sizes take the other form
MLB_API long mlb_moe_few_floats(long N, int k, int E, int C, int I) {
  Sizes z;
  if (sizes(z, N, k, E, C, I) != 0 || N < 1 || N > FEW_TOKENS || z.NK > FEW_COPIES) return 0;
  return z.NK * I / 2;      // (h)
}
MLB_API int mlb_moe_few(void* out, const void* x, const void* weights, const int* idx, const void* gate_up, const void* down, float* part, long N, long ldx, int k, int E, int C, int I,
                        int wbits, cudaStream_t st) {
  if (mlb_moe_few_floats(N, k, E, C, I) == 0 || off16({out, x, gate_up, down, part}) || ldx % 8 != 0 || (wbits != 16 && wbits != 32)) return -7;
  const FewArgs g = {(bf16*)out, (bf16*)part, (const bf16*)x, weights, idx, ldx, (int)N, k, E, C, I, wbits, 1};
  const uint64_t c = C, i = I, n = E;
  const uint64_t da[5] = {c, 8, 2, i / 8, n}, sa[4] = {2 * c, 2 * i * c, 16 * c, 4 * i * c}, db[3] = {i, c, n}, sb[2] = {2 * i, 2 * c * i};
  const uint32_t ba[5] = {64, 8, 2, 1, 1}, bb[3] = {64, 16, 1};
  alignas(64) CUtensorMap a, b;
  if (!mlb_make_tmap_nd(&a, gate_up, 5, da, sa, ba) || !mlb_make_tmap_nd(&b, down, 3, db, sb, bb)) return -2;
  MLB_TRY(launch_few_h(a, g, st));
  // Blocks for most SMs, whole call, us, by 1, 2 and 4 blocks to 16 columns: 2048 columns of 6 experts 26.6, 31.1, 45.5; 768 of 8 tokens' 8 experts 23.8, 20.6, 24.0
  int split = 1;
  while (split < 4 && C / 16 * split * 2 <= mlb_sm_count()) split *= 2;
  return split == 1 ? launch_few_out<1>(b, g, st) : split == 2 ? launch_few_out<2>(b, g, st) : launch_few_out<4>(b, g, st);
}
