// What a generation step decides on the GPU: which cache pages and slots the new tokens get, which continuations of the beams are kept, and the beams' tables,
// histories and half-filled pages in the order of their parents.  Nothing here is read back by the host.
#include "common.cuh"

namespace {

MLB_DEFINE_ERROR_WORD(beam)

// ------------------------------------------------------------------ block tables and slots
// Request r holds lens[r] tokens and gets news[r] more.  It needs ceil((lens + news) / page) - ceil(lens / page) pages, which it gets from the top of the free
// stack if the needs of the requests up to it do not pass what lies there.  Every thread block adds up all requests for itself (12 bytes each: cheaper than
// another launch or a wait for one block that does it) and then writes its share of the slots; the thread that has a page's first token writes the page into
// the table.  What may be an input too (new_lens, left) is written by the block that comes last.
constexpr int TAB_THREADS = 256, TAB_MAX_B = 4096, TAB_MAX_ROWS = 1 << 22;
struct TableArgs {
  int *table, *slots, *pos, *starts, *new_lens, *left, *ticket;
  const int *lens, *news, *stack, *n_free;
  int B, width, page, rows, stack_size;
};
struct Two { int a, b; };
__device__ __forceinline__ Two block_scan(Two v, Two* warps, Two& total) {      // inclusive sums over the thread block
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, v.a, o), b = __shfl_up_sync(0xffffffffu, v.b, o);
    if (lane >= o) v.a += a, v.b += b;
  }
  __syncthreads();
  if (lane == 31) warps[w] = v;
  __syncthreads();
  total = {0, 0};
  for (int k = 0; k < TAB_THREADS / 32; k++) {
    if (k == w) v.a += total.a, v.b += total.b;
    total.a += warps[k].a, total.b += warps[k].b;
  }
  return v;
}
__global__ void __launch_bounds__(TAB_THREADS) block_tables_k(const TableArgs A) {
  mlb_pdl_sync();
  extern __shared__ int smem[];
  int *start = smem, *first = smem + A.B + 1;      // first[r]: pages taken by the requests before, -1 where r gets nothing
  __shared__ Two warps[TAB_THREADS / 32];
  __shared__ int most, last;
  const int tid = threadIdx.x;
  if (tid == 0) most = 0;
  int n_free = *A.n_free;
  if (n_free < 0 || n_free > A.stack_size) {
    if (tid == 0 && blockIdx.x == 0) mlb_set_error(MLB_ERR_BOUNDS, 0xB1);
    n_free = max(0, min(n_free, A.stack_size));
  }
  Two done = {0, 0};
  int taken = 0;
  for (int r0 = 0; r0 < A.B; r0 += TAB_THREADS) {
    const int r = r0 + tid;
    int len = 0, add = 0, need = 0;
    bool fits = false;
    if (r < A.B) {
      len = A.lens[r], add = A.news[r];
      if (len < 0 || add < 0 || add > A.rows) {
        if (blockIdx.x == 0) mlb_set_error(MLB_ERR_BOUNDS, 0xB1);
        add = 0;
      } else if ((long)len + add <= (long)A.width * A.page) {
        fits = true;
        need = (len + add + A.page - 1) / A.page - (len + A.page - 1) / A.page;
      }
    }
    Two total;
    const Two upto = block_scan({need, add}, warps, total);
    if (r < A.B) {
      const int pages = done.a + upto.a, rows = done.b + upto.b;
      if (rows > A.rows && blockIdx.x == 0) mlb_set_error(MLB_ERR_BOUNDS, 0xB2);
      const bool got = fits && pages <= n_free && rows <= A.rows;
      start[r] = rows - add;
      first[r] = got ? pages - need : -1;
      if (got) taken = max(taken, pages);
    }
    done.a += total.a, done.b = min(done.b + total.b, A.rows + 1);      // (past the last place nothing fits any more: no sum overflows)
  }
  if (tid == 0) start[A.B] = done.b;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) taken = max(taken, __shfl_xor_sync(0xffffffffu, taken, o));
  __syncthreads();
  if ((tid & 31) == 0) atomicMax(&most, taken);
  __syncthreads();
  taken = most;
  for (int row = blockIdx.x * TAB_THREADS + tid; row < A.rows; row += gridDim.x * TAB_THREADS) {
    int slot = -1, at = 0;
    if (row < done.b) {
      int r = 0, hi = A.B;      // the last request that starts at or before this row
      while (hi - r > 1) {
        const int mid = (r + hi) >> 1;
        if (start[mid] <= row) r = mid;
        else hi = mid;
      }
      if (first[r] >= 0) {
        const int len = A.lens[r], has = (len + A.page - 1) / A.page;
        at = len + row - start[r];
        const int p = at / A.page, off = at - p * A.page;
        int id;
        if (p < has) {
          id = A.table[(long)r * A.width + p];
        } else {
          id = A.stack[n_free - 1 - (first[r] + p - has)];
          if (off == 0) A.table[(long)r * A.width + p] = id;
        }
        slot = id < 0 ? -1 : id * A.page + off;
      }
    }
    A.slots[row] = slot;
    A.pos[row] = at;
  }
  if (blockIdx.x == 0)
    for (int r = tid; r <= A.B; r += TAB_THREADS) A.starts[r] = start[r];
  if (gridDim.x > 1) {
    __threadfence();
    __syncthreads();
    if (tid == 0) last = atomicAdd(A.ticket, 1) == (int)gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    if (tid == 0) *A.ticket = 0;
  } else {
    __syncthreads();
  }
  for (int r = tid; r < A.B; r += TAB_THREADS) {
    const int len = A.lens[r];
    A.new_lens[r] = first[r] >= 0 ? len + start[r + 1] - start[r] : len;
  }
  if (tid == 0) *A.left = n_free - taken;
}

// ------------------------------------------------------------------ beam selection
// score(k, v) = prev[k] + (z[k, v] - lse[k]), lse[k] = log sum_v exp z[k, v]; of the K V scores of a request the K largest, equal ones by the lowest k V + v.  A
// beam that has ended goes on as itself: its one continuation is (eos, prev[k]).  Within a row the order of the scores is that of the logits, so a row's K
// best can be found before its lse is known, in the one pass that reads it.
//
// Bound by the logits' bytes, then by an exponential for each.  A row is cut into pieces of at most 8192 logits (so many that the machine is filled), a thread
// block keeps its piece in registers.  The K-th largest of 8 (K > 8: 32) maxima of parts of the piece is a bound below which nothing is among its K largest: one comparison beside
// the exponential leaves a handful of candidates, which one warp sorts out.  Too many of them (logits all alike) take K rounds over the registers
// instead.  The request's last thread block merges the pieces' sorted lists.
constexpr int SEL_THREADS = 256, SEL_WARPS = SEL_THREADS / 32, SEL_E = 32, SEL_PIECE = SEL_THREADS * SEL_E, SEL_MAX_K = 32, SEL_CAND = 256, SEL_LISTS = 8192, SEL_HELD = 2048;
typedef unsigned long long u64;
struct SelectArgs {
  float* scores;
  int *tokens, *parents, *done_out;
  const void* logits;
  const float* prev;
  const int* done;
  float2* stats;      // [rows][pieces]: maximum, sum of exponentials
  float* values;      // [rows][pieces][K], largest first
  int* ids;           // [rows][pieces][K], -1: no more
  int* ticket;
  long stride;
  int K, V, eos, pieces, piece;
};
// Order of candidates as whole numbers: larger value first, then the lower index
__device__ __forceinline__ uint32_t ordered(float x) {
  x = x == 0.f ? 0.f : x;      // (-0 is 0)
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u); }
__device__ __forceinline__ u64 rank_of(float x, uint32_t at) { return (u64)ordered(x) << 32 | (uint32_t)~at; }
__device__ __forceinline__ u64 warp_best(u64 k) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 block_best(u64 k, u64* red) {
  k = warp_best(k);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = k;
  __syncthreads();
  k = red[0];
#pragma unroll
  for (int w = 1; w < SEL_WARPS; w++) k = max(k, red[w]);
  return k;
}
__device__ __forceinline__ float logit(float x) { return x != x ? -INFINITY : x; }

template <typename T, bool VEC>
__global__ void __launch_bounds__(SEL_THREADS) beam_select_k(const SelectArgs A) {
  mlb_pdl_sync();
  __shared__ float smax[32], ssum[SEL_WARPS];
  __shared__ u64 cand[SEL_CAND], red[SEL_WARPS];
  __shared__ int n_cand, last;
  __shared__ float prev[SEL_MAX_K], lse[SEL_MAX_K];
  __shared__ int ended[SEL_MAX_K];
  __shared__ uint8_t head[SEL_LISTS];
  __shared__ u64 held[SEL_HELD];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, K = A.K, V = A.V;
  const int row = blockIdx.y, req = row / K;
  const long list = (long)row * A.pieces + blockIdx.x;
  if (!A.done[row]) {
    const int begin = blockIdx.x * A.piece, n = min(A.piece, V - begin);
    const T* z = reinterpret_cast<const T*>(A.logits) + row * A.stride + begin;
    float x[SEL_E];
    auto at = [&](int k) { return VEC ? (k / 8 * SEL_THREADS + tid) * 8 + k % 8 : k * SEL_THREADS + tid; };      // place of element k in the piece
#pragma unroll
    for (int g = 0; g < SEL_E / 8; g++) {
#pragma unroll
      for (int k = 0; k < 8; k++) x[8 * g + k] = -INFINITY;
      if (g * SEL_THREADS * 8 < n) {
        if constexpr (VEC) {
          const int p = at(8 * g);
          if (p + 8 <= n) {
            if constexpr (sizeof(T) == 2) {
              const uint4 w = *reinterpret_cast<const uint4*>(z + p);
              const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int k = 0; k < 4; k++) x[8 * g + 2 * k] = __uint_as_float(u[k] << 16), x[8 * g + 2 * k + 1] = __uint_as_float(u[k] & 0xFFFF0000u);
            } else {
#pragma unroll
              for (int k = 0; k < 2; k++) {
                const float4 w = *reinterpret_cast<const float4*>(z + p + 4 * k);
                x[8 * g + 4 * k] = w.x, x[8 * g + 4 * k + 1] = w.y, x[8 * g + 4 * k + 2] = w.z, x[8 * g + 4 * k + 3] = w.w;
              }
            }
          } else {
#pragma unroll
            for (int k = 0; k < 8; k++)
              if (p + k < n) x[8 * g + k] = (float)z[p + k];
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; k++)
            if (at(8 * g + k) < n) x[8 * g + k] = (float)z[at(8 * g + k)];
        }
      }
    }
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < SEL_E; k++) x[k] = logit(x[k]), m = fmaxf(m, x[k]);
    // maxima of 32 parts of the piece: a part is 8 threads
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((lane & 7) == 0) smax[warp * 4 + (lane >> 3)] = m;
    if (tid == 0) n_cand = 0;
    __syncthreads();
    m = smax[lane];
    int better = 0;
#pragma unroll
    for (int o = 1; o < 32; o++) {
      const float y = __shfl_xor_sync(0xffffffffu, m, o);
      better += y > m || (y == m && (lane ^ o) < lane);
    }
    const float bound = __shfl_sync(0xffffffffu, m, __ffs(__ballot_sync(0xffffffffu, better == K - 1)) - 1);
    m = warp_max(m);
    const float mm = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < SEL_E; k++) {
      s += exp2f((x[k] - mm) * 1.44269504088896f);
      if (x[k] >= bound && at(k) < n) {
        const int c = atomicAdd(&n_cand, 1);
        if (c < SEL_CAND) cand[c] = rank_of(x[k], begin + at(k));
      }
    }
    s = warp_sum(s);
    if (lane == 0) ssum[warp] = s;
    __syncthreads();
    if (tid == 0) {
      s = 0.f;
      for (int w = 0; w < SEL_WARPS; w++) s += ssum[w];
      A.stats[list] = make_float2(m, s);
    }
    if (n_cand <= SEL_CAND) {
      if (warp == 0) {
        u64 mine[SEL_CAND / 32];
#pragma unroll
        for (int c = 0; c < SEL_CAND / 32; c++) mine[c] = c * 32 + lane < n_cand ? cand[c * 32 + lane] : 0ull;
        for (int k = 0; k < K; k++) {
          u64 best = 0;
#pragma unroll
          for (int c = 0; c < SEL_CAND / 32; c++) best = max(best, mine[c]);
          best = warp_best(best);
#pragma unroll
          for (int c = 0; c < SEL_CAND / 32; c++)
            if (mine[c] == best) mine[c] = 0;
          if (lane == 0) {
            A.values[list * K + k] = best ? unordered((uint32_t)(best >> 32)) : -INFINITY;
            A.ids[list * K + k] = best ? (int)~(uint32_t)best : -1;
          }
        }
      }
    } else {
      u64 prior = ~0ull;
      for (int k = 0; k < K; k++) {
        u64 best = 0;
#pragma unroll
        for (int c = 0; c < SEL_E; c++) {
          const u64 r = at(c) < n ? rank_of(x[c], begin + at(c)) : 0ull;
          if (r < prior) best = max(best, r);
        }
        prior = best = block_best(best, red);
        if (tid == 0) {
          A.values[list * K + k] = best ? unordered((uint32_t)(best >> 32)) : -INFINITY;
          A.ids[list * K + k] = best ? (int)~(uint32_t)best : -1;
        }
      }
    }
  }
  // ---- the request's last thread block merges
  __threadfence();
  __syncthreads();
  if (tid == 0) last = atomicAdd(A.ticket + req, 1) == A.pieces * K - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  if (tid == 0) A.ticket[req] = 0;
  if (tid < K) prev[tid] = A.prev[req * K + tid], ended[tid] = A.done[req * K + tid] != 0;
  for (int k = warp; k < K; k += SEL_WARPS) {
    if (A.done[req * K + k]) continue;
    const float2* st = A.stats + (long)(req * K + k) * A.pieces;
    float m = -INFINITY;
    for (int p = lane; p < A.pieces; p += 32) m = fmaxf(m, __ldcg(st + p).x);
    m = warp_max(m);
    float s = 0.f;
    for (int p = lane; p < A.pieces; p += 32) {
      const float2 v = __ldcg(st + p);
      s += v.x == m ? v.y : v.y * exp2f((v.x - m) * 1.44269504088896f);
    }
    s = warp_sum(s);
    if (lane == 0) lse[k] = m + (float)log((double)s);
  }
  const int lists = K * A.pieces;
  for (int l = tid; l < lists; l += SEL_THREADS) head[l] = 0;
  __syncthreads();
  // a beam of no continuation: it was nothing, or its logits have no logarithm of a sum
  auto dead = [&](int k) { return !ended[k] && !(prev[k] > -INFINITY && fabsf(lse[k]) < INFINITY); };
  auto rank = [&](int l, int h) -> u64 {      // entry h of list l, 0: no more
    const int k = l / A.pieces, p = l % A.pieces;
    float x;
    int tok;
    if (ended[k] || dead(k)) {
      if (p != 0) return 0;
      if (ended[k] && A.eos >= 0 && A.eos < V) {
        tok = h == 0 ? A.eos : h - 1 < A.eos ? h - 1 : h;
        x = h == 0 ? prev[k] : -INFINITY;
        if (x != x) x = -INFINITY;
      } else {
        tok = h, x = -INFINITY;
      }
      if (tok >= V) return 0;
    } else {
      const long a = ((long)(req * K + k) * A.pieces + p) * K + h;
      tok = __ldcg(A.ids + a);
      if (tok < 0) return 0;
      x = __fadd_rn(prev[k], __fsub_rn(__ldcg(A.values + a), lse[k]));
      if (x != x) x = -INFINITY;
    }
    return rank_of(x, (uint32_t)k * (uint32_t)V + (uint32_t)tok);
  };
  const bool keep = lists * K <= SEL_HELD;
  if (keep)
    for (int e = tid; e < lists * K; e += SEL_THREADS) held[e] = rank(e / K, e % K);
  __syncthreads();
  u64 best = 0;      // the best head of this thread's lists, and whose it is
  int mine = -1;
  auto choose = [&] {
    best = 0;
    for (int l = tid; l < lists; l += SEL_THREADS) {
      const int h = head[l];
      const u64 r = h >= K ? 0ull : keep ? held[l * K + h] : rank(l, h);
      if (r > best) best = r, mine = l;
    }
  };
  choose();
  for (int k = 0; k < K; k++) {
    const u64 top = block_best(best, red);
    if (best == top && top != 0) {
      const uint32_t flat = ~(uint32_t)top;
      const int from = (int)(flat / (uint32_t)V), tok = (int)(flat % (uint32_t)V), o = req * K + k;
      A.scores[o] = unordered((uint32_t)(top >> 32));
      A.tokens[o] = tok, A.parents[o] = from, A.done_out[o] = ended[from] || tok == A.eos;
      head[mine]++;
      choose();
    }
    if (top == 0 && tid == 0) {      // fewer continuations than beams (V < K)
      const int o = req * K + k;
      A.scores[o] = -INFINITY, A.tokens[o] = A.eos, A.parents[o] = 0, A.done_out[o] = 1;
    }
  }
}

// Logits of a piece, a multiple of 8: at least a wave of thread blocks (4 an SM) where the rows give as much, 1024 logits and more each
int select_piece(int rows, int V) {
  const long least = (V + SEL_PIECE - 1) / SEL_PIECE, most = (V + 1023) / 1024, want = (4L * mlb_sm_count() + rows - 1) / rows;
  const long n = want < least ? least : want > most ? most : want;
  return (int)((V + n - 1) / n + 7) / 8 * 8;
}

// ------------------------------------------------------------------ beams in the order of their parents
// Row b K + k continues row b K + parents[b, k].  Full pages are shared: their numbers are copied from the parent's table.  The page that is being filled belongs to one
// row alone, so a row that continues another one gets that one's tokens copied to its spare page, and the page it had is its spare from then on: nothing
// that is read is written, whatever the order of the rows.  Bound by the copied bytes.
struct OrderArgs {
  uint8_t* pages;
  int *table_out, *spare_out, *hist_out;
  const int *table, *spare, *lens, *hist, *parents, *tokens;
  long n_pages;
  int K, Hkv, page, block_vecs, width, T;      // block_vecs: 16-byte words of a block of 16 tokens
};
constexpr int ORDER_THREADS = 256;
__global__ void __launch_bounds__(ORDER_THREADS) beam_reorder_k(const OrderArgs A) {
  mlb_pdl_sync();
  const int row = blockIdx.x, tid = threadIdx.x;
  int parent = A.parents[row];
  if (parent < 0 || parent >= A.K) {
    if (tid == 0 && blockIdx.y == 0) mlb_set_error(MLB_ERR_BOUNDS, 0xB3);
    parent = row % A.K;
  }
  const int src = row / A.K * A.K + parent;
  const int len = min(max(A.lens[row], 0), A.width * A.page), full = len / A.page, rest = len - full * A.page;
  const bool moved = rest > 0 && src != row;
  if (blockIdx.y == 0) {
    for (int p = tid; p < A.width; p += ORDER_THREADS)
      A.table_out[(long)row * A.width + p] = moved && p == full ? A.spare[row] : A.table[(long)(p < full ? src : row) * A.width + p];
    if (tid == 0) A.spare_out[row] = moved ? A.table[(long)row * A.width + full] : A.spare[row];
    for (int t = tid; t < min(len, A.T); t += ORDER_THREADS) A.hist_out[(long)row * A.T + t] = A.hist[(long)src * A.T + t];
    if (tid == 0 && len < A.T) A.hist_out[(long)row * A.T + len] = A.tokens[row];
    return;
  }
  if (!moved) return;
  const int from = A.table[(long)src * A.width + full], to = A.spare[row];
  if (from < 0 || from >= A.n_pages || to < 0 || to >= A.n_pages) {
    if (tid == 0) mlb_set_error(MLB_ERR_BOUNDS, 0xB4);
    return;
  }
  const int blocks = A.page / 16, each = (rest + 15) / 16 * A.block_vecs;
  const long base = (long)(blockIdx.y - 1) * A.n_pages, head = (long)blocks * A.block_vecs;
  const uint4* f = reinterpret_cast<const uint4*>(A.pages) + (base + from) * A.Hkv * head;
  uint4* t = reinterpret_cast<uint4*>(A.pages) + (base + to) * A.Hkv * head;
  for (int v = tid; v < A.Hkv * each; v += ORDER_THREADS) {
    const long a = v / each * head + v % each;
    t[a] = f[a];
  }
}

}  // namespace

MLB_API int mlb_block_tables(int* table, int* slots, int* pos, int* starts, int* new_lens, int* left, int* ticket, const int* lens, const int* news,
                             const int* stack, const int* n_free, int B, int width, int page, int rows, int stack_size, cudaStream_t st) {
  if (B < 1 || B > TAB_MAX_B || page < 1 || width < 1 || rows < 0 || rows > TAB_MAX_ROWS || (long)B * width >= 1L << 31) return -7;
  const int want = (rows + TAB_THREADS - 1) / TAB_THREADS, most = 2 * mlb_sm_count();
  const TableArgs a{table, slots, pos, starts, new_lens, left, ticket, lens, news, stack, n_free, B, width, page, rows, stack_size};
  return (int)mlb_launch(block_tables_k, dim3(want < 1 ? 1 : want < most ? want : most), dim3(TAB_THREADS), (2 * B + 1) * sizeof(int), st, a);
}

// Pieces that a row of V logits is cut into, and (-7) nothing for what the kernel does not take
MLB_API int mlb_beam_select_pieces(int rows, int K, int V) {
  if (K < 1 || K > SEL_MAX_K || V < 1 || rows < 1 || rows > 65535 || (long)K * V >= 0xFFFFFFFFL) return -7;
  const int piece = select_piece(rows, V), pieces = (V + piece - 1) / piece;
  return (long)pieces * K > SEL_LISTS ? -7 : pieces;
}
// bits: 16 (bf16) or 32 (fp32) logits, rows `stride` elements apart
MLB_API int mlb_beam_select(float* scores, int* tokens, int* parents, int* done_out, const void* logits, const float* prev, const int* done, float* stats,
                            float* values, int* ids, int* ticket, int rows, int K, int V, long stride, int eos, int bits, cudaStream_t st) {
  const int pieces = mlb_beam_select_pieces(rows, K, V);
  if (pieces < 0 || rows % K != 0) return -7;
  const SelectArgs a{scores, tokens, parents, done_out, logits, prev, done, (float2*)stats, values, ids, ticket, stride, K, V, eos, pieces, select_piece(rows, V)};
  const bool vec = ((uintptr_t)logits & 15) == 0 && stride * (bits / 8) % 16 == 0;
  const dim3 grid(pieces, rows), block(SEL_THREADS);
  if (bits == 16) return (int)(vec ? mlb_launch(beam_select_k<bf16, true>, grid, block, 0, st, a) : mlb_launch(beam_select_k<bf16, false>, grid, block, 0, st, a));
  return (int)(vec ? mlb_launch(beam_select_k<float, true>, grid, block, 0, st, a) : mlb_launch(beam_select_k<float, false>, grid, block, 0, st, a));
}

// pages null: no cache to copy in; block_bytes of 16 tokens of a head
MLB_API int mlb_beam_reorder(uint8_t* pages, int* table_out, int* spare_out, int* hist_out, const int* table, const int* spare, const int* lens, const int* hist,
                             const int* parents, const int* tokens, int layers, long n_pages, int Hkv, int page, int block_bytes, int B, int K, int width, int T,
                             cudaStream_t st) {
  if (page < 16 || page % 16 != 0 || block_bytes % 16 != 0 || K < 1 || width < 1 || layers > 65534) return -7;
  const OrderArgs a{pages, table_out, spare_out, hist_out, table, spare, lens, hist, parents, tokens, n_pages, K, Hkv, page, block_bytes / 16, width, T};
  return (int)mlb_launch(beam_reorder_k, dim3(B * K, pages ? layers + 1 : 1), dim3(ORDER_THREADS), 0, st, a);
}
