// What a generation step decides on the GPU: which cache pages and slots the new tokens get, which continuations of the beams are kept, and the beams' tables,
// histories and half-filled pages in the order of their parents.  Nothing here is read back by the host.
#include <type_traits>

#include "tc.cuh"

namespace {

MLB_DEFINE_ERROR_WORD(beam)

// ------------------------------------------------------------------ block tables and slots
// Request r holds lens[r] tokens and gets news[r] more.  It needs ceil((lens + news) / page) - ceil(lens / page) pages, which it gets from the top of the free
// stack if the needs of the requests up to it do not pass what lies there.  Every thread block adds up all requests for itself (12 bytes each: cheaper than
// another launch or a wait for one block that does it) and then writes its share of the slots; the thread that has a page's first token writes the page into
// the table.  What may be an input too (new_lens, left) is written by the block that comes last.  Bound by latency: 64 requests of one token 2.9 us, 300 requests
// of 154 thousand tokens 5.7 (of 0.2 for their bytes; 6.3 with sums over 256 requests at a time).
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
  // a thread has `per` requests, one behind the other: their needs (-1: too long for the table's row) and new tokens, then the sums over those before
  const int per = (A.B + TAB_THREADS - 1) / TAB_THREADS, r0 = tid * per, r1 = min(r0 + per, A.B);
  Two own = {0, 0}, done;
#pragma unroll 1
  for (int r = r0; r < r1; r++) {
    const int len = A.lens[r];
    int add = A.news[r], need = -1;
    if (len < 0 || add < 0 || add > A.rows) {
      if (blockIdx.x == 0) mlb_set_error(MLB_ERR_BOUNDS, 0xB1);
      add = 0;
    } else if ((long)len + add <= (long)A.width * A.page) {
      need = ((unsigned)len + add + A.page - 1) / A.page - ((unsigned)len + A.page - 1) / A.page;
    }
    start[r] = add, first[r] = need;
    own.a += max(need, 0), own.b = min(own.b + add, A.rows + 1);      // (past the last place nothing fits any more: no sum overflows)
  }
  const Two upto = block_scan(own, warps, done);
  int pages = upto.a - own.a, rows = upto.b - own.b, taken = 0;
#pragma unroll 1
  for (int r = r0; r < r1; r++) {
    const int add = start[r], need = first[r];
    start[r] = rows;
    pages += max(need, 0), rows = min(rows + add, A.rows + 1);
    const bool got = need >= 0 && pages <= n_free && rows <= A.rows;
    first[r] = got ? pages - need : -1;
    if (got) taken = max(taken, pages);
    if (rows > A.rows && blockIdx.x == 0) mlb_set_error(MLB_ERR_BOUNDS, 0xB2);
  }
  done.b = min(done.b, A.rows + 1);
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
        const int len = A.lens[r], has = ((unsigned)len + A.page - 1) / A.page;
        at = len + row - start[r];
        const int p = at / A.page, off = at - p * A.page;
        int id;
        if (p < has) {
          id = A.table[(long)r * A.width + p];
        } else {
          id = A.stack[n_free - 1 - (first[r] + p - has)];
          if (off == 0) A.table[(long)r * A.width + p] = id;
        }
        slot = id < 0 ? -1 : (int)min((long)id * A.page + off, 0x7FFFFFFFL);      // (the last number is no slot of any pool)
      }
    }
    A.slots[row] = slot;
    A.pos[row] = at;
  }
  if (blockIdx.x == 0)
    for (int r = tid; r <= A.B; r += TAB_THREADS) A.starts[r] = start[r];
  if (gridDim.x > 1) {
    __syncthreads();
    if (tid == 0) last = mlb_count_block(A.ticket) == (int)gridDim.x - 1;
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
// beam that has ended goes on as itself: its one continuation is (eos, prev[k]).  Within a row a larger logit has no smaller score, so a row's K
// best can be found before its lse is known, in the one pass that reads it - but for logits that differ and have equal scores after both roundings, of which the lowest
// index counts and not the largest logit.  So a piece also gives a limit that no logit passes which it has left out.  Only where the limit's score is the K-th best of all
// can something of a lower index have been left out; then a warp looks closer (some 2 us: 32 beams of bf16 logits, of which many are alike, in a search's first step),
// and if need be goes over the request's rows in order (1 x 4 beams of 50304 with 40 equal scores a row 75 us).
//
// Bound by the logits' bytes, then by an exponential for each.  A row is cut into as many pieces as fill the machine once, and a thread block fetches up to 32 KB of
// its piece at a time into shared memory, by one bulk copy: many bytes on their way, and loops that are short (they run a few times only, so that instructions
// fetched for the first time are a good part of a call).  The (K + 1)-th largest of the maxima of 8 to 32 parts of what came first is a bound below which
// nothing is among the piece's K + 1 largest: one comparison for 8 logits leaves some tens of candidates.  Where they become many, those behind the (K + 1)-th go and it
// is the bound from then on.  A candidate's place is the number of those before it.  More candidates at a time than there is room for (logits all alike) are forgotten:
// then K rounds over the piece find its K largest.  The request's last thread block finds its K best among the pieces' lists in the same way,
// the bound being of its threads' best.
// 32 x 8 beams of 50304 bf16 logits, a quarter of them ended: 15.5 us (1.7 TB/s), of which fetching and the maximum 6.2, the exponentials 1, candidates and their
// bound 2.6, the counters 1.9, the merge 3.4.  1 x 4 beams: 7.1 us (2.3, then 1 for the counters, 3.4 for the merge): latencies one behind the other.  fp32 logits: 1 x 4
// beams 7.2, 32 x 8 with none ended 25.8 (bf16: 17.9), 8 x 32 44.6 (33.8).
constexpr int SEL_THREADS = 256, SEL_WARPS = SEL_THREADS / 32, SEL_CHUNK_BYTES = 32768, SEL_MAX_K = 32, SEL_CAND = 512, SEL_HELD = 1024;
// Thread blocks that an SM has registers for (shared memory leaves room for five whose fetches are whole 32 KB: counted as six, 256 rows of 50304 logits are four pieces a
// row, 1024 blocks, of which 740 are resident at once); the smallest piece
constexpr int SEL_PER_SM = 6, SEL_LEAST = 4096;
typedef unsigned long long u64;
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
struct SelectArgs {
  float* scores;
  int *tokens, *parents, *done_out;
  const void* logits;
  const float* prev;
  const int* done;
  float2* stats;      // [rows][pieces]: maximum, sum of exponentials
  float* values;      // [rows][pieces][L + 1]: the K best and maybe others, and last what no logit passes that is not among them
  int* ids;           // [rows][pieces][L + 1], -1: none
  int* ticket;
  long stride;
  int K, L, V, eos, pieces, piece;
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

// 8 neighbouring logits in shared memory, -inf for NaN, and the largest
template <typename T> struct Eight;
template <> struct Eight<bf16> {
  uint32_t w[4];
  __device__ __forceinline__ float load(const bf16* p) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    bf162 m;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const uint32_t ninf = 0xFF80FF80u;
      const bf162 x = __hmax2(*reinterpret_cast<bf162*>(&w[k]), *reinterpret_cast<const bf162*>(&ninf));
      w[k] = *reinterpret_cast<const uint32_t*>(&x);
      m = k ? __hmax2(m, x) : x;
    }
    return fmaxf(__low2float(m), __high2float(m));
  }
  __device__ __forceinline__ float get(int k) const { return __uint_as_float(k % 2 ? w[k / 2] & 0xFFFF0000u : w[k / 2] << 16); }
};
template <> struct Eight<float> {
  float x[8];
  __device__ __forceinline__ float load(const float* p) {
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + k);
      x[k] = fmaxf(v.x, -INFINITY), x[k + 1] = fmaxf(v.y, -INFINITY), x[k + 2] = fmaxf(v.z, -INFINITY), x[k + 3] = fmaxf(v.w, -INFINITY);
      m = fmaxf(m, fmaxf(fmaxf(x[k], x[k + 1]), fmaxf(x[k + 2], x[k + 3])));
    }
    return m;
  }
  __device__ __forceinline__ float get(int k) const { return x[k]; }
};
// Number of the n keys at `keys` that come before `mine`; keys are distinct
__device__ __forceinline__ int place_of(u64 mine, const u64* keys, int n) {
  int before = 0;
#pragma unroll 8
  for (int c = 0; c < n; c++) before += keys[c] > mine;
  return before;
}

// Parts of a thread block whose maxima bound its K largest: warps, halves or quarters of them
__device__ __forceinline__ int parts_for(int K) { return K <= SEL_WARPS / 2 ? SEL_WARPS : K <= SEL_WARPS ? 2 * SEL_WARPS : 4 * SEL_WARPS; }
// The K-th largest of the maxima of the parts' values: K of these are not below it.  tops: 32 values of shared memory
template <typename X, typename Max>
__device__ __forceinline__ X kth_of_parts(X m, int K, int parts, X* tops, Max larger) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, each = SEL_THREADS / parts;      // 8, 16 or 32 threads
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) m = larger(m, __shfl_xor_sync(0xffffffffu, m, o));
  for (int o = 8; o < each; o <<= 1) m = larger(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane % each == 0) tops[(warp * 32 + lane) / each] = m;
  __syncthreads();
  m = tops[lane % parts];
  int better = 0;
#pragma unroll 8
  for (int o = 0; o < parts; o++) {
    const X y = tops[o];
    better += y > m || (y == m && o < lane);
  }
  return __shfl_sync(0xffffffffu, m, __ffs(__ballot_sync(0xffffffffu, better == K - 1)) - 1);
}
// Natural logarithm of a normal number, off by 2^-22 and a rounding: the exponent's part apart from that of a number of 1 ... 2, ln 2 in two parts of which the first has
// few bits, so that its multiples are exact (Cody and Waite, Software Manual for the Elementary Functions, 1980)
__device__ __forceinline__ float log_of(float x) {
  const int e = (int)(__float_as_uint(x) >> 23) - 127;
  const float f = __uint_as_float((__float_as_uint(x) & 0x007FFFFFu) | 0x3F800000u);
  return fmaf((float)e, 0.693145751953125f, fmaf((float)e, 1.42860682e-6f, __log2f(f) * 0.693147181f));
}

__device__ __forceinline__ float score_of(float z, float prev, float lse) {      // NaN: there is none
  const float x = __fadd_rn(prev, __fsub_rn(z, lse));
  return x != x ? -INFINITY : x;
}
constexpr uint32_t NOTHING = 0x007FFFFFu;      // -inf, `ordered`
template <typename T> __device__ __forceinline__ uint32_t next_below(uint32_t u) {      // the next smaller number of the type, `ordered` (below 0: nothing larger than that)
  return u <= NOTHING ? NOTHING : u - (std::is_same<T, float>::value ? 1u : 0x10000u);
}
// Scores equal to the K-th best one S, for which a warp answers: whether a list has left out one that counts, and the places of those of the lowest indices.
// (As a function that is called it costs 0.3 us of every call, in this place 0.1.)
template <typename T>
__device__ __forceinline__ void equal_scores(const SelectArgs& A, int req, uint32_t S, const u64* keys, bool few, const u64* cand, int found, const float* prev, const float* lse, const int* ended) {
  const int lane = threadIdx.x & 31, K = A.K, V = A.V, lists = K * A.pieces;
  auto dead = [&](int k) { return !(prev[k] > -INFINITY && fabsf(lse[k]) < INFINITY); };
  auto put = [&](int place, int k, int t) {
    const int o = req * K + place;
    A.scores[o] = unordered(S);
    A.tokens[o] = t, A.parents[o] = k, A.done_out[o] = ended[k] || t == A.eos;
  };
  // A list of such a limit has entries of score S itself, or there would be K better ones.  If these are one logit, the limit, what it has left out of that logit has higher
  // indices and does not count; smaller logits do if the next smaller number still has that score
  bool counts = false;
#pragma unroll 1
  for (int e = lane; e < lists * A.L; e += 32)
    if (const u64 key = keys[e]; (uint32_t)(key >> 32) == S) {
      const int l = few ? e % lists : e / A.L, nth = few ? e / lists : e % A.L, k = l / A.pieces;
      if (ended[k] || dead(k)) continue;
      const long list = ((long)req * lists + l) * (A.L + 1);
      const uint32_t z = ordered(__ldcg(A.values + list + nth)), d = ordered(__ldcg(A.values + list + A.L));
      if (d > NOTHING && ordered(score_of(unordered(d), prev[k], lse[k])) == S)
        counts |= z != d || ordered(score_of(unordered(next_below<T>(d)), prev[k], lse[k])) == S;
    }
  if (!__any_sync(0xffffffffu, counts)) {
#pragma unroll 1
    for (int e = lane; e < found; e += 32)
      if (const u64 mine = cand[e]; (uint32_t)(mine >> 32) == S) {
        const uint32_t flat = ~(uint32_t)mine;
        const int place = place_of(mine, cand, found);
        if (place < K) put(place, (int)(flat / (uint32_t)V), (int)(flat % (uint32_t)V));
      }
    return;
  }
  int at = 0;      // better ones, all of them candidates
#pragma unroll 1
  for (int e = lane; e < found; e += 32) at += (uint32_t)(cand[e] >> 32) > S;
  at = __reduce_add_sync(0xffffffffu, at);
  for (int k = 0; k < K && at < K; k++) {
    const T* z = reinterpret_cast<const T*>(A.logits) + ((long)req * K + k) * A.stride;
    const bool end = ended[k] != 0, none = end || dead(k);
    for (long v = 0; v < V && at < K; v += 256) {
      uint32_t hits = 0;
#pragma unroll 8
      for (int e = 0; e < 8; e++) {      // (logits 32 apart: a hit's index is v + 32 e + lane)
        const long t = v + 32 * e + lane;
        float x = -INFINITY;
        if (t < V && !none) x = score_of(fmaxf((float)z[t], -INFINITY), prev[k], lse[k]);
        if (end && t == A.eos && prev[k] > -INFINITY) x = prev[k];
        hits |= t < V && ordered(x) == S ? 1u << e : 0u;
      }
      if (!__any_sync(0xffffffffu, hits != 0)) continue;
#pragma unroll 1
      for (int e = 0; e < 8; e++) {
        const uint32_t those = __ballot_sync(0xffffffffu, hits >> e & 1);
        const int to = at + __popc(those & ((1u << lane) - 1));
        if ((hits >> e & 1) && to < K) put(to, k, (int)v + 32 * e + lane);
        at += __popc(those);
      }
    }
  }
}

// BULK: rows begin on 16-byte boundaries
template <typename T, bool BULK>
__global__ void __launch_bounds__(SEL_THREADS, SEL_PER_SM) beam_select_k(const __grid_constant__ SelectArgs A) {
  extern __shared__ __align__(128) uint8_t fetched[];
  __shared__ uint64_t bar;
  __shared__ float tops[32], sums[SEL_WARPS];
  __shared__ u64 cand[SEL_HELD], red[32];
  __shared__ int n_cand, last;
  __shared__ uint32_t limit;      // the largest score of what lists have left out, `ordered`
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, K = A.K, V = A.V;
  const int row = blockIdx.y, req = row / K;
  const long list = (long)row * A.pieces + blockIdx.x;
  if (tid == 0) {
    n_cand = 0;
    tc::mbar_init(&bar, 1);
    tc::mbar_fence_init();
  }
  mlb_pdl_sync();
  __shared__ float prev[SEL_MAX_K], lse[SEL_MAX_K];      // the request's beams, which the merge will want
  __shared__ int ended[SEL_MAX_K];
  if (tid < K) prev[tid] = A.prev[req * K + tid], ended[tid] = A.done[req * K + tid] != 0;
  __syncthreads();
  if (!ended[row - req * K]) {
    constexpr int CHUNK = SEL_CHUNK_BYTES / sizeof(T);
    T* data = reinterpret_cast<T*>(fetched);
    const int begin = blockIdx.x * A.piece, n = min(A.piece, V - begin);
    const T* z = reinterpret_cast<const T*>(A.logits) + row * A.stride + begin;
    float m = -INFINITY, s = 0.f, bound = -INFINITY;
    // Candidates are down to the N-th: one more than are wanted, so that what is left out has the K-th one's score only if the next one has, too (32 beams have no part more
    // to bound that one by).  What no logit passes that is left out: the bound, where candidates that may be as large have gone, else the next smaller number
    const int parts = parts_for(K), N = K + 1;
    bool cut = false;
    int most = 0;      // candidates up to and with this thread's last
    bool over = false, late = false;
    uint32_t parity = 0;
    for (int c = 0; c < n; c += CHUNK, parity ^= 1) {
      const int count = min(CHUNK, n - c), whole = BULK ? (int)(count * sizeof(T) / 16 * 16 / sizeof(T)) : 0;
      if (BULK && tid == 0 && whole > 0 && !late) {
        tc::mbar_expect_tx(&bar, whole * sizeof(T));
        tc::bulk_load(data, z + c, whole * sizeof(T), &bar);
      }
      for (int e = whole + tid; e < count; e += SEL_THREADS) data[e] = z[c + e];
      if (tid < 8 && count + tid < (count + 7) / 8 * 8) data[count + tid] = (T)-INFINITY;
      if (BULK && whole > 0 && !late && !__all_sync(0xffffffffu, tc::mbar_wait(&bar, parity, 0xD3))) {
        late = true;      // nothing more is fetched, and what is on its way is waited for once more
        tc::mbar_wait(&bar, parity, 0xD4);
        __syncwarp();
      }
      __syncthreads();
      // Too few logits for all threads go to all parts alike (to neighbours 32 eights apart, which only so few can afford: they meet in the same banks)
      const int mine = count < SEL_THREADS * 8 ? 8 * ((lane & 7) * 32 + warp * 4 + (lane >> 3)) : 8 * tid;
      float top = -INFINITY;
      Eight<T> x;
#pragma unroll 2
      for (int e = mine; e < count; e += SEL_THREADS * 8) top = fmaxf(top, x.load(data + e));
      const float kth = kth_of_parts(top, min(N, parts), parts, tops, [](float a, float b) { return fmaxf(a, b); });
      if (c == 0) bound = kth;
      top = warp_max(tops[lane % parts]);
      if (top > m) s *= ex2((m - top) * 1.44269504088896f), m = top;      // (from -inf: 0 times 0)
      const float mm = m == -INFINITY ? 0.f : m;
#pragma unroll 1
      for (int e = mine; e < count; e += SEL_THREADS * 8) {
        const float best = x.load(data + e);
#pragma unroll
        for (int k = 0; k < 8; k++) s += ex2((x.get(k) - mm) * 1.44269504088896f);
        if (best >= bound && !over) {
          uint32_t hits = 0;
#pragma unroll
          for (int k = 0; k < 8; k++) hits |= (x.get(k) >= bound ? 1u : 0u) << k;
          hits &= 0xFFu >> max(0, 8 - (count - e));
          for (; hits != 0; hits &= hits - 1) {
            const int k = __ffs(hits) - 1;
            most = atomicAdd(&n_cand, 1) + 1;
            if (most <= SEL_CAND) cand[most - 1] = rank_of(fmaxf((float)data[e + k], -INFINITY), begin + c + e + k);
          }
        }
      }
      const bool more = c + CHUNK < n;
      if (__syncthreads_or(most > (more ? 2 * K : SEL_CAND))) {
        over |= __syncthreads_or(most > SEL_CAND) != 0;
        if (!over && more) {      // the N best of them stay
          const int found = n_cand;
          u64 mine[SEL_CAND / SEL_THREADS];
          int place[SEL_CAND / SEL_THREADS];
#pragma unroll
          for (int h = 0; h < SEL_CAND / SEL_THREADS; h++) {
            const int e = tid + h * SEL_THREADS;
            mine[h] = e < found ? cand[e] : 0ull;
            place[h] = e < found ? place_of(mine[h], cand, found) : N;
          }
          __syncthreads();
#pragma unroll
          for (int h = 0; h < SEL_CAND / SEL_THREADS; h++)
            if (place[h] < N) cand[place[h]] = mine[h];
          if (tid == 0) n_cand = N;
          __syncthreads();
          bound = unordered((uint32_t)(cand[N - 1] >> 32));
          cut = true;
          __syncthreads();
        }
        most = 0;
      }
      tc::fence_async_smem();      // (the next bulk copy writes what has been read)
      if (more) __syncthreads();
    }
    // the piece's sum
    s = warp_sum(s);
    if (lane == 0) sums[warp] = s;
    __syncthreads();
    if (tid == 0) {
      s = 0.f;
#pragma unroll
      for (int w = 0; w < SEL_WARPS; w++) s += sums[w];
      A.stats[list] = make_float2(m, s);
    }
    const int L = A.L;
    if (!over) {
      const int found = n_cand;
      for (int e = tid; e < found; e += SEL_THREADS) {
        const u64 mine = cand[e];
        const int k = found <= L ? e : place_of(mine, cand, found);      // (the merge needs no order)
        if (k <= L) A.values[list * (L + 1) + k] = unordered((uint32_t)(mine >> 32)), A.ids[list * (L + 1) + k] = (int)~(uint32_t)mine;
      }
      if (tid >= found && tid < L) A.ids[list * (L + 1) + tid] = -1;
      if (tid == L && found <= L) A.values[list * (L + 1) + L] = cut ? bound : unordered(next_below<T>(ordered(bound)));
    } else {
      u64 prior = ~0ull;
      for (int k = 0; k <= K; k++) {      // (one more: the largest that is left out)
        u64 best = 0;
        for (int e = tid; e < n; e += SEL_THREADS) {
          const u64 r = rank_of(fmaxf((float)z[e], -INFINITY), begin + e);
          if (r < prior) best = max(best, r);
        }
        prior = best = block_best(best, red);
        const long a = list * (L + 1) + (k < K ? k : L);
        if (tid == 0) A.values[a] = best == 0 ? -INFINITY : unordered((uint32_t)(best >> 32)), A.ids[a] = (int)~(uint32_t)best;
      }
      if (tid >= K && tid < L) A.ids[list * (L + 1) + tid] = -1;
    }
  }
  // ---- the request's last thread block merges
  __syncthreads();
  if (tid == 0) last = mlb_count_block(A.ticket + req) == A.pieces * K - 1;
  __syncthreads();
  if (!last) return;
  const int lists = K * A.pieces, L = A.L;
  if (tid == 0) A.ticket[req] = 0, n_cand = 0, limit = 0;
  for (int k = warp; k < K; k += SEL_WARPS) {      // (an ended beam's are nothing, and not asked for)
    const float2* st = A.stats + (long)(req * K + k) * A.pieces;
    float2 v[2];      // (pieces past 64 are read again)
    float m = -INFINITY;
#pragma unroll
    for (int h = 0; h < 2; h++) v[h] = lane + 32 * h < A.pieces ? __ldcg(st + lane + 32 * h) : make_float2(-INFINITY, 0.f), m = fmaxf(m, v[h].x);
    for (int p = lane + 64; p < A.pieces; p += 32) m = fmaxf(m, __ldcg(st + p).x);
    m = warp_max(m);
    auto term = [&](const float2& t) { return t.x == m ? t.y : t.y * ex2((t.x - m) * 1.44269504088896f); };
    float s = (lane < A.pieces ? term(v[0]) : 0.f) + (lane + 32 < A.pieces ? term(v[1]) : 0.f);
    for (int p = lane + 64; p < A.pieces; p += 32) s += term(__ldcg(st + p));
    s = warp_sum(s);
    if (lane == 0) lse[k] = s > 0.f ? m + log_of(s) : -INFINITY;
  }
  __syncthreads();
  // The lists' entries.  Of up to 4 beams the lists' first ones go before their second ones: many lists, so that every part has some of each beam.  Of more beams
  // a list's entries go to as many parts of the thread block as there are, so that the parts' best are a bound also where one beam has all of the K best (8 x 32
  // beams of 50304 logits 33 us, the other way 67; 8 x 8 beams 13.4, 14.5; 1 x 4 beams 7.1, 6.8).  Loops kept short, since each runs once or twice.
  const bool few = K <= 4;
  const int mine = few ? tid : warp + 8 * (lane >> 4) + 16 * (lane >> 3 & 1) + 32 * (lane & 7), inner = few ? lists : L;
  u64* keys = reinterpret_cast<u64*>(fetched);
  u64 best = 0;
  uint32_t most_left = 0;
  const float per_inner = 1.f / inner, per_beam = 1.f / A.pieces;      // ((x + 1/2) / n rounded down is exact for the few thousands that these are)
#pragma unroll 1
  for (int e = mine; e < lists * L; e += SEL_THREADS) {
    const int outer = (int)((e + 0.5f) * per_inner), rest = e - outer * inner, l = few ? rest : outer, nth = few ? outer : rest, k = (int)((l + 0.5f) * per_beam);
    const long a = ((long)req * lists + l) * (L + 1) + nth;
    int t = __ldcg(A.ids + a);
    float x = __ldcg(A.values + a), y = nth == L - 1 ? __ldcg(A.values + a + 1) : -INFINITY;
    // a beam that has ended, and one of no continuation: it was nothing, or its logits have no logarithm of a sum
    const bool end = ended[k] != 0, dead = !end && !(prev[k] > -INFINITY && fabsf(lse[k]) < INFINITY);
    if (end || dead) {
      x = -INFINITY, t = nth;
      if (end && A.eos >= 0 && A.eos < V) {
        t = nth == 0 ? A.eos : nth - 1 < A.eos ? nth - 1 : nth;
        if (nth == 0) x = prev[k];
      }
      if (l != k * A.pieces || t >= V) t = -1;
    } else {
      x = score_of(x, prev[k], lse[k]), y = score_of(y, prev[k], lse[k]);
      if (y > -INFINITY) most_left = max(most_left, ordered(y));
    }
    const u64 key = t < 0 ? 0ull : rank_of(x != x ? -INFINITY : x, (uint32_t)k * (uint32_t)V + (uint32_t)t);
    keys[e] = key;
    best = max(best, key);
  }
  most_left = __reduce_max_sync(0xffffffffu, most_left);
  if (lane == 0 && most_left != 0) atomicMax(&limit, most_left);
  const u64 bound = kth_of_parts(best, K, parts_for(K), red, [](u64 a, u64 b) { return a > b ? a : b; });
#pragma unroll 1
  for (int e = tid; e < lists * L; e += SEL_THREADS) {
    const u64 key = keys[e];
    if (key != 0 && key >= bound) cand[atomicAdd(&n_cand, 1)] = key;
  }
  __syncthreads();
  const int found = n_cand;      // (K or more: every beam has a continuation, if one of -inf)
  // What lists have left out scores S at most, S being the K-th best score.  If one does score S, the warp that has the K-th decides on all of that score
  most_left = limit;
  bool tied = false;
  for (int e = tid; e < found; e += SEL_THREADS) {
    const u64 mine = cand[e];
    const int k = place_of(mine, cand, found);
    if (k >= K) continue;
    if ((uint32_t)(mine >> 32) == most_left) {
      tied |= k == K - 1;
      continue;
    }
    const uint32_t flat = ~(uint32_t)mine;
    const int from = (int)(flat / (uint32_t)V), t = (int)(flat % (uint32_t)V), o = req * K + k;
    A.scores[o] = unordered((uint32_t)(mine >> 32));
    A.tokens[o] = t, A.parents[o] = from, A.done_out[o] = ended[from] || t == A.eos;
  }
  if (__any_sync(0xffffffffu, tied)) equal_scores<T>(A, req, most_left, keys, few, cand, found, prev, lse, ended);
}

// Logits of a piece, a multiple of 8: the machine's thread blocks once over the rows, but no more of a row than one fetch where there are enough of them, SEL_LEAST
// logits and more each, and no more lists than a thread block holds to merge
int select_list(int K) { return K <= 16 ? 2 * K : K; }      // entries of a piece's list, the limit apart: usually all its candidates, which then need no places
int select_piece(int rows, int K, int V, int bits) {
  const long fill = (long)SEL_PER_SM * mlb_sm_count() / rows, one = ((long)V * (bits / 8) + SEL_CHUNK_BYTES - 1) / SEL_CHUNK_BYTES, most = (V - 1) / SEL_LEAST + 1,
             held = SEL_HELD / (K * select_list(K));
  long n = fill > one ? fill : one;
  n = n < most ? n : most;
  n = n < held ? n : held;
  n = n < 1 ? 1 : n;
  return (int)(((V + n - 1) / n + 7) / 8 * 8);
}
template <typename T, bool BULK>
cudaError_t launch_select(const SelectArgs& a, int rows, cudaStream_t st) {
  const int bytes = a.piece * (int)sizeof(T) < SEL_CHUNK_BYTES ? a.piece * (int)sizeof(T) : SEL_CHUNK_BYTES;
  const int least = SEL_HELD * (int)sizeof(u64);      // (the merge's)
  return mlb_launch(beam_select_k<T, BULK>, dim3(a.pieces, rows), dim3(SEL_THREADS), bytes > least ? (bytes + 127) / 128 * 128 : least, st, a);
}

// ------------------------------------------------------------------ beams in the order of their parents
// Row b K + k continues row b K + parents[b, k].  Full pages are shared: their numbers are copied from the parent's table.  The page that is being filled belongs to one
// row alone, so a row that continues another one gets that one's tokens copied to its spare page, and the page it had is its spare from then on: nothing
// that is read is written, whatever the order of the rows.  Bound by the copied bytes: 128 beams of 12 layers of 12 heads of 64, 52 tokens of a page each for 44 % of
// them, 15.3 us (74 MB moved, 4.8 TB/s); 4 beams 3.1 us.
struct OrderArgs {
  uint8_t* pages;
  int *table_out, *spare_out, *hist_out;
  const int *table, *spare, *lens, *hist, *parents, *tokens;
  long n_pages;
  int K, Hkv, page, block_vecs, width, T, parts;      // block_vecs: 16-byte words of a block of 16 tokens; parts: thread blocks that copy a layer's page
};
constexpr int ORDER_THREADS = 256;
__global__ void __launch_bounds__(ORDER_THREADS) beam_reorder_k(const OrderArgs A) {
  mlb_pdl_sync();
  const int row = blockIdx.x, tid = threadIdx.x;
  int parent = A.parents[row];
  const int spare = A.spare[row];
  if (parent < 0 || parent >= A.K) {
    if (tid == 0 && blockIdx.y == 0) mlb_set_error(MLB_ERR_BOUNDS, 0xB3);
    parent = row % A.K;
  }
  const int src = row / A.K * A.K + parent;
  const int len = min(max(A.lens[row], 0), A.width * A.page), full = len / A.page, rest = len - full * A.page;
  const bool moved = rest > 0 && src != row;
  if (blockIdx.y == 0) {
    for (int p = tid; p < A.width; p += ORDER_THREADS)
      A.table_out[(long)row * A.width + p] = moved && p == full ? spare : A.table[(long)(p < full ? src : row) * A.width + p];
    if (tid == 0) A.spare_out[row] = moved ? A.table[(long)row * A.width + full] : spare;
    for (int t = tid; t < min(len, A.T); t += ORDER_THREADS) A.hist_out[(long)row * A.T + t] = A.hist[(long)src * A.T + t];
    if (tid == 0 && len < A.T) A.hist_out[(long)row * A.T + len] = A.tokens[row];
    return;
  }
  if (!moved) return;
  const int from = A.table[(long)src * A.width + full], to = spare;
  if (from < 0 || from >= A.n_pages || to < 0 || to >= A.n_pages) {
    if (tid == 0) mlb_set_error(MLB_ERR_BOUNDS, 0xB4);
    return;
  }
  // `parts` blocks a layer: this one's words of the Hkv heads' tokens, 4 on their way at a time
  const int layer = (blockIdx.y - 1) / A.parts, part = (blockIdx.y - 1) % A.parts;
  const unsigned blocks = A.page / 16, each = (rest + 15) / 16 * A.block_vecs, head = blocks * A.block_vecs, total = A.Hkv * each;
  const unsigned v0 = (unsigned)((unsigned long long)total * part / A.parts), v1 = (unsigned)((unsigned long long)total * (part + 1) / A.parts);
  const uint4* f = reinterpret_cast<const uint4*>(A.pages) + ((long)layer * A.n_pages + from) * A.Hkv * head;
  uint4* t = reinterpret_cast<uint4*>(A.pages) + ((long)layer * A.n_pages + to) * A.Hkv * head;
  for (unsigned v = v0 + tid; v < v1; v += 4 * ORDER_THREADS) {
    uint4 w[4];
    unsigned at[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const unsigned x = v + k * ORDER_THREADS;
      at[k] = x / each * head + x % each;      // (a page of all heads is below 2^32 bytes)
      if (x < v1) w[k] = f[at[k]];
    }
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (v + k * ORDER_THREADS < v1) t[at[k]] = w[k];
  }
}

}  // namespace

MLB_API int mlb_block_tables(int* table, int* slots, int* pos, int* starts, int* new_lens, int* left, int* ticket, const int* lens, const int* news,
                             const int* stack, const int* n_free, int B, int width, int page, int rows, int stack_size, cudaStream_t st) {
  if (B < 1 || B > TAB_MAX_B || page < 1 || width < 1 || rows < 0 || rows > TAB_MAX_ROWS || (long)B * width >= 1L << 31 || (long)width * page >= 1L << 31) return -7;
  const int want = (rows + TAB_THREADS - 1) / TAB_THREADS, most = 2 * mlb_sm_count();
  const TableArgs a{table, slots, pos, starts, new_lens, left, ticket, lens, news, stack, n_free, B, width, page, rows, stack_size};
  return (int)mlb_launch(block_tables_k, dim3(want < 1 ? 1 : want < most ? want : most), dim3(TAB_THREADS), (2 * B + 1) * sizeof(int), st, a);
}

// Pieces that a row of V logits is cut into, and (-7) nothing for what the kernel does not take
MLB_API int mlb_beam_select_pieces(int rows, int K, int V, int bits) {
  if (K < 1 || K > SEL_MAX_K || V < 1 || rows < 1 || rows > 65535 || (long)K * V >= 0xFFFFFFFFL) return -7;
  const int piece = select_piece(rows, K, V, bits);
  return (V - 1) / piece + 1;
}
// bits: 16 (bf16) or 32 (fp32) logits, rows `stride` elements apart; stats: 2 floats for each piece of each row, values and ids 2 K + 1
MLB_API int mlb_beam_select(float* scores, int* tokens, int* parents, int* done_out, const void* logits, const float* prev, const int* done, float* stats,
                            float* values, int* ids, int* ticket, int rows, int K, int V, long stride, int eos, int bits, cudaStream_t st) {
  const int pieces = mlb_beam_select_pieces(rows, K, V, bits);
  if (pieces < 0 || rows % K != 0) return -7;
  const SelectArgs a{scores, tokens, parents, done_out, logits, prev, done, (float2*)stats, values, ids, ticket, stride, K, select_list(K), V, eos, pieces, select_piece(rows, K, V, bits)};
  const bool bulk = ((uintptr_t)logits & 15) == 0 && stride * (bits / 8) % 16 == 0;
  if (bits == 16) return (int)(bulk ? launch_select<bf16, true>(a, rows, st) : launch_select<bf16, false>(a, rows, st));
  return (int)(bulk ? launch_select<float, true>(a, rows, st) : launch_select<float, false>(a, rows, st));
}

// pages null: no cache to copy in; block_bytes of 16 tokens of a head
MLB_API int mlb_beam_reorder(uint8_t* pages, int* table_out, int* spare_out, int* hist_out, const int* table, const int* spare, const int* lens, const int* hist,
                             const int* parents, const int* tokens, int layers, long n_pages, int Hkv, int page, int block_bytes, int B, int K, int width, int T,
                             cudaStream_t st) {
  if (page < 16 || page % 16 != 0 || block_bytes % 16 != 0 || ((uintptr_t)pages & 15) != 0 || K < 1 || width < 1 || layers > 65534 || (long)width * page >= 1L << 31) return -7;
  // a part is 1024 words (16 KB) of a page or more
  const long words = (long)Hkv * (page / 16) * (block_bytes / 16), most = layers > 0 ? 65534 / layers : 1;
  if (words >= 1L << 28) return -7;
  const int parts = (int)(words / 1024 < 1 ? 1 : words / 1024 < most ? words / 1024 : most);
  const OrderArgs a{pages, table_out, spare_out, hist_out, table, spare, lens, hist, parents, tokens, n_pages, K, Hkv, page, block_bytes / 16, width, T, parts};
  return (int)mlb_launch(beam_reorder_k, dim3(B * K, pages ? layers * parts + 1 : 1), dim3(ORDER_THREADS), 0, st, a);
}
