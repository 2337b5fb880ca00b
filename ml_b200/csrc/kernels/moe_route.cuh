// Routing of tokens to experts: the k best of E scores a token, their weights, the experts' mean probabilities, and the logits' gradient.
//
// A warp has a token, lane l the experts l, l + 32, ...  A logit of NaN counts as -inf and an expert at -inf is not there.  Scores are a softmax over the experts or a
// sigmoid each.  Experts are chosen by their logits, or, with a bias or groups, by score + bias in 64 bits: in 32 the last bits of two roundings would decide between
// neighbours, and another way of adding up would choose other experts.  Equal ones go to the lowest index.
// Bound by instructions: 8192 tokens to 8 of 256 experts 7.8 us by logits (700 a token; 1.3 for the bytes), 17.3 with a bias and 4 of 8 groups (1550; with 64 bits for
// every expert 31.0, with them for the candidates and two experts of each group 21.5); 16 tokens 3.1 and 5.6, of which a launch is 2.
#pragma once
#include <algorithm>
#include <type_traits>

#include "../common.cuh"

namespace {

constexpr int ROUTE_WARPS = 8, MAX_E = 1024, MAX_K = 32, MAX_GROUPS = 32, LIST = 34;      // (ops/ref_moe.py refuses more)
struct RouteArgs {
  const void* logits;
  const float* bias;
  void* weights;
  int* idx;
  float* part;      // [blocks][E] sums of probabilities (null: not asked for)
  long N, ld;
  int E, k, groups, top, sigmoid, renorm, wide_w;
  float scale;
};
__host__ __device__ constexpr int own_doubles(int E) { return E > 32 ? E : 32; }      // a warp's shared memory where the choice is not by logits: numbers of the experts, or of candidates
template <typename T> __device__ __forceinline__ float logit(const T* z, int i);
template <> __device__ __forceinline__ float logit<float>(const float* z, int i) { return __ldg(z + i); }
template <> __device__ __forceinline__ float logit<bf16>(const bf16* z, int i) { return __bfloat162float(z[i]); }
// NaN -> -inf, -0 -> 0.  Numbers below the normal ones stay: these are compared, too, and the compiler's own instructions take them for 0.
__device__ __forceinline__ float seen(float z) {
  float r;
  asm("max.f32 %0, %1, %2;" : "=f"(r) : "f"(z), "f"(-INFINITY));
  asm("add.f32 %0, %0, %1;" : "+f"(r) : "f"(0.f));
  return r;
}
__device__ __forceinline__ double wide(float v) {
  double r;
  asm("cvt.f64.f32 %0, %1;" : "=d"(r) : "f"(v));
  return r;
}
// exp(x) for x <= 0 to a few 2^-24: the product with log2 e in two parts
__device__ __forceinline__ float exp_fine(float x) {
  const float hi = x * 1.44269504f, lo = fmaf(x, 1.44269504f, -hi) + x * 1.92596299e-8f;
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(hi));
  return fmaf(e, lo * 0.693147182f, e);
}
// exp(a - b), 1 where they are equal (infinite ones too), 0 where a is not there
__device__ __forceinline__ float exp_from(float a, float b) { return a == b ? 1.f : a == -INFINITY ? 0.f : exp_fine(fmaxf(a - b, -200.f)); }
__device__ __forceinline__ float sigmoid_fine(float z) {
  const float e = exp_fine(fmaxf(-fabsf(z), -200.f));
  return __fdividef(z >= 0.f ? 1.f : e, 1.f + e);      // (2 steps of 2^-23; the denominator is 1 to 2)
}
// The same to (7 + 1.23 |z|) 2^-24 of itself below 0 (ex2 4, the sum 1, rcp 2; the product with log2 e is rounded, and so is log2 e: an exponent's error grows with it), 0 for -inf and
// below 2^-126: says what may be chosen
__device__ __forceinline__ float sigmoid_fast(float z) {
  float e, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.44269504f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
  return s;
}
// sigmoid(z) / exp(top) for top = min(0, largest z): scores for shares, whose sum is not too small for fp32
__device__ __forceinline__ float sigmoid_from(float z, float top) {
  return z == -INFINITY ? 0.f : z >= 0.f ? sigmoid_fine(z) : __fdividef(exp_from(z, top), 1.f + exp_fine(fmaxf(z, -200.f)));
}
// numbers in the order of their values, as unsigned ones
__device__ __forceinline__ uint32_t order32(float v) {
  const uint32_t u = __float_as_uint(v);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ uint64_t order64(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
  return u ^ ((u >> 63) ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ double value64(uint64_t key) { return __longlong_as_double((long long)(key ^ ((key >> 63) ? 1ull << 63 : ~0ull))); }
constexpr uint32_t GONE32 = 0x007fffffu;                    // order32(-inf)
constexpr uint64_t GONE64 = 0x000fffffffffffffull;          // order64(-inf)
__device__ __forceinline__ uint32_t warp_best(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ uint64_t warp_best(uint64_t v) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return (uint64_t)hi << 32 | lo;
}

// The k best of the warp's keys, best first: lane j keeps the index of the j-th (-1: none left)
template <int V>
__device__ __forceinline__ int choose(uint32_t (&key)[V], int k, int lane) {
  typedef uint32_t K;
  int mine = -1;
  K best = key[0];
  int at = 0;
#pragma unroll
  for (int v = 1; v < V; v++)
    if (key[v] > best) best = key[v], at = v;
  for (int j = 0; j < k; j++) {
    const K top = warp_best(best);
    if (top <= GONE32) break;
    const unsigned i = __reduce_min_sync(0xffffffffu, best == top ? (unsigned)(at * 32 + lane) : 0xffffffffu);
    if (lane == j) mine = (int)i;
    if ((int)(i & 31) == lane) {
#pragma unroll
      for (int v = 0; v < V; v++)
        if (v == at) key[v] = 0;
      best = key[0], at = 0;
#pragma unroll
      for (int v = 1; v < V; v++)
        if (key[v] > best) best = key[v], at = v;
    }
  }
  return mine;
}

// What may be chosen of many keys a lane.  A bound that k + 1 lanes' best keys or a few more reach is no better than the k + 1-th best key, so what is chosen, and what comes
// behind it, is among the keys that reach it (or, with `below`, come near it): usually some more than k.  They are put side by side, a lane each.  Returns how many;
// over 32 (many equal ones): the list is not complete.  8192 tokens, 8 of 256 experts, by logits: 13.3 us with the bound out of a sort of the lanes' best, 7.8 so.
template <int V>
__device__ __forceinline__ int candidates(const uint32_t (&key)[V], int k, int lane, uint2* s, float below) {
  uint32_t best = key[0];
#pragma unroll
  for (int v = 1; v < V; v++) best = max(best, key[v]);
  uint32_t least = max(__reduce_min_sync(0xffffffffu, best), GONE32 + 1), over = __reduce_max_sync(0xffffffffu, best);
  if (over < least) return 0;
#pragma unroll 1
  for (int i = 0; i < 12 && least < over; i++) {      // (a bound that is kept is reached by k + 1 lanes, or by all)
    const uint32_t mid = least + ((over - least + 1) >> 1);
    const int n = __popc(__ballot_sync(0xffffffffu, best >= mid));
    if (n > k) least = mid;
    else over = mid - 1;
    if (n > k && n <= k + 4) break;
  }
  if (below > 0.f) least = max(order32(value_of(least) - below), GONE32 + 1);
  int count = 0;
  __syncwarp();
#pragma unroll
  for (int v = 0; v < V; v++) {
    const bool here = key[v] >= least;
    const unsigned all = __ballot_sync(0xffffffffu, here);
    s[here ? min(count + __popc(all & ((1u << lane) - 1)), 32) : 32] = make_uint2(key[v], v * 32 + lane);      // (place 32: for those that are none)
    count += __popc(all);
  }
  __syncwarp();
  return count;
}
// The k best of them, as choose() returns them
template <int V>
__device__ __forceinline__ int choose_many(uint32_t (&key)[V], int k, int lane, uint2* s) {
  const int count = k < 32 ? candidates(key, k, lane, s, 0.f) : 33;
  if (count > 32) return choose<V>(key, k, lane);
  const uint2 own = lane < count ? s[lane] : make_uint2(0, 0);
  int rank = 0;
#pragma unroll 4
  for (int j = 0; j < count; j++) {
    const uint2 x = s[j];
    rank += x.x > own.x || (x.x == own.x && x.y < own.y);
  }
  __syncwarp();
  if (lane < count) s[rank] = own;
  __syncwarp();
  return lane < k && lane < count ? (int)s[lane].y : -1;
}

// Groups: the experts' choice numbers t stand in s[E].  As many lanes as go into 32 share a group.  Lane l gets group l's three best numbers.
struct Best { float a, b, c; };
__device__ __forceinline__ Best best_of_groups(const float* s, int size, int groups, int lane) {
  const int bits = groups > 1 ? 32 - __clz(groups - 1) : 0, shift = 5 - bits, share = 1 << shift;
  const int g = lane >> shift, sub = lane & (share - 1), steps = (size + share - 1) >> shift;
  Best r = {-INFINITY, -INFINITY, -INFINITY};
  if (g < groups)
    for (int j = 0, x = (g * steps) >> bits; j < steps; j++, x = x + 1 == steps ? 0 : x + 1) {      // (begun at another place by each group: other banks)
      const int i = x * share + sub;
      const float t = i < size ? s[g * size + i] : -INFINITY;
      r.c = fmaxf(r.c, fminf(r.b, t));
      r.b = fmaxf(r.b, fminf(r.a, t));
      r.a = fmaxf(r.a, t);
    }
  for (int o = 1; o < share; o <<= 1) {
    const float x = __shfl_xor_sync(0xffffffffu, r.a, o), y = __shfl_xor_sync(0xffffffffu, r.b, o), z = __shfl_xor_sync(0xffffffffu, r.c, o);
    const float low = fminf(r.a, x), mid = fmaxf(r.b, y);      // the second best of all is one of these, and the third the other one or a third
    r.a = fmaxf(r.a, x);
    r.c = fmaxf(fminf(low, mid), fmaxf(r.c, z));
    r.b = fmaxf(low, mid);
  }
  const int from = (lane << shift) & 31;
  return {__shfl_sync(0xffffffffu, r.a, from), __shfl_sync(0xffffffffu, r.b, from), __shfl_sync(0xffffffffu, r.c, from)};
}
// The bits of the groups that stay, by the sums of their two best (lane l: of group l); `margin`: by how much the worst of them is ahead of the best of the others
__device__ __forceinline__ uint32_t order(float v) { return order32(v); }
__device__ __forceinline__ uint64_t order(double v) { return order64(v); }
__device__ __forceinline__ float value_of(uint64_t key) { return (float)value64(key); }
template <typename R>
__device__ __forceinline__ unsigned keep_groups(R sum, int groups, int top, int lane, float& margin) {
  auto key = lane < groups ? order(sum) : 0;
  auto low = key;
  unsigned stays = 0;
  for (int j = 0; j < top; j++) {
    low = warp_best(key);
    const int g = __ffs(__ballot_sync(0xffffffffu, key == low)) - 1;
    stays |= 1u << g;
    if (lane == g) key = 0;
  }
  const auto high = warp_best(key);
  margin = high == 0 ? INFINITY : value_of(low) - value_of(high);
  return stays;
}

// The choice by score + bias, in 64 bits throughout, the numbers in shared memory (s[E]).  For softmax with a bias where 32 bits leave it open, and many equal numbers.
template <typename T>
__device__ __noinline__ int choose_exact(const RouteArgs& A, const T* row, double* s, float m) {
  const int lane = threadIdx.x & 31, E = A.E;
  double all = 0;
  __syncwarp();
#pragma unroll 1
  for (int i = lane; i < E; i += 32) {
    const float z = seen(logit(row, i));
    const double x = exp(A.sigmoid ? -(double)z : z == m ? 0.0 : (double)z - (double)m);
    const double t = z == -INFINITY ? 0.0 : A.sigmoid ? 1.0 / (1.0 + x) : x;
    all += t;
    s[i] = t;
  }
  if (!A.sigmoid)
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
#pragma unroll 1
  for (int i = lane; i < E; i += 32) {
    const float z = seen(logit(row, i));
    const double t = A.sigmoid ? s[i] : all > 0 ? s[i] / all : 0.0;
    s[i] = z == -INFINITY ? -INFINITY : A.bias != nullptr ? t + wide(__ldg(A.bias + i)) : t;
  }
  __syncwarp();
  unsigned stays = 0xffffffffu;
  const int size = E / A.groups;
  if (A.groups > 1) {
    double a = -INFINITY, b = -INFINITY;
    float margin;
#pragma unroll 1
    for (int i = 0; lane < A.groups && i < size; i++) {
      const double t = s[lane * size + i];
      if (t > a) b = a, a = t;
      else if (t > b) b = t;
    }
    stays = keep_groups(a + (b > -INFINITY ? b : 0.0), A.groups, A.top, lane, margin);
  }
  int mine = -1;
#pragma unroll 1
  for (int j = 0; j < A.k; j++) {
    double best = -INFINITY;
    int at = 0;
#pragma unroll 1
    for (int i = lane; i < E; i += 32)
      if (s[i] > best && ((stays >> (A.groups > 1 ? i / size : 0)) & 1)) best = s[i], at = i;
    const uint64_t key = order64(best), top = warp_best(key);
    if (top <= GONE64) break;
    const unsigned i = __reduce_min_sync(0xffffffffu, key == top ? (unsigned)at : 0xffffffffu);
    if (lane == j) mine = (int)i;
    if ((int)(i & 31) == lane) s[i] = -INFINITY;
    __syncwarp();
  }
  __syncwarp();
  return mine;
}

// An expert's number in 64 bits where that is the expert's own affair: sigmoids; a softmax without bias over its common factor
// (one function: every token asks for it, so its code is at hand for the few that do so for groups, too)
template <typename T>
__device__ __noinline__ double own_number(const RouteArgs& A, const T* row, int i, float m) {
  const double z = (double)seen(logit(row, i)), x = exp(A.sigmoid ? -z : z - (double)m);
  return A.sigmoid ? 1.0 / (1.0 + x) + (A.bias != nullptr ? wide(__ldg(A.bias + i)) : 0.0) : x;
}

// PLAIN: by the logits alone
template <int V, typename T, bool PLAIN>
__global__ void __launch_bounds__(32 * ROUTE_WARPS, V <= 4 ? 6 : V == 8 ? 4 : 2) moe_route_k(const RouteArgs A) {
  mlb_pdl_sync();
  extern __shared__ double route_sm[];      // not PLAIN: the scores of each warp's token; lists of candidates; behind the loop: sums of probabilities
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, E = A.E;
  const uint32_t magic = 0xffffffffu / (uint32_t)(E / A.groups) + 1;      // (0, and not used so, where a group is one expert)
  uint2* list = (uint2*)(route_sm + (PLAIN ? 0 : ROUTE_WARPS * own_doubles(E))) + LIST * w;
  float sum_p[V];
#pragma unroll
  for (int v = 0; v < V; v++) sum_p[v] = 0.f;
  for (long n = (long)blockIdx.x * ROUTE_WARPS + w; n < A.N; n += (long)gridDim.x * ROUTE_WARPS) {
    const T* row = (const T*)A.logits + n * A.ld;
    float z[V], m = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; v++) {
      const int i = v * 32 + lane;
      z[v] = i < E ? seen(logit(row, i)) : -INFINITY;
      m = fmaxf(m, z[v]);
    }
    m = warp_max(m);
    float e[V], total = 0.f;      // exp(z - m) or scores, and their sum (for shares of sigmoids, below: relative to the largest)
    const bool sums = !A.sigmoid && (A.part != nullptr || !A.renorm || !PLAIN);
    if (sums || !PLAIN) {
#pragma unroll
      for (int v = 0; v < V; v++) {
        e[v] = A.sigmoid ? sigmoid_fast(z[v]) : z[v] == -INFINITY ? 0.f : exp_from(z[v], m);
        total += e[v];
      }
      if (sums) total = warp_sum(total);
    }
    if (A.part != nullptr) {
      float x[V], all = total;
      if (A.sigmoid) {
        all = 0.f;
#pragma unroll
        for (int v = 0; v < V; v++) x[v] = z[v] == -INFINITY ? 0.f : sigmoid_from(z[v], fminf(m, 0.f)), all += x[v];
        all = warp_sum(all);
      } else {
#pragma unroll
        for (int v = 0; v < V; v++) x[v] = e[v];
      }
      const float inv = all > 0.f ? __fdividef(1.f, all) : 0.f;
#pragma unroll
      for (int v = 0; v < V; v++) sum_p[v] = fmaf(x[v], inv, sum_p[v]);
    }
    int mine;
    if constexpr (PLAIN) {
      uint32_t key[V];
#pragma unroll
      for (int v = 0; v < V; v++) key[v] = order32(z[v]);
      if constexpr (V >= 4) mine = choose_many<V>(key, A.k, lane, list);
      else mine = choose<V>(key, A.k, lane);
    } else {
      // 32 bits say what may be chosen, 64 bits what is.  In 32 score + bias is off by less than slack, in steps of 2^-24 of `size`, the row's largest score + |bias|, of which the addition
      // is one.  An exponential of z - m has 7, and where the sum does not cancel (softmax with a bias) as much in its terms, 4.5 for their arguments' roundings (on average, of 1024 terms at
      // most), V + 4 for its additions, and 5 for the division and the product.  Sigmoids: of s |z| (1 - s) none is over size max(1.28, -m), so 8 + 1.23 max(1.28, -m) is all.
      // 2^-124 stands for what is flushed to 0.  (With 64 bits for the few tokens alone that 32 leave open, these wait some 10 us for code that no cache has.)
      float t[V], size = 0.f;
      const float inv = A.sigmoid || A.bias == nullptr ? 1.f : total > 0.f ? __fdividef(1.f, total) : 0.f;
#pragma unroll
      for (int v = 0; v < V; v++) {
        const int i = v * 32 + lane;
        const float b = i < E && A.bias != nullptr ? __ldg(A.bias + i) : 0.f, s = e[v] * inv;
        t[v] = z[v] == -INFINITY ? -INFINITY : fmaxf(s + b, -INFINITY);      // (NaN, of a bias: not there)
        if (z[v] > -INFINITY) size = fmaxf(size, s + fabsf(b));
      }
      const float steps = A.sigmoid ? 16.f + 1.3f * fminf(fmaxf(-m, 0.f), 128.f) : A.bias != nullptr ? 32.f + V : 16.f;      // (below -128 all scores are 0)
      const float slack = fmaf(5.9604645e-8f * steps, __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(size))), 4.7019774e-38f);
      const bool single = A.sigmoid || A.bias == nullptr;      // own_number() has them
      bool sure = slack < 1e30f && m < INFINITY;
      if (A.groups > 1) {
        float* s = (float*)(route_sm + w * own_doubles(E));
        __syncwarp();
#pragma unroll
        for (int v = 0; v < V; v++)
          if (v * 32 + lane < E) s[v * 32 + lane] = t[v];
        __syncwarp();
        const Best g = best_of_groups(s, E / A.groups, A.groups, lane);
        float margin;
        unsigned stays = keep_groups(g.b > -INFINITY ? g.a + g.b : g.a, A.groups, A.top, lane, margin);      // (a group without experts stays at -inf)
        if (!(margin > 4.f * slack)) {      // sums of two come near each other: 64 bits, where no third number comes near a group's second
          if (!single || __any_sync(0xffffffffu, lane < A.groups && g.c > -INFINITY && g.b - g.c <= 2.f * slack)) {
            sure = false;
          } else {
            const int size = E / A.groups;
            int ai = -1, bi = -1;
            for (int i = lane * size; lane < A.groups && i < lane * size + size; i++) {
              const float t = s[i];
              if (ai < 0 && t == g.a) ai = i;
              else if (bi < 0 && t == g.b) bi = i;
            }
            double sum = g.a;
            if (lane < A.groups && g.a > -INFINITY) sum = own_number(A, row, ai, m);
            if (lane < A.groups && g.b > -INFINITY) sum += own_number(A, row, bi, m);
            stays = keep_groups(sum, A.groups, A.top, lane, margin);
          }
        }
#pragma unroll
        for (int v = 0; v < V; v++)      // ((i magic) >> 32 is i / (experts of a group) for i < 2^16)
          if (!((stays >> ((magic ? __umulhi(v * 32 + lane, magic) : v * 32 + lane) & 31)) & 1)) t[v] = -INFINITY;
      }
      uint32_t key[V];
#pragma unroll
      for (int v = 0; v < V; v++) key[v] = order32(t[v]);
      const int count = A.k < 32 && sure ? candidates(key, A.k, lane, list, 4.f * slack) : 33;
      mine = -1;
      if (count <= 32) {
        const uint2 c = lane < count ? list[lane] : make_uint2(0, 0);
        double own = value_of(c.x);
        if (single && lane < count) own = own_number(A, row, (int)c.y, m);
        const uint64_t k64 = lane < count ? order64(own) : 0;
        uint64_t* keys = (uint64_t*)(route_sm + w * own_doubles(E));
        __syncwarp();
        keys[lane] = k64;
        __syncwarp();
        double near = INFINITY;      // (softmax with a bias: the distance to the next better one)
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < count; j++) {      // (the list is in the order of the experts but for v: of equal ones the index decides)
          const uint64_t x = keys[j];
          rank += x > k64 || (x == k64 && list[j].y < c.y);
          if (!single && j != lane) near = fmin(near, fabs(value64(x) - own));
        }
        if (!single) sure = !__any_sync(0xffffffffu, lane < count && rank <= A.k && near <= 2.0 * slack);
        __syncwarp();
        if (lane < count) list[rank].x = c.y;
        __syncwarp();
        if (lane < A.k && lane < count) mine = (int)list[lane].x;
      }
      if (count > 32 || !sure) mine = choose_exact(A, row, route_sm + w * own_doubles(E), m);
    }
    // lane j: the weight of the j-th
    const float zj = mine >= 0 ? seen(logit(row, mine)) : -INFINITY;
    float wj = 0.f;
    if (A.renorm) {      // relative to the largest chosen one, so that the sum is not too small for fp32
      const float top = warp_max(zj);
      wj = zj == -INFINITY ? 0.f : A.sigmoid ? sigmoid_from(zj, fminf(top, 0.f)) : exp_from(zj, top);
      const float sum = warp_sum(wj);
      wj = sum > 0.f ? __fdividef(wj, sum) : 0.f;
    } else if (zj > -INFINITY) {
      wj = A.sigmoid ? sigmoid_fine(zj) : __fdividef(exp_from(zj, m), total);
    }
    if (lane < A.k) {
      A.idx[n * A.k + lane] = mine;
      wj *= A.scale;
      if (A.wide_w) ((float*)A.weights)[n * A.k + lane] = wj;
      else ((bf16*)A.weights)[n * A.k + lane] = __float2bfloat16(wj);
    }
  }
  if (A.part != nullptr) {
    float* s = (float*)route_sm;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; v++)
      if (v * 32 + lane < E) s[w * E + v * 32 + lane] = sum_p[v];
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += 32 * ROUTE_WARPS) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < ROUTE_WARPS; k++) t += s[k * E + e];
      A.part[(long)blockIdx.x * E + e] = t;
    }
  }
}
// mean[e] = the blocks' sums / N: 32 threads to an expert, always the same blocks to a thread
__global__ void __launch_bounds__(1024) moe_mean_k(float* mean, const float* __restrict__ part, int blocks, int E, float inv) {
  mlb_pdl_sync();
  const int lane = threadIdx.x & 31, e = blockIdx.x * 32 + lane, s = threadIdx.x >> 5;
  __shared__ float red[32][33];
  float t = 0.f;
  if (e < E) {
#pragma unroll 10
    for (int b = s; b < blocks; b += 32) t += part[(long)b * E + e];
  }
  red[s][lane] = t;
  __syncthreads();
  t = warp_sum(red[lane][s]);      // (expert s of these 32)
  if (lane == 0 && blockIdx.x * 32 + s < E) mean[blockIdx.x * 32 + s] = t * inv;
}

// ------------------------------------------------------------------ backward
// g_j = scale dweights_j, h = dmean / N, p = softmax (or s / sum s), q = chosen weights / scale.
//   softmax, renorm: dz_j = q_j (g_j - sum q g) at the chosen; else dz_i = p_i (g_i - sum p g), g 0 elsewhere
//   sigmoid, renorm: dz_j = q_j (1 - s_j) (g_j - sum q g);       else dz_j = g_j s_j (1 - s_j)
//   mean: + p_i (h_i - sum p h), for sigmoids times 1 - s_i
struct RouteBwdArgs {
  void* dlogits;
  const void *dweights, *logits;
  const float* dmean;
  const int* idx;
  long N, ld;
  int E, k, sigmoid, renorm, wide_w;
  float scale;
};
template <int V, typename T>
__global__ void __launch_bounds__(32 * ROUTE_WARPS) moe_route_bwd_k(const RouteBwdArgs A) {
  mlb_pdl_sync();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, E = A.E;
  const float inv_n = __fdiv_rn(1.f, (float)A.N);
  for (long n = (long)blockIdx.x * ROUTE_WARPS + w; n < A.N; n += (long)gridDim.x * ROUTE_WARPS) {
    const T* row = (const T*)A.logits + n * A.ld;
    float z[V], d[V], m = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; v++) {
      const int i = v * 32 + lane;
      z[v] = i < E ? seen(logit(row, i)) : -INFINITY;
      m = fmaxf(m, z[v]);
      d[v] = 0.f;
    }
    m = warp_max(m);
    const int j = lane < A.k ? A.idx[n * A.k + lane] : -1;
    if (j >= E) mlb_set_error(MLB_ERR_BOUNDS, 0xD2);
    const int mine = j < E ? j : -1;
    const float g = mine < 0 ? 0.f : A.scale * (A.wide_w ? ((const float*)A.dweights)[n * A.k + lane] : __bfloat162float(((const bf16*)A.dweights)[n * A.k + lane]));
    const float zj = mine >= 0 ? seen(logit(row, mine)) : -INFINITY;
    const bool dense = A.dmean != nullptr || (!A.sigmoid && !A.renorm);
    float p[V], total = 0.f, inv = 0.f;
    if (dense) {
#pragma unroll
      for (int v = 0; v < V; v++) {
        p[v] = z[v] == -INFINITY ? 0.f : A.sigmoid ? sigmoid_from(z[v], fminf(m, 0.f)) : exp_from(z[v], m);
        total += p[v];
      }
      total = warp_sum(total);
      inv = total > 0.f ? __fdividef(1.f, total) : 0.f;
#pragma unroll
      for (int v = 0; v < V; v++) p[v] *= inv;
    }
    float own = 0.f, all = 0.f;      // what lane j's expert gets, and what every expert gets times its p
    if (A.renorm) {
      const float top = warp_max(zj);
      float q = zj == -INFINITY ? 0.f : A.sigmoid ? sigmoid_from(zj, fminf(top, 0.f)) : exp_from(zj, top);
      const float sum = warp_sum(q);
      q = sum > 0.f ? __fdividef(q, sum) : 0.f;
      own = q * (g - warp_sum(q * g));
      if (A.sigmoid) own *= sigmoid_fine(-zj);
    } else if (A.sigmoid) {
      own = zj == -INFINITY ? 0.f : g * sigmoid_fine(zj) * sigmoid_fine(-zj);
    } else {
      const float pj = zj == -INFINITY ? 0.f : exp_from(zj, m) * inv;
      all = -warp_sum(pj * g);
      own = pj * g;
    }
    if (A.dmean != nullptr) {
      float h[V], dot = 0.f;
#pragma unroll
      for (int v = 0; v < V; v++) {
        const int i = v * 32 + lane;
        h[v] = i < E ? __ldg(A.dmean + i) * inv_n : 0.f;
        dot = fmaf(p[v], h[v], dot);
      }
      dot = warp_sum(dot);
#pragma unroll
      for (int v = 0; v < V; v++) {
        const float r = p[v] * (h[v] - dot);
        d[v] = z[v] == -INFINITY ? 0.f : A.sigmoid ? r * sigmoid_fine(-z[v]) : r;
      }
    }
    if (!A.sigmoid && !A.renorm) {
#pragma unroll
      for (int v = 0; v < V; v++) d[v] = fmaf(p[v], all, d[v]);
    }
    for (int x = 0; x < A.k; x++) {      // (the same expert twice gets both)
      const int e = __shfl_sync(0xffffffffu, mine, x);
      const float o = __shfl_sync(0xffffffffu, own, x);
      if (e >= 0 && (e & 31) == lane) {
#pragma unroll
        for (int v = 0; v < V; v++)
          if (v == e >> 5) d[v] += o;
      }
    }
    T* out = (T*)A.dlogits + n * E;
#pragma unroll
    for (int v = 0; v < V; v++) {
      const int i = v * 32 + lane;
      if (i < E) out[i] = (T)d[v];
    }
  }
}

// A warp has a token, or some where the blocks' sums of probabilities are to be added up (or there are very many tokens)
int route_blocks(long N, bool sums) {
  const long want = (N + ROUTE_WARPS - 1) / ROUTE_WARPS, most = sums ? (long)mlb_sm_count() * 4 : 1L << 16;
  return (int)std::max(1L, std::min(want, most));
}
constexpr size_t ROUTE_LISTS = sizeof(uint2) * ROUTE_WARPS * LIST;
template <auto KERN>
int launch_route(const RouteArgs& A, int blocks, size_t smem, cudaStream_t st) {
  if (smem > 48 * 1024) {
    static std::atomic<unsigned long long> done{0};
    const cudaError_t e = mlb_allow_smem(KERN, ROUTE_LISTS + sizeof(double) * ROUTE_WARPS * MAX_E, done);
    if (e != cudaSuccess) return (int)e;
  }
  return (int)mlb_launch(KERN, dim3(blocks), dim3(32 * ROUTE_WARPS), smem, st, A);
}
template <typename F>
int by_width(int E, F&& f) {
  if (E <= 32) return f(std::integral_constant<int, 1>());
  if (E <= 64) return f(std::integral_constant<int, 2>());
  if (E <= 128) return f(std::integral_constant<int, 4>());
  if (E <= 256) return f(std::integral_constant<int, 8>());
  if (E <= 512) return f(std::integral_constant<int, 16>());
  return f(std::integral_constant<int, 32>());
}

}  // namespace

// floats of the workspace of a call with means
MLB_API long mlb_moe_route_part(long N, int E) { return (long)route_blocks(N, true) * E; }
MLB_API int mlb_moe_route(void* weights, int* idx, float* mean, float* part, const void* logits, const float* bias, long N, long ld, int E, int k, int sigmoid, int groups, int top, int renorm,
                          float scale, int zbits, int wbits, cudaStream_t st) {
  if (N < 0 || E < 1 || E > MAX_E || k < 1 || k > MAX_K || k > E || groups < 1 || groups > MAX_GROUPS || E % groups != 0 || top < 1 || top > groups || (zbits != 16 && zbits != 32) ||
      (wbits != 16 && wbits != 32))
    return -7;
  if (N == 0) return 0;
  const RouteArgs A = {logits, bias, weights, idx, mean ? part : nullptr, N, ld, E, k, groups, top, sigmoid, renorm, wbits == 32, scale};
  const int blocks = route_blocks(N, mean != nullptr);
  const bool plain = bias == nullptr && groups == 1;
  const size_t smem = std::max(ROUTE_LISTS + (plain ? 0 : sizeof(double) * ROUTE_WARPS * own_doubles(E)), mean ? sizeof(float) * ROUTE_WARPS * E : 0);
  int rc = by_width(E, [&](auto V) {
    if (plain) return zbits == 16 ? launch_route<moe_route_k<V.value, bf16, true>>(A, blocks, smem, st) : launch_route<moe_route_k<V.value, float, true>>(A, blocks, smem, st);
    return zbits == 16 ? launch_route<moe_route_k<V.value, bf16, false>>(A, blocks, smem, st) : launch_route<moe_route_k<V.value, float, false>>(A, blocks, smem, st);
  });
  if (rc == 0 && mean != nullptr)
    rc = (int)mlb_launch(moe_mean_k, dim3((E + 31) / 32), dim3(1024), 0, st, mean, (const float*)part, blocks, E, 1.f / (float)N);
  return rc;
}
MLB_API int mlb_moe_route_bwd(void* dlogits, const void* dweights, const float* dmean, const void* logits, const int* idx, long N, long ld, int E, int k, int sigmoid, int renorm, float scale,
                              int zbits, int wbits, cudaStream_t st) {
  if (N < 0 || E < 1 || E > MAX_E || k < 1 || k > MAX_K || k > E || (zbits != 16 && zbits != 32) || (wbits != 16 && wbits != 32)) return -7;
  if (N == 0) return 0;
  const RouteBwdArgs A = {dlogits, dweights, logits, dmean, idx, N, ld, E, k, sigmoid, renorm, wbits == 32, scale};
  return by_width(E, [&](auto V) {
    auto go = [&](auto kern) { return (int)mlb_launch(kern, dim3(route_blocks(N, false)), dim3(32 * ROUTE_WARPS), 0, st, A); };
    return zbits == 16 ? go(moe_route_bwd_k<V.value, bf16>) : go(moe_route_bwd_k<V.value, float>);
  });
}
