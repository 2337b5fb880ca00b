// Routing of tokens to experts: the k best of E scores a token, their weights, the experts' mean probabilities, and the logits' gradient.
//
// A warp has a token, lane l the experts l, l + 32, ...  A logit of NaN counts as -inf and an expert at -inf is not there.  Scores are a softmax over the experts or a
// sigmoid each.  Experts are chosen by their logits, or, with a bias or groups, by score + bias in 64 bits: in 32 the last bits of two roundings would decide between
// neighbours, and another way of adding up would choose other experts.  Equal ones go to the lowest index.
#pragma once
#include <algorithm>
#include <type_traits>

#include "../common.cuh"

namespace {

constexpr int ROUTE_WARPS = 8, MAX_E = 1024, MAX_K = 32, MAX_GROUPS = 32;      // (ops/ref_moe.py refuses more)
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
template <typename T> __device__ __forceinline__ float logit(const T* z, int i);
template <> __device__ __forceinline__ float logit<float>(const float* z, int i) { return __ldg(z + i); }
template <> __device__ __forceinline__ float logit<bf16>(const bf16* z, int i) { return __bfloat162float(z[i]); }
// (NaN -> -inf, -0 -> 0)
__device__ __forceinline__ float seen(float z) { return z != z ? -INFINITY : z + 0.f; }
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
  return __fdiv_rn(z >= 0.f ? 1.f : e, 1.f + e);
}
// sigmoid(z) / exp(top) for top = min(0, largest z): scores for shares, whose sum is not too small for fp32
__device__ __forceinline__ float sigmoid_from(float z, float top) {
  return z == -INFINITY ? 0.f : z >= 0.f ? sigmoid_fine(z) : __fdiv_rn(exp_from(z, top), 1.f + exp_fine(fmaxf(z, -200.f)));
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
constexpr uint32_t GONE32 = 0x007fffffu;                    // order32(-inf)
constexpr uint64_t GONE64 = 0x000fffffffffffffull;          // order64(-inf)
template <typename K> __device__ __forceinline__ constexpr K gone() { return sizeof(K) == 4 ? (K)GONE32 : (K)GONE64; }
__device__ __forceinline__ uint32_t warp_best(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ uint64_t warp_best(uint64_t v) {
  const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return (uint64_t)hi << 32 | lo;
}

// The k best of the warp's keys, best first: lane j keeps the index of the j-th (-1: none left).
template <int V, typename K>
__device__ __forceinline__ int choose(K (&key)[V], int k, int lane) {
  int mine = -1;
  K best = key[0];
  int at = 0;
#pragma unroll
  for (int v = 1; v < V; v++)
    if (key[v] > best) best = key[v], at = v;
  for (int j = 0; j < k; j++) {
    const K top = warp_best(best);
    if (top <= gone<K>()) break;
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

template <int V, typename T>
__global__ void __launch_bounds__(32 * ROUTE_WARPS) moe_route_k(const RouteArgs A) {
  mlb_pdl_sync();
  extern __shared__ double route_sm[];      // with groups: the scores of each warp's token; behind the loop: sums of probabilities
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, E = A.E;
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
    float total = 0.f;      // of exp(z - m), or of scores relative to the largest
    if (A.part != nullptr || (!A.sigmoid && !A.renorm)) {
      float e[V];
#pragma unroll
      for (int v = 0; v < V; v++) {
        e[v] = z[v] == -INFINITY ? 0.f : A.sigmoid ? sigmoid_from(z[v], fminf(m, 0.f)) : exp_from(z[v], m);
        total += e[v];
      }
      total = warp_sum(total);
      if (A.part != nullptr) {
        const float inv = total > 0.f ? __fdiv_rn(1.f, total) : 0.f;
#pragma unroll
        for (int v = 0; v < V; v++) sum_p[v] = fmaf(e[v], inv, sum_p[v]);
      }
    }
    int mine;
    if (A.bias == nullptr && A.groups == 1) {
      uint32_t key[V];
#pragma unroll
      for (int v = 0; v < V; v++) key[v] = order32(z[v]);
      mine = choose<V>(key, A.k, lane);
    } else {
      double t[V], all = 0;
#pragma unroll
      for (int v = 0; v < V; v++) {
        t[v] = z[v] == -INFINITY ? 0.0 : A.sigmoid ? 1.0 / (1.0 + exp(-(double)z[v])) : z[v] == m ? 1.0 : exp((double)z[v] - (double)m);
        all += t[v];
      }
      if (!A.sigmoid) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
      }
#pragma unroll
      for (int v = 0; v < V; v++) {
        const int i = v * 32 + lane;
        if (!A.sigmoid) t[v] = all > 0 ? t[v] / all : 0.0;
        if (i < E && A.bias != nullptr) t[v] += (double)__ldg(A.bias + i);
        if (z[v] == -INFINITY) t[v] = -INFINITY;
      }
      if (A.groups > 1) {      // lane l has group l: its two best
        double* s = route_sm + w * E;
        const int size = E / A.groups;
#pragma unroll
        for (int v = 0; v < V; v++)
          if (v * 32 + lane < E) s[v * 32 + lane] = t[v];
        __syncwarp();
        double a = -INFINITY, b = -INFINITY;
        if (lane < A.groups)
          for (int j = 0, i = lane % size; j < size; j++, i = i + 1 == size ? 0 : i + 1) {      // (begun at another place by each lane: other banks)
            const double x = s[lane * size + i];
            if (x > a) b = a, a = x;
            else if (x > b) b = x;
          }
        __syncwarp();
        uint64_t key[1] = {lane < A.groups ? order64(a + (b > -INFINITY ? b : 0.0)) : 0};
        unsigned stays = 0;
        for (int j = 0; j < A.top; j++) {
          const uint64_t best = warp_best(key[0]);
          const int g = __ffs(__ballot_sync(0xffffffffu, key[0] == best)) - 1;
          stays |= 1u << g;
          if (lane == g) key[0] = 0;
        }
#pragma unroll
        for (int v = 0; v < V; v++)
          if (v * 32 + lane < E && !((stays >> ((v * 32 + lane) / size)) & 1)) t[v] = -INFINITY;
      }
      uint64_t key[V];
#pragma unroll
      for (int v = 0; v < V; v++) key[v] = order64(t[v]);
      mine = choose<V>(key, A.k, lane);
    }
    // lane j: the weight of the j-th
    const float zj = mine >= 0 ? seen(logit(row, mine)) : -INFINITY;
    float wj = 0.f;
    if (A.renorm) {      // relative to the largest chosen one, so that the sum is not too small for fp32
      const float top = warp_max(zj);
      wj = zj == -INFINITY ? 0.f : A.sigmoid ? sigmoid_from(zj, fminf(top, 0.f)) : exp_from(zj, top);
      const float sum = warp_sum(wj);
      wj = sum > 0.f ? __fdiv_rn(wj, sum) : 0.f;
    } else if (zj > -INFINITY) {
      wj = A.sigmoid ? sigmoid_fine(zj) : __fdiv_rn(exp_from(zj, m), total);
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
// mean[e] = the blocks' sums / N: 8 threads to an expert, always the same blocks to a thread
__global__ void __launch_bounds__(256) moe_mean_k(float* mean, const float* __restrict__ part, int blocks, int E, float inv) {
  mlb_pdl_sync();
  const int e = blockIdx.x * 32 + (threadIdx.x & 31), s = threadIdx.x >> 5;
  __shared__ float red[8][32];
  float t = 0.f;
  if (e < E) {
#pragma unroll 8
    for (int b = s; b < blocks; b += 8) t += part[(long)b * E + e];
  }
  red[s][threadIdx.x & 31] = t;
  __syncthreads();
  if (s == 0 && e < E) {
    t = 0.f;
#pragma unroll
    for (int k = 0; k < 8; k++) t += red[k][threadIdx.x];
    mean[e] = t * inv;
  }
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
      inv = total > 0.f ? __fdiv_rn(1.f, total) : 0.f;
#pragma unroll
      for (int v = 0; v < V; v++) p[v] *= inv;
    }
    float own = 0.f, all = 0.f;      // what lane j's expert gets, and what every expert gets times its p
    if (A.renorm) {
      const float top = warp_max(zj);
      float q = zj == -INFINITY ? 0.f : A.sigmoid ? sigmoid_from(zj, fminf(top, 0.f)) : exp_from(zj, top);
      const float sum = warp_sum(q);
      q = sum > 0.f ? __fdiv_rn(q, sum) : 0.f;
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

int route_blocks(long N, int E) {
  const long want = (N + ROUTE_WARPS - 1) / ROUTE_WARPS, most = (long)mlb_sm_count() * 6;
  return (int)std::max(1L, std::min(want, most));
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
MLB_API long mlb_moe_route_part(long N, int E) { return (long)route_blocks(N, E) * E; }
MLB_API int mlb_moe_route(void* weights, int* idx, float* mean, float* part, const void* logits, const float* bias, long N, long ld, int E, int k, int sigmoid, int groups, int top, int renorm,
                          float scale, int zbits, int wbits, cudaStream_t st) {
  if (N < 0 || E < 1 || E > MAX_E || k < 1 || k > MAX_K || k > E || groups < 1 || groups > MAX_GROUPS || E % groups != 0 || top < 1 || top > groups || (zbits != 16 && zbits != 32) ||
      (wbits != 16 && wbits != 32))
    return -7;
  if (N == 0) return 0;
  const RouteArgs A = {logits, bias, weights, idx, mean ? part : nullptr, N, ld, E, k, groups, top, sigmoid, renorm, wbits == 32, scale};
  const int blocks = route_blocks(N, E);
  const size_t smem = std::max(groups > 1 ? sizeof(double) * ROUTE_WARPS * E : 0, mean ? sizeof(float) * ROUTE_WARPS * E : 0);
  int rc = by_width(E, [&](auto V) {
    auto go = [&](auto kern) {
      if (smem > 48 * 1024) {
        static std::atomic<unsigned long long> done{0};
        const cudaError_t e = mlb_allow_smem(kern, sizeof(double) * ROUTE_WARPS * MAX_E, done);
        if (e != cudaSuccess) return (int)e;
      }
      return (int)mlb_launch(kern, dim3(blocks), dim3(32 * ROUTE_WARPS), smem, st, A);
    };
    return zbits == 16 ? go(moe_route_k<V.value, bf16>) : go(moe_route_k<V.value, float>);
  });
  if (rc == 0 && mean != nullptr)
    rc = (int)mlb_launch(moe_mean_k, dim3((E + 31) / 32), dim3(256), 0, st, mean, (const float*)part, blocks, E, 1.f / (float)N);
  return rc;
}
MLB_API int mlb_moe_route_bwd(void* dlogits, const void* dweights, const float* dmean, const void* logits, const int* idx, long N, long ld, int E, int k, int sigmoid, int renorm, float scale,
                              int zbits, int wbits, cudaStream_t st) {
  if (N < 0 || E < 1 || E > MAX_E || k < 1 || k > MAX_K || k > E || (zbits != 16 && zbits != 32) || (wbits != 16 && wbits != 32)) return -7;
  if (N == 0) return 0;
  const RouteBwdArgs A = {dlogits, dweights, logits, dmean, idx, N, ld, E, k, sigmoid, renorm, wbits == 32, scale};
  return by_width(E, [&](auto V) {
    auto go = [&](auto kern) { return (int)mlb_launch(kern, dim3(route_blocks(N, E)), dim3(32 * ROUTE_WARPS), 0, st, A); };
    return zbits == 16 ? go(moe_route_bwd_k<V.value, bf16>) : go(moe_route_bwd_k<V.value, float>);
  });
}
