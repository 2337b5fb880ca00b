// Key / value cache held in 4 bits: writing new tokens into it (with rotary embedding), reading them back, attention over it.
//
// Layout.  pages[n_pages][Hkv][page / 16][18 hd] bytes: a block of 16 tokens of one head is one contiguous piece that a single bulk copy fetches, so
// that the page size only says how finely the pool is dealt out.  In a block: 16 rows of key codes (hd / 2 bytes each), 16 rows of value codes, 16
// rows of key scales (NG = hd / 32 bf16), 16 rows of value scales.  32 neighbouring elements (a group g) of a row share the scale s; code c in 0..15
// stands for (c - 8) s.  s = -m / 8 rounded to bf16, m the element of largest magnitude (of a tie the negative one): it gets code 0 and is held exactly
// where s is, and the step is 1/8 of the largest magnitude instead of the 1/7 of a scale without a sign.
// The order in a row is that of the matrix instructions' registers in the attention kernel (lane = 4 i + j):
//   key row:   32-bit word j NG + g has the elements 32 g + 8 j + e, e = 0..7, in its e-th four bits
//   value row: 16-bit word i NG + g has the elements 32 g + 4 i + e, e = 0..3
#include <cuda_fp16.h>

#include <type_traits>

#include "tc.cuh"

namespace {

MLB_DEFINE_ERROR_WORD(kv4)

constexpr int TOK = 16;                 // tokens of a block
template <int HD> struct Block {
  static constexpr int NG = HD / 32, ROW = HD / 2, BYTES = 18 * HD;
  static constexpr int V = 8 * HD, KS = 16 * HD, VS = 17 * HD;      // where value codes, key scales and value scales begin
};
constexpr float TINY = 7.52316385e-37f;      // 2^-120: a smaller scale is held as 0 (below it quotients would meet subnormal numbers)

__device__ __forceinline__ float bf16_bits(uint32_t hi) { return __uint_as_float(hi << 16); }
__device__ __forceinline__ float lo_bf16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_bf16(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

__device__ __forceinline__ uint32_t low_codes(uint32_t w) { return w & 0x000F000Fu; }       // two codes as fp16 c 2^-24
__device__ __forceinline__ uint32_t high_codes(uint32_t w) { return w & 0x00F000F0u; }      // c 2^-20
__device__ __forceinline__ uint32_t less(uint32_t x, uint32_t k) {      // of two bf16 numbers
  const bf162 y = __hsub2(*reinterpret_cast<const bf162*>(&x), *reinterpret_cast<const bf162*>(&k));
  return *reinterpret_cast<const uint32_t*>(&y);
}
__device__ __forceinline__ uint32_t value_codes(uint32_t w) { return less(low_codes(w) | 0x43004300u, 0x43084308u); }      // two codes as bf16 c - 8: 128 + c, 136
__device__ __forceinline__ uint32_t sixteen_times(uint32_t w) {
  const uint32_t k = 0x41804180u;
  const bf162 y = __hmul2(*reinterpret_cast<const bf162*>(&w), *reinterpret_cast<const bf162*>(&k));
  return *reinterpret_cast<const uint32_t*>(&y);
}
// ------------------------------------------------------------------ append
// A thread has 8 neighbouring elements of one head, 4 threads a group, and goes over rows.  Products and sums of the rotation are rounded one by one, so that the value
// which is cut to 4 bits does not depend on what the compiler contracts (a packed product and sum of two values did come out contracted).  Bound by the bytes of the
// rows, and as much by instructions, some 200 for 8 elements, so the quotients share a reciprocal and the codes are put together by multiply-adds.
// 8192 rows of 12 + 24 heads of 64, written and read back by the kernel below: 23.6 us, 3.8 TB/s of what has to move; 16 rows of 16 + 32 heads of 128: 3.6 us.
__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int k = 0; k < 4; k++) x[2 * k] = lo_bf16(u[k]), x[2 * k + 1] = hi_bf16(u[k]);
}
// Two numbers an instruction, each rounded as by itself
struct Pair { unsigned long long v; };
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ void split(Pair p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair p;
  asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(a.v), "l"(b.v));
  return p;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair p;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(p.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return p;
}
struct Group { uint32_t codes; uint16_t scale; };
// x / s as rounded to nearest: the rounded reciprocal's product corrected by its remainder is that (Markstein, Computation of elementary functions on the IBM RISC
// System/6000 processor, 1990), as long as nothing on the way is subnormal
__device__ __forceinline__ Pair quotients(Pair x, Pair minus_s, Pair rs) {
  const Pair q = mul2(x, rs);
  return fma2(fma2(q, minus_s, x), rs, q);
}
__device__ __forceinline__ Group to_codes(const float (&x)[8], unsigned mask) {
  // a number's bits turned left by one have its magnitude above its sign: the largest are of the largest magnitude, of a tie the negative one's
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) top = max(top, __funnelshift_l(__float_as_uint(x[e]), __float_as_uint(x[e]), 1));
  top = max(top, __shfl_xor_sync(mask, top, 1));
  top = max(top, __shfl_xor_sync(mask, top, 2));
  const bf16 sb = __float2bfloat16_rn(__uint_as_float(__funnelshift_r(top, top, 1)) * -0.125f);
  const float s = __bfloat162float(sb);
  Group g{0x88888888u, __bfloat16_as_ushort(sb)};
  if (top >= 0xFF000000u) {      // an infinity or NaN among them
    g.scale = 0x7FC0;      // NaN
  } else if (fabsf(s) < TINY) {
    g.scale = 0;
  } else {
    // Quotients go from -8 to 8 and the scale's rounding: 8 alone is one code too many.  1.5 2^23 + 8: the sum's last bits are the quotient rounded to nearest even, + 8
    uint32_t w = 0;
    auto add = [&](float q) { w = w * 16u + __float_as_uint(fminf(q, 7.f) + 12582920.f); };
    if (fabsf(s) >= 8.67361738e-19f) {      // 2^-60
      const float rs = __frcp_rn(s);
      const Pair rr = pair(rs, rs), ms = pair(-s, -s);
#pragma unroll
      for (int e = 6; e >= 0; e -= 2) {
        float a, b;
        split(quotients(pair(x[e], x[e + 1]), ms, rr), a, b);
        add(b), add(a);
      }
    } else {
#pragma unroll 1
      for (int e = 7; e >= 0; e--) add(__fdiv_rn(x[e], s));
    }
    g.codes = w - 0x3F400000u;      // (the constant's other bits, 0x4B400000 at each of the 8 places, modulo 2^32)
  }
  return g;
}

template <int HD>
__global__ void __launch_bounds__(512, 2) kv4_append_k(uint8_t* __restrict__ pages, bf16* __restrict__ q_out, const bf16* __restrict__ qkv,
                                                    const int* __restrict__ slots, const int* __restrict__ pos, const float* __restrict__ cos,
                                                    const float* __restrict__ sin, long n_pages, int page_log, int N, long stride, int H, int Hkv, int T) {
  mlb_pdl_sync();
  using L = Block<HD>;
  constexpr int PER = HD / 8, HALF = PER / 2, NG = L::NG;
  const int idx = blockIdx.x * blockDim.x + threadIdx.x, head = idx / PER, t = idx % PER, j = t & 3, g = t >> 2;
  const bool any = head < H + 2 * Hkv, query = head < H, value = head >= H + Hkv, turn = cos != nullptr && head < H + Hkv;
  const int kv = head - H - (value ? Hkv : 0);
  const unsigned group = __ballot_sync(0xffffffffu, any && !query);      // lanes that cut their elements to codes
  if (!any || (query && q_out == nullptr)) return;
  const int other = 8 * (t < HALF ? t + HALF : t - HALF), angle = 8 * (t < HALF ? t : t - HALF);
  const uint32_t minus = t < HALF ? 0x80008000u : 0u;      // the first half loses what the second one gains
  const bf16* src = qkv + (long)head * HD;
  // the next row is on its way while one is worked on
  int row = blockIdx.y, slot = 0, p = 0;
  uint4 near = {0, 0, 0, 0}, far = near;
  auto fetch = [&] {
    if (row >= N) return;
    const bf16* r = src + row * stride;
    near = *reinterpret_cast<const uint4*>(r + 8 * t);
    if (turn) far = *reinterpret_cast<const uint4*>(r + other), p = pos[row];
    if (!query) slot = slots[row];
  };
  fetch();
#pragma unroll 1
  for (int now = row; now < N; now = row) {
    float x[8];
    unpack8(near, x);
    const int here = slot;
    if (turn) {
      if (p < 0 || p >= T) {
        if (t == 0) mlb_set_error(MLB_ERR_BOUNDS, 0xC3);
        p = 0;
      }
      float y[8];
      far.x ^= minus, far.y ^= minus, far.z ^= minus, far.w ^= minus;
      unpack8(far, y);
      const float4* cp = reinterpret_cast<const float4*>(cos + (long)p * (HD / 2) + angle);
      const float4* sp = reinterpret_cast<const float4*>(sin + (long)p * (HD / 2) + angle);
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const float4 c = cp[k], s = sp[k];
        const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int e = 0; e < 4; e++) x[4 * k + e] = __fadd_rn(__fmul_rn(x[4 * k + e], cc[e]), __fmul_rn(y[4 * k + e], ss[e]));
      }
    }
    row += gridDim.y;
    fetch();
    if (query) {
      const uint4 w = {pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
      *reinterpret_cast<uint4*>(q_out + ((long)now * H + head) * HD + 8 * t) = w;
      continue;
    }
    if (here < 0) continue;      // (all lanes of a row's group go together)
    const int pg = here >> page_log, off = here & ((1 << page_log) - 1), r = off % TOK;
    if (pg >= n_pages) {
      if (t == 0) mlb_set_error(MLB_ERR_BOUNDS, 0xC2);
      continue;
    }
    const Group c = to_codes(x, group);
    uint8_t* b = pages + ((((long)pg * Hkv + kv) << (page_log - 4)) + off / TOK) * L::BYTES;
    if (!value) {
      *reinterpret_cast<uint32_t*>(b + r * L::ROW + 4 * (j * NG + g)) = c.codes;
    } else {
      uint8_t* v = b + L::V + r * L::ROW;
      *reinterpret_cast<uint16_t*>(v + 2 * (2 * j * NG + g)) = (uint16_t)c.codes;
      *reinterpret_cast<uint16_t*>(v + 2 * ((2 * j + 1) * NG + g)) = (uint16_t)(c.codes >> 16);
    }
    if (j == 0) *reinterpret_cast<uint16_t*>(b + (value ? L::VS : L::KS) + 2 * (r * NG + g)) = c.scale;
  }
}

// Head sizes 64 and 128, whose halves are whole groups: a thread has the 8 elements of both halves that the rotation mixes, so rows, angles and addresses are fetched and
// unpacked once for 16 elements (8192 rows of 36 heads of 64, written and read back: 25.4 us then, 27.7 with 8 a thread).
template <int HD>
__global__ void __launch_bounds__(512, 2) kv4_append_halves_k(uint8_t* __restrict__ pages, bf16* __restrict__ q_out, const bf16* __restrict__ qkv,
                                                              const int* __restrict__ slots, const int* __restrict__ pos, const float* __restrict__ cos,
                                                              const float* __restrict__ sin, long n_pages, int page_log, int N, long stride, int H, int Hkv, int T) {
  mlb_pdl_sync();
  using L = Block<HD>;
  constexpr int PER = HD / 16, NG = L::NG;
  const int idx = blockIdx.x * blockDim.x + threadIdx.x, head = idx / PER, t = idx % PER, j = t & 3, g = t >> 2;      // groups g and g + NG / 2
  const bool any = head < H + 2 * Hkv, query = head < H, value = head >= H + Hkv, turn = cos != nullptr && head < H + Hkv;
  const int kv = head - H - (value ? Hkv : 0);
  const unsigned group = __ballot_sync(0xffffffffu, any && !query), values = __ballot_sync(0xffffffffu, any && value);      // lanes that cut their elements to codes
  if (!any || (query && q_out == nullptr)) return;
  const bf16* src = qkv + (long)head * HD + 8 * t;
  // the next row is on its way while one is worked on
  int row = blockIdx.y, slot = 0, p = 0;
  uint4 low = {0, 0, 0, 0}, high = low;
  auto fetch = [&] {
    if (row >= N) return;
    const bf16* r = src + row * stride;
    low = *reinterpret_cast<const uint4*>(r), high = *reinterpret_cast<const uint4*>(r + HD / 2);
    if (turn) p = pos[row];
    if (!query) slot = slots[row];
  };
  fetch();
#pragma unroll 1
  for (int now = row; now < N; now = row) {
    float x[8], y[8];
    unpack8(low, x);
    unpack8(high, y);
    const int here = slot;
    if (turn) {
      if (p < 0 || p >= T) {
        if (t == 0) mlb_set_error(MLB_ERR_BOUNDS, 0xC3);
        p = 0;
      }
      const float4* cp = reinterpret_cast<const float4*>(cos + (long)p * (HD / 2) + 8 * t);
      const float4* sp = reinterpret_cast<const float4*>(sin + (long)p * (HD / 2) + 8 * t);
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const float4 cv = cp[k], sv = sp[k];
        const float c[4] = {cv.x, cv.y, cv.z, cv.w}, s[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float a = x[4 * k + e], b = y[4 * k + e];
          x[4 * k + e] = __fsub_rn(__fmul_rn(a, c[e]), __fmul_rn(b, s[e]));
          y[4 * k + e] = __fadd_rn(__fmul_rn(b, c[e]), __fmul_rn(a, s[e]));
        }
      }
    }
    row += gridDim.y;
    fetch();
    if (query) {
      bf16* to = q_out + ((long)now * H + head) * HD + 8 * t;
      *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
      *reinterpret_cast<uint4*>(to + HD / 2) = make_uint4(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]), pack_bf16(y[4], y[5]), pack_bf16(y[6], y[7]));
      continue;
    }
    if (here < 0) continue;      // (all lanes of a row's group go together)
    const int pg = here >> page_log, off = here & ((1 << page_log) - 1), r = off % TOK;
    if (pg >= n_pages) {
      if (t == 0) mlb_set_error(MLB_ERR_BOUNDS, 0xC2);
      continue;
    }
    const Group a = to_codes(x, group), b = to_codes(y, group);
    uint8_t* blk = pages + ((((long)pg * Hkv + kv) << (page_log - 4)) + off / TOK) * L::BYTES;
    uint8_t* codes = blk + (value ? L::V : 0) + r * L::ROW;
    uint8_t* scale = blk + (value ? L::VS : L::KS) + 2 * (r * NG + g);
    if constexpr (NG == 2) {      // both groups of the row
      const uint2 w = value ? make_uint2(__byte_perm(a.codes, b.codes, 0x5410), __byte_perm(a.codes, b.codes, 0x7632)) : make_uint2(a.codes, b.codes);
      *reinterpret_cast<uint2*>(codes + 8 * j) = w;
      if (j == 0) *reinterpret_cast<uint32_t*>(scale) = a.scale | (uint32_t)b.scale << 16;
    } else {
      if (value) {      // a 64-bit unit has a half of all four groups: lanes of groups 0, 2 and of 1, 3 swap theirs, and have unit 2 j and unit 2 j + 1
        const uint32_t give = g == 0 ? __byte_perm(a.codes, b.codes, 0x7632) : __byte_perm(a.codes, b.codes, 0x5410);
        const uint32_t keep = g == 0 ? __byte_perm(a.codes, b.codes, 0x5410) : __byte_perm(a.codes, b.codes, 0x7632);
        const uint32_t got = __shfl_xor_sync(values, give, 4);
        const uint2 w = g == 0 ? make_uint2(__byte_perm(keep, got, 0x5410), __byte_perm(keep, got, 0x7632))
                               : make_uint2(__byte_perm(got, keep, 0x5410), __byte_perm(got, keep, 0x7632));
        *reinterpret_cast<uint2*>(codes + 8 * (2 * j + g)) = w;
      } else {
        *reinterpret_cast<uint32_t*>(codes + 4 * (j * NG + g)) = a.codes;
        *reinterpret_cast<uint32_t*>(codes + 4 * (j * NG + g + 2)) = b.codes;
      }
      if (j == 0) *reinterpret_cast<uint16_t*>(scale) = a.scale, *reinterpret_cast<uint16_t*>(scale + 4) = b.scale;
    }
  }
}

// ------------------------------------------------------------------ read
template <int HD>
__global__ void __launch_bounds__(512, 3) kv4_read_k(bf16* __restrict__ k, bf16* __restrict__ v, const uint8_t* __restrict__ pages, const int* __restrict__ slots,
                                                     long n_pages, int page_log, int N, int Hkv) {
  mlb_pdl_sync();
  using L = Block<HD>;
  constexpr int PER = HD / 8;
  const int idx = blockIdx.x * blockDim.x + threadIdx.x, t = idx % PER, kv = idx / PER, j = t & 3, gi = t >> 2;
  if (kv >= Hkv) return;
#pragma unroll 1
  for (int row = blockIdx.y; row < N; row += gridDim.y) {
    const int slot = slots[row], pg = slot >> page_log;
    uint4 wk = {0, 0, 0, 0}, wv = wk;
    if (slot >= 0 && pg >= n_pages) {
      if (t == 0 && kv == 0) mlb_set_error(MLB_ERR_BOUNDS, 0xC2);
    } else if (slot >= 0) {
      const int off = slot & ((1 << page_log) - 1), r = off % TOK;
      const uint8_t* b = pages + ((((long)pg * Hkv + kv) << (page_log - 4)) + off / TOK) * L::BYTES;
      const uint16_t* h = reinterpret_cast<const uint16_t*>(b + L::V + r * L::ROW);
      const uint32_t ck = *reinterpret_cast<const uint32_t*>(b + r * L::ROW + 4 * (j * L::NG + gi));
      const uint32_t cv = h[2 * j * L::NG + gi] | (uint32_t)h[(2 * j + 1) * L::NG + gi] << 16;
      const uint32_t sk = *reinterpret_cast<const uint16_t*>(b + L::KS + 2 * (r * L::NG + gi)) * 0x10001u;
      const uint32_t sv = *reinterpret_cast<const uint16_t*>(b + L::VS + 2 * (r * L::NG + gi)) * 0x10001u;
      // (c - 8) s rounded once: both factors are bf16 numbers
      auto values = [](uint32_t c, uint32_t s) {
        const uint32_t a = value_codes(c), b = value_codes(c >> 4), d = value_codes(c >> 8), e = value_codes(c >> 12);      // elements 0 4, 1 5, 2 6, 3 7
        auto times = [&](uint32_t x) {
          const bf162 y = __hmul2(*reinterpret_cast<const bf162*>(&x), *reinterpret_cast<const bf162*>(&s));
          return *reinterpret_cast<const uint32_t*>(&y);
        };
        return make_uint4(times(__byte_perm(a, b, 0x5410)), times(__byte_perm(d, e, 0x5410)), times(__byte_perm(a, b, 0x7632)), times(__byte_perm(d, e, 0x7632)));
      };
      wk = values(ck, sk);
      wv = values(cv, sv);
    }
    const long to = ((long)row * Hkv + kv) * HD + 8 * t;
    *reinterpret_cast<uint4*>(k + to) = wk;
    *reinterpret_cast<uint4*>(v + to) = wv;
  }
}

// ------------------------------------------------------------------ attention
// O[r] = sum_t p_rt (c_t - 8) s_t / sum_t p_rt,  p_rt = exp(scale q_r . k_t - m_r), over the tokens t that query row r sees; r runs over the G = H / Hkv
// heads and the Tq tokens that share a key / value head, 8 NT of them at a time.
//
// Bound by the cache's bytes (4.5 bits an element), as long as an SM's 4 issue slots keep up with the 23 bytes a clock that reach it: 16 tokens of
// 128 + 128 elements are 98 clocks, 390 instructions.  So the tensor cores do both products (mma.sync, tokens or elements as the 16 rows, query rows as
// the 8 columns: tcgen05 would want 128 rows and its operands unpacked to shared memory).  What the codes become is as few instructions as can be:
//   K: four bits at the bottom of a 16-bit word are the fp16 number c 2^-24, the next four c 2^-20 (both subnormal, both exact), so one bitwise instruction
//      makes two operands and only the upper byte's codes need a shift; the factor 16 is taken out of the queries, which a power of two of each row brings to fp16
//      exactly.  The product starts from -8 sum(q) instead of subtracting 8 from each code; every group's sum is scaled by s_t behind its two
//      products, in fp32.  (The tensor core lines products up by their operands' nominal exponents, 2^-14 for a subnormal: a score is off by some 2^-16 of |q| s.)
//   V: the same bits as bf16 numbers are c 2^-133 and 16 c 2^-133 (these reach into the exponent's last bit, and are counted on without a gap there), less 8 and 128
//      of which all is exact and what is 0 adds 0: two instructions for two codes, a shift for eight.  For the products' sake the weights are 2^88 times what they are
//      (a sum of 2^31 of them, each up to 2^8, still is a number), O is 2^-45 times: what a token adds below 2^-81 is lost, and with a scale of 2^31 and more a weight
//      may pass bf16's range.  So a warp looks at its O.  Where that is not finite, or all of a group below 2^-50 (zeros are, too), it goes over its blocks once more with codes as
//      numbers of the size that they are, and O 2^-45 or 2^48 times.  Shares are averages times 2^-5 and the power of two that brings their sum of weights to 1 ... 2: the
//      cache's smallest number, 2^-120, and its largest ones stay what they are.  (What is below 2^-81 stays lost beside more than 2^-50 in its own
//      group, and beside more than some 2^50, which 2^48 times would pass fp32's range, in any.)
//      The scale goes into P, in fp32 before its one rounding to bf16.  That rounding, 2^-8 of each weight at most and independent from token to token, is
//      the only one on the way to O.  (Codes as 128 + c less 136 with the weights as they are, a shift for each two: 64 x 8192 tokens, below, 91 us instead of 79.  The
//      8 or 128 taken off by a product with a constant was no faster, 82, and leaves 2^-24 of a weight where the code stands for 0.)
// Scores stand transposed (token rows, query columns), so that softmax weights become the second product's operand by two matrix transpositions in
// registers.  The largest score m is the reference of all weights so far and moves only when a score passes it by 2^8 (O and the sums are then rescaled): most
// blocks need a vote instead of reductions over the warp.
//
// Work: all heads' blocks of 16 tokens stand in one row of units, each thread block takes an equal piece of it whatever the lengths are, and its 4 warps a quarter
// each of every head's part in it.  A head has PAD more units, which stand for what it costs to begin and end one (without them, 16 sequences of up to 2048 tokens
// took 39 us where two of them were empty, and 23 with 2 units).  A warp fetches its own blocks by bulk copies through a ring of its own.  A head whose blocks are
// shared is put together by the thread block that comes last, in the order of the pieces, so that a call repeats its bits.
//
// Measured: 64 sequences of 1024 to 8192 tokens, 32 heads over 8 of 128: 79 us, 4.4 TB/s (67 % of the measured copy rate; 60 us with the arithmetic left out.  What is
// missing is instructions, 306 a block, of which 146 go through the pipe of bitwise operations and shifts at half the rate, and that three warps an issue slot
// leave 44 % of the slots empty).  16 sequences of up to 2048 tokens, 16 heads of 128: 21.1 us, of which some 9 are that arithmetic and 8 beginnings, ends and
// the joining of shares.  One sequence of 1000 tokens, 12 heads of 64: 6.8 us, 1.4 of them an empty kernel's, 2.4 the joining (a counter, another block's
// results).  12 warps an SM: 8 are 4 to 8 % slower, 16 (of 128 registers, with places of 32 tokens) 79 -> 85.
struct AttnArgs {
  bf16* out;
  float* lse;
  const bf16* q;
  const uint8_t* pages;
  const int *table, *lens;
  float* part;
  int* count;
  long q_stride, n_pages;
  int B, Tq, G, Hkv, width, page_log;
  float scale_log2;            // > 0: a negative scale turns the queries' signs, and none makes them zeros
  uint32_t q_keep, q_flip;
  float inv_g;
};
constexpr int WARPS = 4;
constexpr int MAX_B = 2048;       // sequences of a launch: their first blocks' numbers stand in shared memory
// A warp's ring: N places of STEP blocks (hd = 128: 3 thread blocks' rings fill an SM's shared memory), which are worked on two at a time.  PAD: see the kernel
constexpr int STEP = 4, PAD = 12;
constexpr int PER_SM = 3;      // thread blocks that an SM holds (of 2 where the sequences' numbers leave no room for the third's ring)
template <int HD> struct Ring { static constexpr int N = HD == 64 ? 3 : HD == 32 ? 6 : 2, BYTES = STEP * Block<HD>::BYTES; };

// D = A B + C: keys' codes and queries in fp16, values' codes and weights in bf16
__device__ __forceinline__ void mma_keys(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1, float c2,
                                         float c3) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma_values(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int N> struct Words { uint32_t w[N]; };
template <int N> __device__ __forceinline__ Words<N> load_words(const uint8_t* p) {      // N 32-bit words at a multiple of 4 N bytes (3: of 4)
  Words<N> r;
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    r.w[0] = v.x, r.w[1] = v.y;
  } else {
#pragma unroll
    for (int k = 0; k < N; k++) r.w[k] = *reinterpret_cast<const uint32_t*>(p + 4 * k);
  }
  return r;
}
template <int N> __device__ __forceinline__ void load_halves(const uint8_t* p, uint32_t (&h)[N]) {      // N 16-bit words: value h[g] in the low half
  if constexpr (N % 2 == 0) {
    const auto r = load_words<N / 2>(p);
#pragma unroll
    for (int k = 0; k < N; k++) h[k] = k % 2 ? r.w[k / 2] >> 16 : r.w[k / 2];
  } else {
#pragma unroll
    for (int k = 0; k < N; k++) h[k] = *reinterpret_cast<const uint16_t*>(p + 2 * k);
  }
}
template <int N> __device__ __forceinline__ void load_scales(const uint8_t* p, float (&s)[N]) {
  uint32_t h[N];
  load_halves<N>(p, h);
#pragma unroll
  for (int k = 0; k < N; k++) s[k] = bf16_bits(h[k]);
}

template <int HD, int NT> struct Rows {      // a warp's share of 8 NT query rows
  float o[NT][HD / 16][4];
  float m[NT][2], neg[NT][2], l[NT][2];      // largest score (scaled), -m (NONE before the first one), sum of this thread's tokens
};
constexpr float NONE = 1e30f;      // in place of -m: any score passes it, and -inf with it is -inf
template <int HD, int NT> struct Queries {      // of a thread block's query rows, in shared memory
  uint4 b[NT][HD / 32][32];          // a lane's operands of a group's two products
  float4 start[NT][HD / 32][4];      // -8 2^-24 sum over a group of the query: of columns 2 j, 2 j + 1, twice (an accumulator's four)
  float back[NT][8];                 // score of a column = back * product
};

// Weights are 2^UP times what they are, so that with the values' codes as subnormal numbers, c 2^-133 (of odd elements 16 times that), O is 2^-45 times what it is
constexpr float UP = 88.f;
// With codes as they are: weights times this, and O is 2^-45 or 2^48 times what it is (in two factors: one would be subnormal)
struct Size { float a, b; };
__device__ __forceinline__ Size size_for(bool large) { return large ? Size{3.23117426778526e-27f, 2.8421709430404007e-14f} : Size{9.094947017729282e-13f, 1.f}; }      // 2^-88 2^-45, 2^-40
constexpr int SHARE = -5;      // shares' O is 2^SHARE times an average

// NB blocks of 16 tokens, one behind the other.  first: their first token; seen[n][c]: tokens that column c sees, asked only where MASKED.  WIDE: codes as they are
template <int HD, int NT, int NB, bool MASKED, bool WIDE>
__device__ __forceinline__ void attend(Rows<HD, NT>& r, const Queries<HD, NT>& q, const float (&c)[NT][2], const uint8_t* blk, int first,
                                       const int (&seen)[NT][2], Size size, int i, int j) {
  using L = Block<HD>;
  constexpr int NG = L::NG;
  // Row x of the products is token x ^ (x / 2 & 1): the tokens whose values a lane reads are then of both parities in each load, half the conflicts
  const int ta = i ^ (i >> 1 & 1), v0 = 2 * j + (j & 1), v1 = 2 * j + 1 - (j & 1);
  float s[NB][NT][4];
  Words<NG> ka[NB], kb[NB];
  float ska[NB][NG], skb[NB][NG];
#pragma unroll
  for (int b = 0; b < NB; b++) {
    const uint8_t* at = blk + b * L::BYTES;
    ka[b] = load_words<NG>(at + ta * L::ROW + 4 * j * NG), kb[b] = load_words<NG>(at + (ta + 8) * L::ROW + 4 * j * NG);
    load_scales<NG>(at + L::KS + 2 * ta * NG, ska[b]);
    load_scales<NG>(at + L::KS + 2 * (ta + 8) * NG, skb[b]);
  }
#pragma unroll
  for (int g = 0; g < NG; g++)
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const uint4 qb = q.b[n][g][i * 4 + j];
      const float4 st = q.start[n][g][j];
#pragma unroll
      for (int b = 0; b < NB; b++) {
        const uint32_t xa = ka[b].w[g], xb = kb[b].w[g], ya = xa >> 8, yb = xb >> 8;
        float d[4];
        mma_keys(d, low_codes(xa), low_codes(xb), high_codes(xa), high_codes(xb), qb.x, qb.y, st.x, st.y, st.z, st.w);
        mma_keys(d, low_codes(ya), low_codes(yb), high_codes(ya), high_codes(yb), qb.z, qb.w, d[0], d[1], d[2], d[3]);
#pragma unroll
        for (int k = 0; k < 4; k++) s[b][n][k] = g ? fmaf(k < 2 ? ska[b][g] : skb[b][g], d[k], s[b][n][k]) : (k < 2 ? ska[b][g] : skb[b][g]) * d[k];
      }
    }
  const int t0 = first + ta;      // token of block 0's elements 0 and 1; 2 and 3: 8 on
  if constexpr (MASKED) {
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (t0 + 16 * b + k / 2 * 8 >= seen[n][k & 1]) s[b][n][k] = -INFINITY;
  }
  auto power = [&](int b, int n, int k) {      // (a masked token's is -inf where a tiny scale's c has become 0 too)
    const float x = fmaf(s[b][n][k], c[n][k & 1], r.neg[n][k & 1]);
    return MASKED && s[b][n][k] == -INFINITY ? -INFINITY : x;
  };
  float y[NB][NT][4], top = -INFINITY;
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int k = 0; k < 4; k++) y[b][n][k] = power(b, n, k), top = fmaxf(top, y[b][n][k]);
  if (__any_sync(0xffffffffu, top > UP + 8.f)) {
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float x = -INFINITY;
#pragma unroll
        for (int b = 0; b < NB; b++) x = fmaxf(x, fmaxf(s[b][n][h], s[b][n][h + 2]) * c[n][h]);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
        x = fmaxf(x, r.m[n][h]);
        if (x > -INFINITY) {
          const float f = ex2(r.m[n][h] - x);      // (from -inf: 0)
          r.m[n][h] = x;
          r.neg[n][h] = UP - x;
          r.l[n][h] *= f;
#pragma unroll
          for (int d = 0; d < HD / 16; d++) r.o[n][d][h] *= f, r.o[n][d][h + 2] *= f;
        }
#pragma unroll
        for (int b = 0; b < NB; b++) y[b][n][h] = power(b, n, h), y[b][n][h + 2] = power(b, n, h + 2);
      }
  }
#pragma unroll
  for (int b = 0; b < NB; b++)
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int k = 0; k < 4; k++) {
        y[b][n][k] = ex2(y[b][n][k]);
        r.l[n][k & 1] += y[b][n][k];
      }
#pragma unroll
  for (int b = 0; b < NB; b++) {
    const uint8_t* at = blk + b * L::BYTES;
    float sa[NG], sb[NG];
    load_scales<NG>(at + L::VS + 2 * ta * NG, sa);
    load_scales<NG>(at + L::VS + 2 * (ta + 8) * NG, sb);
    uint32_t w0[NG], w1[NG], w2[NG], w3[NG];
    load_halves<NG>(at + L::V + v0 * L::ROW + 2 * i * NG, w0);
    load_halves<NG>(at + L::V + v1 * L::ROW + 2 * i * NG, w1);
    load_halves<NG>(at + L::V + (v0 + 8) * L::ROW + 2 * i * NG, w2);
    load_halves<NG>(at + L::V + (v1 + 8) * L::ROW + 2 * i * NG, w3);
#pragma unroll
    for (int g = 0; g < NG; g++) {
      const uint32_t x0 = __byte_perm(w0[g], w1[g], 0x5410), x1 = __byte_perm(w2[g], w3[g], 0x5410);
      uint32_t a[8];
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const uint32_t u = x0 >> 4 * e, v = x1 >> 4 * e;
        if constexpr (WIDE)
          a[2 * e] = value_codes(u), a[2 * e + 1] = sixteen_times(value_codes(u >> 4)), a[2 * e + 2] = value_codes(v), a[2 * e + 3] = sixteen_times(value_codes(v >> 4));
        else
          a[2 * e] = less(low_codes(u), 0x00080008u), a[2 * e + 1] = less(high_codes(u), 0x00800080u), a[2 * e + 2] = less(low_codes(v), 0x00080008u), a[2 * e + 3] = less(high_codes(v), 0x00800080u);
      }
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float p[4];
#pragma unroll
        for (int k = 0; k < 4; k++) p[k] = (WIDE ? y[b][n][k] * size.a * size.b : y[b][n][k]) * (k < 2 ? sa[g] : sb[g]);
        if constexpr (MASKED) {      // (a scale that is not seen may be anything)
#pragma unroll
          for (int k = 0; k < 4; k++)
            if (t0 + 16 * b + k / 2 * 8 >= seen[n][k & 1]) p[k] = 0.f;
        }
        const uint32_t b0 = transposed(pack_bf16(p[0], p[1])), b1 = transposed(pack_bf16(p[2], p[3]));
        mma_values(r.o[n][2 * g], a[0], a[1], a[2], a[3], b0, b1);
        mma_values(r.o[n][2 * g + 1], a[4], a[5], a[6], a[7], b0, b1);
      }
    }
  }
}

template <int HD, int NT> constexpr int merge_floats() { return 8 * NT * (HD + 2); }
template <int HD, int NT> constexpr int attn_ring() {      // bytes of the rings, and of the warps' shares that take their place
  const int ring = WARPS * Ring<HD>::N * Ring<HD>::BYTES, merge = WARPS * merge_floats<HD, NT>() * 4;
  return ring > merge ? ring : merge;
}
template <int HD, int NT> int attn_smem(int B) { return attn_ring<HD, NT>() + (int)sizeof(Queries<HD, NT>) + (B + 1) * 4; }

template <int HD, int NT>
__global__ void __launch_bounds__(WARPS * 32, PER_SM) kv4_attn_k(const AttnArgs A) {
  using L = Block<HD>;
  constexpr int NG = L::NG, NST = Ring<HD>::N, R = 8 * NT, PART = merge_floats<HD, NT>();
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[WARPS][NST];
  __shared__ int scan[WARPS], last;
  Queries<HD, NT>& q = *reinterpret_cast<Queries<HD, NT>*>(smem + attn_ring<HD, NT>());
  int* start = reinterpret_cast<int*>(smem + attn_ring<HD, NT>() + sizeof(q));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, i = lane >> 2, j = lane & 3;
  if (lane == 0) {
    for (int k = 0; k < NST; k++) tc::mbar_init(&bars[warp][k], 1);
    tc::mbar_fence_init();
  }
  mlb_pdl_sync();
  // first units of work of the sequences, per key / value head: its blocks and PAD, what it takes to begin and end one; an empty one has a unit, for its zeros
  const int longest = A.width << A.page_log;
  int done = 0;
  for (int b = 0; b < A.B; b += WARPS * 32) {
    int n = 0;
    if (b + tid < A.B) {
      n = A.lens[b + tid];
      if (n > longest && blockIdx.x == 0) mlb_set_error(MLB_ERR_BOUNDS, 0xC4);
      n = n <= 0 ? 1 : (min(n, longest) + TOK - 1) / TOK + PAD;
    }
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) scan[warp] = x;
    __syncthreads();
    int before = done;
    for (int w = 0; w < WARPS; w++) {
      if (w < warp) before += scan[w];
      done += scan[w];
    }
    if (b + tid < A.B) start[b + tid] = before + x - n;
    __syncthreads();
  }
  if (tid == 0) start[A.B] = done;
  __syncthreads();
  const unsigned total = (unsigned)done * A.Hkv, per = max((unsigned)WARPS, (total + gridDim.x - 1) / gridDim.x);      // (the host sees to it that total fits)
  unsigned s = per * blockIdx.x;
  const unsigned e = min(total, s + per);
  const int rows = A.G * A.Tq, row0 = blockIdx.y * R;
  uint8_t* ring = smem + warp * NST * Ring<HD>::BYTES;
  float* mrg = reinterpret_cast<float*>(smem);
  const int bpl = A.page_log - 4;      // log2 of the blocks of a page
  const unsigned page_bytes = (unsigned)A.Hkv * L::BYTES << bpl;      // of all heads (below 2^32: a page is at most 128 tokens)
  uint32_t parity = 0;                 // of the next phase of each place of this warp's ring
  bool dead = false;
  int b = 0;
  if (s < e) {      // the sequence of the first block
    int hi = A.B;
    while (hi - b > 1) {
      const int mid = (b + hi) >> 1;
      if ((unsigned)start[mid] * A.Hkv <= s) b = mid;
      else hi = mid;
    }
  }
  while (s < e) {
    while ((unsigned)start[b + 1] * A.Hkv <= s) b++;
    const unsigned nb = start[b + 1] - start[b], kv = (s - (unsigned)start[b] * A.Hkv) / nb;
    const unsigned item0 = (unsigned)start[b] * A.Hkv + kv * nb, item1 = item0 + nb;
    const int len = max(0, min(A.lens[b], longest)), blocks = (len + TOK - 1) / TOK;
    const int u0 = (int)(s - item0), u1 = min((int)(min(e, item1) - item0), blocks);
    auto token = [&](int r) { return (int)(((float)r + 0.5f) * A.inv_g); };      // r / G (exact: r < 2^20)
    auto finish = [&](int r, int d, float m, float l, const float4& o) {         // elements 4 d ... of row r, whole
      const int tok = token(row0 + r), head = (int)kv * A.G + row0 + r - tok * A.G;
      const float inv = l > 0.f ? (float)(1 << -SHARE) / l : (l == 0.f ? 0.f : l);      // (nothing seen: zeros; NaN stays)
      bf16* out = A.out + ((long)b * A.Tq + tok) * A.G * A.Hkv * HD + (long)head * HD + 4 * d;
      *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
      if (d == 0 && A.lse != nullptr)
        A.lse[((long)b * A.G * A.Hkv + head) * A.Tq + tok] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147180559945f;
    };
    const int live = min(R, rows - row0);
    if (u0 >= u1) {
      if (blocks == 0)
        for (int x = tid; x < live * (HD / 4); x += WARPS * 32) finish(x / (HD / 4), x % (HD / 4), 0.f, 0.f, make_float4(0, 0, 0, 0));
      s = min(e, item1);
      continue;
    }

    // ---- this warp's blocks [w0, w1)
    const int w0 = u0 + (u1 - u0) * warp / WARPS, w1 = u0 + (u1 - u0) * (warp + 1) / WARPS;
    Rows<HD, NT> acc;
    auto clear = [&] {
#pragma unroll
      for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int d = 0; d < HD / 16; d++)
#pragma unroll
          for (int k = 0; k < 4; k++) acc.o[n][d][k] = 0.f;
#pragma unroll
        for (int h = 0; h < 2; h++) acc.m[n][h] = -INFINITY, acc.neg[n][h] = NONE, acc.l[n][h] = 0.f;
      }
    };
    clear();
    const bool some = w0 < w1;
    const int* trow = A.table + (long)b * A.width;
    int have = 0, ids = -1;      // page numbers [have, have + 32) of the table, one a lane
    uint32_t there = 0;          // blocks in the ring whose page is one of the pool, STEP bits a place
    const uint8_t* base = A.pages + (size_t)(kv << bpl) * L::BYTES;
    auto names = [&](int p) {
      have = p;
      ids = p + lane < A.width ? trow[p + lane] : -1;
    };
    auto fetch = [&](int u, int k) {      // blocks u ... u + STEP - 1 into place k, a lane each
      const int mine = u + lane;
      if (((min(u + STEP, w1) - 1) >> bpl) >= have + 32) names(u >> bpl);
      const int id = __shfl_sync(0xffffffffu, ids, (mine >> bpl) - have);
      const bool wanted = lane < STEP && mine < w1, ok = wanted && (unsigned)id < (unsigned)A.n_pages;
      const uint32_t oks = __ballot_sync(0xffffffffu, ok);
      there = (there & ~(((1u << STEP) - 1) << k * STEP)) | oks << k * STEP;
      if (lane == 0) tc::mbar_expect_tx(&bars[warp][k], __popc(oks) * L::BYTES);
      __syncwarp();
      if (ok)
        tc::bulk_load(ring + k * Ring<HD>::BYTES + lane * L::BYTES, base + (size_t)(unsigned)id * page_bytes + (mine & ((1 << bpl) - 1)) * L::BYTES, L::BYTES,
                      &bars[warp][k]);
      else if (wanted)
        mlb_set_error(MLB_ERR_BOUNDS, 0xC1);
    };
    auto begin = [&] {
      names(w0 >> bpl);
#pragma unroll
      for (int k = 0; k < NST; k++)
        if (w0 + k * STEP < w1) fetch(w0 + k * STEP, k);
    };
    if (some && !dead) begin();
    // ---- the queries, while the first blocks are on their way: a group and tile of 8 rows a warp
#pragma unroll 1
    for (int x = warp; x < NT * NG; x += WARPS) {
      const int n = x / NG, own = x % NG, r = row0 + 8 * n + i, tok = token(r);
      const bf16* src = A.q + ((long)b * A.Tq + tok) * A.q_stride + ((int)kv * A.G + r - tok * A.G) * HD + 8 * j;
      uint32_t top = 0;
      uint4 w = {0, 0, 0, 0};
#pragma unroll
      for (int g = 0; g < NG; g++) {
        uint4 v = {0, 0, 0, 0};
        if (r < rows) v = *reinterpret_cast<const uint4*>(src + 32 * g);
        if (g == own) w = v;
        const uint32_t u[4] = {v.x & A.q_keep, v.y & A.q_keep, v.z & A.q_keep, v.w & A.q_keep};
#pragma unroll
        for (int k = 0; k < 4; k++) top = max(top, max(u[k] << 16 & 0x7F800000u, u[k] & 0x7F800000u));
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the row's largest element comes to 2^13 ... 2^14: exact for all elements above 2^-23 of it.  A row of zeros, or below 2^-100, as if its exponent were that
      const int ex = min(max((int)(top >> 23), 27), 243);
      const float f = __uint_as_float((uint32_t)(267 - ex) << 23);
      w.x = (w.x & A.q_keep) ^ A.q_flip, w.y = (w.y & A.q_keep) ^ A.q_flip, w.z = (w.z & A.q_keep) ^ A.q_flip, w.w = (w.w & A.q_keep) ^ A.q_flip;
      float v[8], y = 0.f;
      unpack8(w, v);
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] *= f, y += v[k];
      q.b[n][own][lane] = {pack_half(v[0], v[4]), pack_half(v[1] * 0.0625f, v[5] * 0.0625f), pack_half(v[2], v[6]), pack_half(v[3] * 0.0625f, v[7] * 0.0625f)};
      y += __shfl_xor_sync(0xffffffffu, y, 1);
      y += __shfl_xor_sync(0xffffffffu, y, 2);
      if (j == 0) {
        float* st = reinterpret_cast<float*>(&q.start[n][own][i / 2]) + i % 2;
        st[0] = st[2] = y * -4.76837158203125e-7f;      // -8 2^-24
        q.back[n][i] = A.scale_log2 * __uint_as_float((uint32_t)(ex + 11) << 23);
      }
    }
    float c[NT][2];
    int seen[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int col = row0 + 8 * n + 2 * j + h;
        seen[n][h] = col < rows ? len - A.Tq + token(col) + 1 : len;
      }
    const int all = len - A.Tq + token(row0) + 1;      // tokens that every column sees: the first row of the tile sees the fewest
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; n++) c[n][0] = q.back[n][2 * j], c[n][1] = q.back[n][2 * j + 1];
    auto walk = [&](auto wide, Size size) {
      constexpr bool WIDE = decltype(wide)::value;
      int k = 0;
#pragma unroll 1
      for (int u = w0; u < w1; u += STEP) {
        if (!__all_sync(0xffffffffu, tc::mbar_wait(&bars[warp][k], parity >> k & 1, 0xD1))) {
          dead = true;      // no more is fetched; what is on its way is waited for, the late one once more
          for (int x = 0; x < NST && u + x * STEP < w1; x++) tc::mbar_wait(&bars[warp][(k + x) % NST], parity >> (k + x) % NST & 1, 0xD2);
          __syncwarp();
          break;
        }
        parity ^= 1u << k;
        const uint32_t oks = there >> k * STEP & ((1u << STEP) - 1);
        const uint8_t* blk = ring + k * Ring<HD>::BYTES;
#pragma unroll 1
        for (int x = 0; x < STEP; x += 2) {
          if (!WIDE && (oks >> x & 3) == 3 && (u + x + 2) * TOK <= all) {
            attend<HD, NT, 2, false, false>(acc, q, c, blk + x * L::BYTES, (u + x) * TOK, seen, size, i, j);
          } else {
#pragma unroll 1
            for (int y = x; y < x + 2; y++)
              if (oks >> y & 1) attend<HD, NT, 1, true, WIDE>(acc, q, c, blk + y * L::BYTES, (u + y) * TOK, seen, size, i, j);
          }
        }
        __syncwarp();
        if (u + NST * STEP < w1) fetch(u + NST * STEP, k);
        k = k + 1 == NST ? 0 : k + 1;
      }
    };
    bool small = false;
    if (some && !dead) {
      walk(std::false_type(), Size{});
      // A scale of 2^31 or more may have made a weight infinite, and then it made all rows of the group's O infinite or NaN.  What is tiny or 0 may be so because it was lost.
      // First a look at one element in four, then at all, whose numbers without their signs lie in one range if all is well (together they are below it only if each is)
      constexpr uint32_t LOW = 32u << 24, HIGH = 255u << 24;      // 2^-95 (O of 2^-50), infinity
      auto outside = [&](auto every) {
        uint32_t far = 0;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            uint32_t f = 0;
#pragma unroll
            for (int g = 0; g < NG; g++) {
              uint32_t x = __float_as_uint(acc.o[n][2 * g][h]);
              if constexpr (decltype(every)::value) x |= __float_as_uint(acc.o[n][2 * g][h + 2]) | __float_as_uint(acc.o[n][2 * g + 1][h]) | __float_as_uint(acc.o[n][2 * g + 1][h + 2]);
              f = max(f, 2u * x - LOW);
            }
            if (acc.m[n][h] > -INFINITY) far = max(far, f);      // (a row that sees nothing here has zeros)
          }
        return __any_sync(0xffffffffu, far >= HIGH - LOW) != 0;
      };
      if (outside(std::false_type()) && outside(std::true_type())) {
        auto endless = [&] {
          float x = 0.f;
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int g = 0; g < NG; g++) x = fmaf(acc.o[n][2 * g][0], 0.f, fmaf(acc.o[n][2 * g][1], 0.f, x));
          return __any_sync(0xffffffffu, x != 0.f) != 0;
        };
        uint32_t least = ~0u;      // of the groups' largest elements
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int g = 0; g < NG; g++) {
              uint32_t top = 0;
#pragma unroll
              for (int e = 0; e < 4; e++) top = max(top, 2u * __float_as_uint(acc.o[n][2 * g + e / 2][h + e % 2 * 2]));
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
              if (acc.m[n][h] > -INFINITY) least = min(least, top);
            }
        bool large = endless();
        small = !large && __any_sync(0xffffffffu, least < LOW);
        while (!dead && (large || small)) {
          clear();
          tc::fence_async_smem();
          __syncwarp();
          begin();
          walk(std::true_type(), size_for(large));
          if (large || !endless()) break;
          large = true, small = false;
        }
      }
    }
    // ---- the warps' shares put together (in the rings' memory, which nothing is on its way to)
    __syncthreads();
    float* mine = mrg + warp * PART;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float l = acc.l[n][h];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        const int col = 8 * n + 2 * j + h;
        // l is 2^UP times the sum of weights (88 + 127 is 1's exponent): the power of two that brings it to 1 ... 2 goes to m, and with those of O and of the share into the factor
        const int ex = min(max((int)(__float_as_uint(l) >> 23), 200), 253);
        const float even = __uint_as_float((uint32_t)(127 + 215 + SHARE + (small ? -48 : 45) - ex) << 23), odd = even * 0.0625f;
        l *= __uint_as_float((uint32_t)(254 - ex) << 23);
        if (i == 0) mine[col] = acc.m[n][h] + (float)(ex - 215), mine[R + col] = l;
#pragma unroll
        for (int g = 0; g < NG; g++) {
          if (col < live)
            *reinterpret_cast<float4*>(mine + 2 * R + col * HD + 32 * g + 4 * i) =
                make_float4(acc.o[n][2 * g][h] * even, acc.o[n][2 * g][h + 2] * odd, acc.o[n][2 * g + 1][h] * even, acc.o[n][2 * g + 1][h + 2] * odd);
        }
      }
    __syncthreads();
    const unsigned c0 = item0 / per, c1 = (item0 + blocks - 1) / per;      // the thread blocks that share this head
    const int item = (int)((blockIdx.y * (unsigned)A.B + b) * A.Hkv + kv), n_shares = (int)(c1 - c0 + 1);
    float* part = A.part + (long)blockIdx.y * gridDim.x * 2 * PART;
    float* my = part + (blockIdx.x * 2 + (s == per * blockIdx.x ? 0 : 1)) * (long)PART;
    for (int x = tid; x < live * (HD / 4); x += WARPS * 32) {
      const int r = x / (HD / 4), d = x % (HD / 4);
      float m = -INFINITY, l = 0.f;
      for (int w = 0; w < WARPS; w++) m = fmaxf(m, mrg[w * PART + r]);
      float4 o = {0, 0, 0, 0};
      for (int w = 0; w < WARPS; w++) {
        const float mw = mrg[w * PART + r], f = mw == m ? (m == -INFINITY ? 0.f : 1.f) : ex2(mw - m);
        const float4 v = *reinterpret_cast<const float4*>(mrg + w * PART + 2 * R + r * HD + 4 * d);
        l = fmaf(f, mrg[w * PART + R + r], l);
        o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
      }
      if (n_shares > 1) {
        if (d == 0) my[r] = m, my[R + r] = l;
        *reinterpret_cast<float4*>(my + 2 * R + r * HD + 4 * d) = o;
      } else {
        finish(r, d, m, l, o);
      }
    }
    if (n_shares > 1) {
      __syncthreads();
      if (tid == 0) last = mlb_count_block(A.count + item) == n_shares - 1;
      __syncthreads();
      if (last) {
        if (tid == 0) A.count[item] = 0;      // for the next call
        // elements to the threads; few elements: the shares too, `ways` threads an element
        const int elems = live * (HD / 4), ways = elems >= WARPS * 32 ? 1 : WARPS * 32 / elems;
        for (int x = tid; x < elems * ways; x += NT * WARPS * 32) {      // (of two tiles of rows two elements a thread, their loads on their way together)
          constexpr int BATCH = 8;      // shares on their way at a time
          const int way = ways > 1 ? x / elems : 0;
          int row[NT], word[NT];
          bool is[NT];
          float m[NT], l[NT];
          float4 o[NT];
#pragma unroll
          for (int n = 0; n < NT; n++) {
            const int y = x - way * elems + n * WARPS * 32;
            is[n] = n == 0 || (ways == 1 && y < elems);
            row[n] = y / (HD / 4), word[n] = y % (HD / 4);
            m[n] = -INFINITY, l[n] = 0.f, o[n] = make_float4(0, 0, 0, 0);
          }
          for (int c = way; c < n_shares; c += ways * BATCH) {
            float ms[NT][BATCH], ls[NT][BATCH];
            float4 os[NT][BATCH];
#pragma unroll
            for (int k = 0; k < BATCH; k++) {
              const int z = c + k * ways;
              const float* p = part + ((c0 + z) * 2 + (z > 0 || item0 == c0 * per ? 0 : 1)) * (long)PART;
#pragma unroll
              for (int n = 0; n < NT; n++) {
                ms[n][k] = -INFINITY, ls[n][k] = 0.f, os[n][k] = make_float4(0, 0, 0, 0);
                if (z < n_shares && is[n])
                  ms[n][k] = __ldcg(p + row[n]), ls[n][k] = __ldcg(p + R + row[n]), os[n][k] = __ldcg(reinterpret_cast<const float4*>(p + 2 * R + row[n] * HD + 4 * word[n]));
              }
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
              float top = m[n];
#pragma unroll
              for (int k = 0; k < BATCH; k++) top = fmaxf(top, ms[n][k]);
              const float g = top == -INFINITY ? 1.f : ex2(m[n] - top);
              l[n] *= g, o[n].x *= g, o[n].y *= g, o[n].z *= g, o[n].w *= g, m[n] = top;
#pragma unroll
              for (int k = 0; k < BATCH; k++) {
                const float f = top == -INFINITY ? 0.f : ex2(ms[n][k] - top);
                const float4 v = os[n][k];
                l[n] = fmaf(f, ls[n][k], l[n]);
                o[n].x = fmaf(f, v.x, o[n].x), o[n].y = fmaf(f, v.y, o[n].y), o[n].z = fmaf(f, v.z, o[n].z), o[n].w = fmaf(f, v.w, o[n].w);
              }
            }
          }
          if (ways == 1) {
#pragma unroll
            for (int n = 0; n < NT; n++)
              if (is[n]) finish(row[n], word[n], m[n], l[n], o[n]);
          } else {      // (the warps' shares in shared memory have been read)
            float* t = mrg + x * 6;
            t[0] = m[0], t[1] = l[0], t[2] = o[0].x, t[3] = o[0].y, t[4] = o[0].z, t[5] = o[0].w;
          }
        }
        if (ways > 1) {
          __syncthreads();
          if (tid < elems) {
            float m = -INFINITY, l = 0.f;
            float4 o = {0, 0, 0, 0};
            for (int w = 0; w < ways; w++) m = fmaxf(m, mrg[(w * elems + tid) * 6]);
            for (int w = 0; w < ways; w++) {
              const float* t = mrg + (w * elems + tid) * 6;
              const float f = m == -INFINITY ? 0.f : ex2(t[0] - m);
              l = fmaf(f, t[1], l), o.x = fmaf(f, t[2], o.x), o.y = fmaf(f, t[3], o.y), o.z = fmaf(f, t[4], o.z), o.w = fmaf(f, t[5], o.w);
            }
            finish(tid / (HD / 4), tid % (HD / 4), m, l, o);
          }
        }
      }
    }
    tc::fence_async_smem();      // (bulk copies will write where the shares were)
    __syncthreads();
    s = min(e, item1);
  }
}

template <int HD, int NT>
cudaError_t launch_attn(const AttnArgs& a, int grid, int tiles, cudaStream_t st) {
  static std::atomic<unsigned long long> allowed{0};
  const cudaError_t e = mlb_allow_smem(kv4_attn_k<HD, NT>, attn_smem<HD, NT>(MAX_B), allowed);
  if (e != cudaSuccess) return e;
  return mlb_launch(kv4_attn_k<HD, NT>, dim3(grid, tiles), dim3(WARPS * 32), attn_smem<HD, NT>(a.B), st, a);
}
bool known_head(int hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128; }
int page_shift(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : page == 128 ? 7 : -1; }
// query rows a thread block takes at a time: 8 where that is all of them, else 16
int row_tiles(long rows, int& nt) {
  nt = rows <= 8 ? 1 : 2;
  return (int)((rows + 8 * nt - 1) / (8 * nt));
}
// Shared memory of a thread block: for the grid, which has to be resident at once, all row tiles of it, to be worth its division of the work (a grid of that
// size for each row tile: 64 tokens behind 5000, 8 heads of 64, 14.5 -> 32.7 us; 2 x 8 tokens behind 16000, 64 heads over 8 of 128, 49 -> 79)
int attn_smem_of(int hd, int nt, int B) {
#define MLB_SMEM(HD) return nt == 1 ? attn_smem<HD, 1>(B) : attn_smem<HD, 2>(B)
  switch (hd) {
    case 32: MLB_SMEM(32);
    case 64: MLB_SMEM(64);
    case 96: MLB_SMEM(96);
    default: MLB_SMEM(128);
  }
#undef MLB_SMEM
}
int attn_most(long B, int Hkv, int width, int page) {      // a thread block has a unit for each warp
  const long most = B * Hkv * (((long)width * page + TOK - 1) / TOK + PAD), all = (long)PER_SM * mlb_sm_count(), want = (most + WARPS - 1) / WARPS;
  return (int)(want < all ? (want > 0 ? want : 1) : all);
}
int attn_grid(long B, int Hkv, int width, int page, int hd, int nt, int tiles) {      // of each row tile
  const long all = 228L * 1024 / (attn_smem_of(hd, nt, (int)B) + 1024 + 128) * mlb_sm_count();      // (1 KB of a block's is the system's)
  const long fit = (all + tiles - 1) / tiles, want = attn_most(B, Hkv, width, page);
  return (int)(want < fit ? want : fit);
}
// Threads of a row (`per_row`) in blocks of up to 512, and rows twice as often as the machine holds 1024 threads an SM (append's registers: two waves; reading back: one).  Blocks
// go over the rows in equal steps, so that a wave of a few blocks more is what costs: 8192 rows of 12 + 24 heads of 64 written and read 23.6 us (25.3 once, 25.3
// three times, 25.8 with 4 rows a block), of 16 + 32 heads of 128 54.7 (63.7, 56.2, 59.3), 4096 rows of 32 + 16 heads of 128 27.0 (28.0, 28.0, 30.3)
struct Shape { dim3 grid; unsigned threads; };
Shape rows_shape(long per_row, long N) {
  if (per_row < 1 || per_row >= 1L << 30 || N < 1 || N >= (1L << 31) - 65536) return {dim3(), 0};
  const long blocks = (per_row + 511) / 512, threads = ((per_row + blocks - 1) / blocks + 31) / 32 * 32;
  const long fit = 2 * (1024 / threads) * mlb_sm_count() / blocks, rows = N < fit ? N : fit > 1 ? fit : 1;
  return {dim3((unsigned)blocks, (unsigned)rows), (unsigned)threads};
}
// Rows, tables and workspaces are read and written 16 bytes at a time (null: none)
template <typename... P> bool on_16_bytes(P... p) { return ((... | (uintptr_t)p) & 15) == 0; }
#define MLB_BY_HEAD(hd, F) \
  switch (hd) {            \
    case 32: F(32); break; \
    case 64: F(64); break; \
    case 96: F(96); break; \
    default: F(128);       \
  }

}  // namespace

// qkv[N] rows of (H + 2 Hkv) heads, `stride` elements apart: queries (and keys) rotated by cos / sin[pos] (null: not) go to q_out[N, H hd] (null: nowhere), keys and
// values to the slots of the pool; a negative slot is none.  Returns -7 for what the kernel does not take.
MLB_API int mlb_kv4_append(uint8_t* pages, void* q_out, const void* qkv, const int* slots, const int* pos, const float* cos, const float* sin, long n_pages,
                           int page, long N, long stride, int H, int Hkv, int hd, int T, cudaStream_t st) {
  if (!known_head(hd) || page_shift(page) < 0 || stride % 8 != 0 || H < 0 || Hkv < 1 || !on_16_bytes(pages, q_out, qkv, cos, sin)) return -7;
  const bool halves = hd % 64 == 0;
  const Shape z = rows_shape((long)(H + 2 * Hkv) * (hd / (halves ? 16 : 8)), N);
  if (z.threads == 0) return -7;
#define MLB_GO(KERNEL)                                                                                                                        \
  return (int)mlb_launch(KERNEL, z.grid, dim3(z.threads), 0, st, pages, (bf16*)q_out, (const bf16*)qkv, slots, pos, cos, sin, n_pages, page_shift(page), (int)N, stride, H, Hkv, T)
  switch (hd) {
    case 32: MLB_GO(kv4_append_k<32>);
    case 64: MLB_GO(kv4_append_halves_k<64>);
    case 96: MLB_GO(kv4_append_k<96>);
    default: MLB_GO(kv4_append_halves_k<128>);
  }
#undef MLB_GO
}

// k, v[N, Hkv, hd]: what the slots hold; zeros for a negative slot
MLB_API int mlb_kv4_read(void* k, void* v, const uint8_t* pages, const int* slots, long n_pages, int page, long N, int Hkv, int hd, cudaStream_t st) {
  if (!known_head(hd) || page_shift(page) < 0 || Hkv < 1 || !on_16_bytes(k, v, pages)) return -7;
  const Shape z = rows_shape((long)Hkv * (hd / 8), N);
  if (z.threads == 0) return -7;
  cudaError_t e = cudaSuccess;
#define MLB_GO(HD) e = mlb_launch(kv4_read_k<HD>, z.grid, dim3(z.threads), 0, st, (bf16*)k, (bf16*)v, pages, slots, n_pages, page_shift(page), (int)N, Hkv)
  MLB_BY_HEAD(hd, MLB_GO)
#undef MLB_GO
  return (int)e;
}

// fp32 words of workspace that attention wants - two shares of each thread block of its launches - and (negative) nothing for sizes that it does not take; counters:
// B Hkv row tiles, zero before the first call
MLB_API long mlb_kv4_attn_scratch(int B, int Tq, int H, int Hkv, int hd, int width, int page) {
  if (!known_head(hd) || page_shift(page) < 0 || Hkv < 1 || H < 1 || H % Hkv != 0 || Tq < 1) return -7;
  int nt;
  const int tiles = row_tiles((long)(H / Hkv) * Tq, nt);
  int grid = attn_grid(B < MAX_B ? B : MAX_B, Hkv, width, page, hd, nt, tiles);
  if (B > MAX_B && B % MAX_B != 0) {      // the last launch: fewer sequences, whose numbers leave room for more blocks
    const int last = attn_grid(B % MAX_B, Hkv, width, page, hd, nt, tiles);
    grid = last > grid ? last : grid;
  }
  return (long)grid * tiles * 2 * 8 * nt * (hd + 2);
}
// out[B Tq, H hd] = attention of q (rows `q_stride` elements apart) over table[B, width], lens[B] tokens each; lse[B, H, Tq] or null
MLB_API int mlb_kv4_attn(void* out, float* lse, const void* q, const uint8_t* pages, const int* table, const int* lens, float* part, int* count, long n_pages,
                         long q_stride, int B, int Tq, int H, int Hkv, int hd, int width, int page, float scale, cudaStream_t st) {
  const int shift = page_shift(page);
  if (!known_head(hd) || shift < 0 || Hkv < 1 || H < 1 || H % Hkv != 0 || Tq < 1 || q_stride % 8 != 0 || !on_16_bytes(out, q, pages, part)) return -7;
  int nt;
  const int tiles = row_tiles((long)(H / Hkv) * Tq, nt);
  if (tiles > 65535 || (long)n_pages > 0x7FFFFFFFL || (long)width * page >= 1L << 31 || (long)Hkv * page * hd * 9 / 8 >= 1L << 32 || ((long)width * page / TOK + PAD) * (B < MAX_B ? B : MAX_B) * Hkv >= 1L << 31) return -7;
  cudaError_t e = cudaSuccess;
  for (int b = 0; b < B && e == cudaSuccess; b += MAX_B) {
    const int n = B - b < MAX_B ? B - b : MAX_B;
    const AttnArgs a{(bf16*)out + (long)b * Tq * H * hd, lse ? lse + (long)b * H * Tq : nullptr, (const bf16*)q + (long)b * Tq * q_stride, pages,
                     table + (long)b * width, lens + b, part, count, q_stride, n_pages, n, Tq, H / Hkv, Hkv, width, shift, (scale == 0.f ? 1.f : fabsf(scale)) * 1.44269504088896f,
                     scale == 0.f ? 0u : ~0u, scale < 0.f ? 0x80008000u : 0u, 1.f / (H / Hkv)};
    const int grid = attn_grid(n, Hkv, width, page, hd, nt, tiles);
#define MLB_GO(HD) e = nt == 1 ? launch_attn<HD, 1>(a, grid, tiles, st) : launch_attn<HD, 2>(a, grid, tiles, st)
    MLB_BY_HEAD(hd, MLB_GO)
#undef MLB_GO
  }
  return (int)e;
}
