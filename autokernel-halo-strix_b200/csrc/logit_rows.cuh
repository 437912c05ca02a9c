// Device helpers shared by the operators over rows of logits (token log-probabilities,
// distillation): addressing of strided rows, 32-byte groups, running softmax statistics.
#pragma once

#include "ak_common.cuh"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace ak {

// Rows of logits: row r is (outer, inner) = (r / inner, r % inner) and starts at
// base + outer * s_outer + inner * s_inner elements, so a (B, T, V) view such as
// logits[:, :-1] needs no copy.  Elements of a row are adjacent.
struct RowAddr {
  int64_t inner, s_outer, s_inner;
  __host__ __device__ __forceinline__ int64_t off(int64_t r) const {
    if (r < inner) return r * s_inner;
    const uint32_t o = (uint32_t)r / (uint32_t)inner;  // fewer than 2^27 rows
    return (int64_t)o * s_outer + (int64_t)((uint32_t)r - o * (uint32_t)inner) * s_inner;
  }
};

// What a logit x means: y = softcap(x), log-probabilities of y / temperature.
// kl = log2(e) / temperature turns a difference of y into an exponent of 2.
// -inf stays -inf under softcap: a masked token has no probability there either.
// temperature >= kLowestTemperature: its reciprocal and products with raise_floor stay finite; so does
// the reciprocal of a softcap >= kLowestSoftcap.
struct Squash {
  float cap, inv_cap, inv_t, kl;
  float rkl;   // 1 / kl
  float kc;    // -2 log2(e) / cap
};

// What the kernels are instantiated for (CAP): no softcap, one, or one so wide that its far form has
// to keep small logits as well.
enum SoftcapForm : int { kNoCap = 0, kCap = 1, kWideCap = 2 };
inline int cap_form(const Squash& q) { return q.cap == 0.f ? kNoCap : q.cap <= 64.f ? kCap : kWideCap; }

constexpr float kLowestTemperature = 7.888609052210118e-31f, kLowestSoftcap = kLowestTemperature;  // 2^-100

inline Squash make_squash(float temperature, float softcap) {
  Squash q;
  q.cap = softcap > 0.f ? softcap : 0.f;
  q.inv_cap = softcap > 0.f ? 1.f / softcap : 0.f;
  q.kc = softcap > 0.f ? (float)(-2.0 * 1.4426950408889634 / (double)softcap) : 0.f;
  q.inv_t = 1.f / temperature;
  q.kl = (float)(1.4426950408889634 / (double)temperature);
  q.rkl = 1.f / q.kl;
  return q;
}

// A statement with CAP as the constant that q's softcap stands for.
#define AK_DISPATCH_CAP(q, CAP, ...)                                                  \
  do {                                                                                \
    switch (cap_form(q)) {                                                            \
      case kNoCap: { constexpr int CAP = kNoCap; __VA_ARGS__; } break;                \
      case kCap: { constexpr int CAP = kCap; __VA_ARGS__; } break;                    \
      default: { constexpr int CAP = kWideCap; __VA_ARGS__; } break;                  \
    }                                                                                 \
  } while (0)

// cap tanh(x / cap), by one of two forms.  u = 2^-24.
//
// |x| <= cap: x P(w), w = (x / cap)^2, where P is the polynomial of degree 6 with P(0) = 1 whose largest
// relative distance from tanh(z) / z on 0 < z <= 1 is smallest.  Its coefficients were rounded to fp32
// one after the other, the later ones fitted anew to those that were (linear programs over a grid of
// w): 0.93 u, as without the rounding.  w is off by 5 u, of which 0.22 reach tanh(z) / z; Horner's
// steps add 1.2 u and the product 1 u: within 5 u of its value, small logits under a large cap too.
//
// Beyond: (1 - E) / (1 + E) with E = e^(-2 |x| / cap) and x's sign, two special-unit operations.  E's
// argument is off by 2 u relative and the hardware's exponential by 4 u, which reaches tanh as
// 2 E / (1 + E)^2 (4 |x / cap| + 4) u <= 2.4 u; the difference, the sum and the quick division add
// 6 u of tanh itself: at most 9 u of cap.  1 - E cancels for small logits, which come here beside one
// beyond the cap (a mask of the type's lowest value).  Up to a cap of 64 that is 3e-5 at most.  Above
// it (kWideCap) logits below cap / 16 take x (1 - w / 3 + 2 w^2 / 15), whose next term is 0.05 u, so that
// each is within 40 u of its value as well.  Taken under every cap, that cost the softcap's cases 2 to
// 20 % (4096 x 50304 bf16, most logits beyond the cap: 175 + 227 us to 200 + 277).
//
// The second form holds everywhere, but its special-unit operations bound the kernels.  With the first
// where a warp's logits allow it, 4096 x 50304 bf16 under a softcap of 30 takes 121 us forward and 165
// backward (167 and 198 without it), distillation of 8192 rows 711 us (917); logits that mostly lie
// beyond the cap pay 5 to 24 % for the test.
__device__ constexpr float tanh_coef(int i) {  // of w^(i + 1)
  const float c[6] = {-0.333329886f, 0.133264288f, -0.0534994751f, 0.0203611124f, -0.00626045559f, 0.00105861423f};
  return c[i];
}

__device__ __forceinline__ float squash_near(float x, const Squash& q) {
  const float z = x * q.inv_cap, w = z * z;
  float p = tanh_coef(5);
#pragma unroll
  for (int i = 4; i >= 0; --i) p = fmaf(p, w, tanh_coef(i));
  return x * fmaf(p, w, 1.f);
}
__device__ __forceinline__ float2 squash_near(float2 x, const Squash& q) {
  const float2 z = __fmul2_rn(x, make_float2(q.inv_cap, q.inv_cap)), w = __fmul2_rn(z, z);
  float2 p = make_float2(tanh_coef(5), tanh_coef(5));
#pragma unroll
  for (int i = 4; i >= 0; --i) p = __ffma2_rn(p, w, make_float2(tanh_coef(i), tanh_coef(i)));
  return __fmul2_rn(x, __ffma2_rn(p, w, make_float2(1.f, 1.f)));
}

template <int CAP>
__device__ __forceinline__ float squash_far(float x, const Squash& q) {  // holds for every x
  const float e = ex2(fabsf(x) * q.kc);
  float y = copysignf(q.cap * __fdividef(1.f - e, 1.f + e), x);
  if constexpr (CAP == kWideCap) {
    const float z = x * q.inv_cap, w = z * z;
    if (w < 0.00390625f) y = x * fmaf(fmaf(w, 2.f / 15.f, -1.f / 3.f), w, 1.f);
  }
  return x == -INFINITY ? x : y;
}

template <int CAP>
__device__ __forceinline__ float squash(float x, const Squash& q) {  // one logit
  if constexpr (!CAP) return x;
  return fabsf(x) <= q.cap ? squash_near(x, q) : squash_far<kCap>(x, q);
}

// Derivative of squash at its output y.
template <int CAP>
__device__ __forceinline__ float squash_slope(float y, const Squash& q) {
  if constexpr (!CAP) return 1.f;
  const float t = y * q.inv_cap;
  return y == -INFINITY ? 0.f : 1.f - t * t;
}
__device__ __forceinline__ float2 squash_slope_near(float2 y, const Squash& q) {
  float2 t = __fmul2_rn(y, make_float2(q.inv_cap, q.inv_cap));
  t = make_float2(fmaxf(t.x, -1.f), fmaxf(t.y, -1.f));  // 0 at -inf; a NaN reaches the result by y
  return __ffma2_rn(make_float2(-t.x, -t.y), t, make_float2(1.f, 1.f));
}

// A row is cut into a head (elements before the first 32-byte boundary), groups of 16
// elements (32 bytes of a 16-bit type, 64 bytes of fp32) and a tail of fewer than 16.
constexpr int kGroup = 16;

struct RowCut {
  int head, groups, tail;
};

template <typename T>
__device__ __forceinline__ RowCut cut_row(const T* row, int V) {
  RowCut c;
  const int mis = (int)(reinterpret_cast<uintptr_t>(row) & 31u);
  c.head = min(V, mis ? (32 - mis) / (int)sizeof(T) : 0);
  c.groups = (V - c.head) / kGroup;
  c.tail = V - c.head - c.groups * kGroup;
  return c;
}

// 32 bytes with one load or store (addresses 32-byte aligned).
struct Words8 {
  uint32_t w[8];
};
__device__ __forceinline__ Words8 load32(const void* p) {
  Words8 r;
  asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]),
                 "=r"(r.w[7])
               : "l"(p));
  return r;
}
__device__ __forceinline__ void store32(void* p, const Words8& r) {
  asm volatile("st.global.v8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]),
               "r"(r.w[3]), "r"(r.w[4]), "r"(r.w[5]), "r"(r.w[6]), "r"(r.w[7]), "l"(p)
               : "memory");
}

// One group as it lies in memory, and as fp32 values.
template <typename T>
struct RawGroup {
  Words8 r[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ RawGroup<T> load_group(const T* p) {
  RawGroup<T> g;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) g.r[i] = load32(reinterpret_cast<const char*>(p) + 32 * i);
  return g;
}

__device__ __forceinline__ float2 unpack2(uint32_t w, const __nv_bfloat16*) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack2(uint32_t w, const __half*) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __nv_bfloat16*) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __half*) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T>
__device__ __forceinline__ void unpack_group(float (&x)[kGroup], const RawGroup<T>& g) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = __uint_as_float(g.r[i / 8].w[i % 8]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 v = unpack2(g.r[0].w[i], (const T*)nullptr);
      x[2 * i] = v.x;
      x[2 * i + 1] = v.y;
    }
  }
}

// Stores 16 values rounded to T: one or two 32-byte stores where the address allows, else
// element by element (the output's rows start at another phase than the input's).
template <typename T>
__device__ __forceinline__ void store_group(T* p, const float (&x)[kGroup], bool vec) {
  if (vec) {
    RawGroup<T> g;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 16; ++i) g.r[i / 8].w[i % 8] = __float_as_uint(x[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) g.r[0].w[i] = pack2(x[2 * i], x[2 * i + 1], (const T*)nullptr);
    }
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) store32(reinterpret_cast<char*>(p) + 32 * i, g.r[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = from_f<T>(x[i]);
  }
}

// ---------------------------------------------------------------------------
// Values as they lie in memory: words of two 16-bit elements, or of one fp32
// ---------------------------------------------------------------------------
template <typename T>
__host__ __device__ constexpr int elems_per_word() { return 4 / (int)sizeof(T); }

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b, const __nv_bfloat16*) {
  const __nv_bfloat162 r = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b, const __half*) {
  const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b, const float*) {
  return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
}
__device__ __forceinline__ uint32_t word_max_nan(uint32_t a, uint32_t b, const __nv_bfloat16*) {
  const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t word_max_nan(uint32_t a, uint32_t b, const __half*) {
  const __half2 r = __hmax2_nan(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t word_max_nan(uint32_t a, uint32_t b, const float*) {
  return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
}

// Largest value of NW words; NaN is passed over (all NaN: NaN).
template <typename T, int NW>
__device__ __forceinline__ float words_max(const uint32_t (&w)[NW]) {
  uint32_t m = w[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) m = word_max(m, w[i], (const T*)nullptr);
  if constexpr (sizeof(T) == 4) return __uint_as_float(m);
  else {
    const float2 v = unpack2(m, (const T*)nullptr);
    return fmaxf(v.x, v.y);
  }
}

// Pairs of values: pair i of NW words (16-bit: word i; fp32: words 2 i and 2 i + 1).
template <typename T, int NW>
__device__ __forceinline__ float2 word_pair(const uint32_t (&w)[NW], int i) {
  if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
  else return unpack2(w[i], (const T*)nullptr);
}

// Whether squash_near holds for all NW words, lm their largest value: none beyond the cap but -inf and
// NaN, which it passes on (its last coefficient is positive).  One answer for the lanes that are here
// together: the form that holds everywhere is cheaper than both in turn.
__device__ __forceinline__ uint32_t abs_but_inf(uint32_t w, const __nv_bfloat16*) {
  const uint32_t inf = 0xff80ff80u;
  return w & 0x7fff7fffu & ~__heq2_mask(*reinterpret_cast<const __nv_bfloat162*>(&w),
                                        *reinterpret_cast<const __nv_bfloat162*>(&inf));
}
__device__ __forceinline__ uint32_t abs_but_inf(uint32_t w, const __half*) {
  const uint32_t inf = 0xfc00fc00u;
  return w & 0x7fff7fffu & ~__heq2_mask(*reinterpret_cast<const __half2*>(&w), *reinterpret_cast<const __half2*>(&inf));
}
template <typename T, int NW>
__device__ __forceinline__ bool all_near(const uint32_t (&w)[NW], float lm, const Squash& q) {
  if constexpr (sizeof(T) == 4) {  // the bits without the sign, turned so that infinity comes to 0 and NaN next
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) m = max(m, 2u * w[i] + 0x01000000u);
    return __all_sync(__activemask(), m <= 2u * __float_as_uint(q.cap) + 0x01000000u && lm <= q.cap);
  } else {
    uint32_t m = abs_but_inf(w[0], (const T*)nullptr);
#pragma unroll
    for (int i = 1; i < NW; ++i) m = word_max(m, abs_but_inf(w[i], (const T*)nullptr), (const T*)nullptr);
    const float2 v = unpack2(m, (const T*)nullptr);
    return __all_sync(__activemask(), fmaxf(v.x, v.y) <= q.cap && lm <= q.cap);
  }
}

// The same value twice, as an operand of paired arithmetic in plain registers: where the compiler
// knows that a value is the same in the whole warp it keeps it in uniform registers, and each paired
// instruction then costs moves.
__device__ __forceinline__ float2 both(float v) {
  float2 r = make_float2(v, v);
  asm volatile("" : "+f"(r.x), "+f"(r.y));
  return r;
}

// ---------------------------------------------------------------------------
// Running softmax statistics of a set of logits
// ---------------------------------------------------------------------------
// Exponents are taken against a reference point given in powers of two: e = 2^d with
//   d = (y - sh) * kl - k,    k an integer, sh = 0
// so that a logit costs one fused multiply-add, which rounds once, whatever y is; moving the
// reference multiplies by an exact power of two.  (kl itself is rounded: all results are those of a
// temperature off by half a unit in the last place.)  Where |y * kl| reaches 2^22 -- rows that hold
// nothing but a mask of the type's lowest value, whose product with kl would overflow -- y is
// subtracted first (sh = y, k = 0).
struct Ref {
  float sh, k;
};

__device__ __forceinline__ float exponent(float y, const Ref& r, const Squash& q) {
  return fmaf(y - r.sh, q.kl, -r.k);
}

// 2^d for an integer d <= 0 (0 below the normal numbers).
__device__ __forceinline__ float pow2i(float d) {
  return d < -126.f ? 0.f : __int_as_float((127 + (int)d) << 23);
}

// How far reference a lies above b, in powers of two (at least -1e30), and the factor 2 to that.
__device__ __forceinline__ float ref_diff(const Ref& a, const Ref& b, const Squash& q) {
  if (a.sh == b.sh) return a.k - b.k;
  return fmaxf((a.sh - b.sh) * q.kl + (a.k - b.k), -1e30f);
}
__device__ __forceinline__ float ref_scale(const Ref& a, const Ref& b, const Squash& q) {
  const float d = ref_diff(a, b, q);
  return a.sh == b.sh && d <= 0.f ? pow2i(d) : ex2(d);
}

// Where a product of e = 2^d with d is formed, -inf has to be raised to a finite logit whose e is
// still 0: to `raise_floor`, which the type represents, and whose d is finite at the lowest
// temperature (-2^20 log2(e) 2^100).  Holds for a reference far enough above it, so for rows whose
// largest logit is above -10^6 up to a temperature of some thousands; elsewhere the terms are cut off
// one by one.
template <typename T>
__device__ __forceinline__ float raise_floor() {
  return std::is_same<T, __half>::value ? -65504.f : -1048576.f;
}
template <typename T>
__device__ __forceinline__ bool can_raise(const Ref& r, const Squash& q) {
  return r.sh == 0.f && r.k - raise_floor<T>() * q.kl > 200.f;
}
template <typename T>
__device__ __forceinline__ uint32_t floor_word(float floor = raise_floor<T>()) {
  if constexpr (sizeof(T) == 4) return __float_as_uint(floor);
  else return pack2(floor, floor, (const T*)nullptr);
}

// A gradient multiplies d by what comes from upstream, which may be large: there -inf is raised no
// lower than it has to be, about 300 powers of 2 below the reference.  (1/64 of the reference more,
// so that rounding the logit to T, 2^-9 of it at most, leaves its term 0.)  `floor` receives the
// logit and the answer is whether its term is 0.
template <typename T>
__device__ __forceinline__ bool raise_to(float& floor, const Ref& r, const Squash& q) {
  const float f = fmaxf((r.k - (300.f + fabsf(r.k) * (1.f / 64.f))) * q.rkl, sizeof(T) == 2 ? -65504.f : -1e30f);
  floor = to_f<T>(from_f<T>(f));
  return r.sh == 0.f && fmaf(floor, q.kl, -r.k) <= -200.f;
}
// The same where the terms are cut off one by one.
constexpr float kNoTerm = -200.f;

__device__ __forceinline__ float redux_max(float v) {  // over the warp; NaN is passed over
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

constexpr float kHugeExponent = 4194304.f;  // 2^22
constexpr float kSlack = 16.f;              // a maximum this far above the reference moves it

//   m    largest x (before squash; -inf for an empty set, NaN is passed over)
//   r    the reference;  lim  the y above which it moves (-inf: nothing seen yet)
//   s    sum of e;  w  sum of e * d (entropy only)
// A -inf logit adds nothing (its term of w is cut off at a finite d); a NaN reaches s.
template <int CAP, bool ENT>
struct RowStats {
  float m, lim, s, w;
  Ref r;

  __device__ __forceinline__ void init() {
    m = lim = -INFINITY;
    s = w = 0.f;
    r = Ref{0.f, 0.f};
  }
  __device__ __forceinline__ bool unset() const { return lim == -INFINITY; }  // then s is 0 or NaN

  __device__ __forceinline__ void rebase(const Ref& to, const Squash& q) {
    if (!unset()) {
      const float f = ref_scale(r, to, q);
      if constexpr (ENT) w = f * fmaf(ref_diff(r, to, q), s, w);
      s *= f;
    }
    r = to;
  }

  // Takes the reference to the logit y.
  __device__ __forceinline__ void move(float y, const Squash& q) {
    const float t = y * q.kl;
    const bool huge = !(fabsf(t) < kHugeExponent);
    rebase(huge ? Ref{y, 0.f} : Ref{0.f, rintf(t)}, q);
    lim = huge ? y : (r.k + kSlack) * q.rkl;
  }

  // One logit (a row's head and tail).
  __device__ __forceinline__ void add1(float x, const Squash& q) {
    const float y = squash<CAP>(x, q);
    if (y > lim) move(y, q);
    m = fmaxf(m, x);
    const float d = exponent(y, r, q), e = ex2(d);
    s += e;
    if constexpr (ENT) w = fmaf(e, fmaxf(d, -1e30f), w);
  }

  // NW words as they lie in memory, lm their largest value.  Two elements at a time: 3.5 (with the
  // entropy 4.5) instructions an element for 16-bit types.
  template <typename T, int NW>
  __device__ __forceinline__ void add_words(const uint32_t (&w_)[NW], float lm, const Squash& q) {
    constexpr int P = NW * elems_per_word<T>() / 2;
    const float ly = squash<CAP>(lm, q);
    if (ly > lim) move(ly, q);
    m = fmaxf(m, lm);
    float2 s2 = make_float2(s, 0.f), w2 = make_float2(w, 0.f);
    const float2 kl = both(q.kl), nk = both(-r.k);
    if (!CAP && (ENT ? can_raise<T>(r, q) : r.sh == 0.f)) {
      uint32_t x[NW];
#pragma unroll
      for (int i = 0; i < NW; ++i) x[i] = ENT ? word_max_nan(w_[i], floor_word<T>(), (const T*)nullptr) : w_[i];
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float2 d = __ffma2_rn(word_pair<T>(x, i), kl, nk);
        const float2 e = make_float2(ex2(d.x), ex2(d.y));
        s2 = __fadd2_rn(s2, e);
        if constexpr (ENT) w2 = __ffma2_rn(e, d, w2);
      }
    } else if (CAP && r.sh == 0.f && all_near<T>(w_, lm, q)) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float2 d = __ffma2_rn(squash_near(word_pair<T>(w_, i), q), kl, nk);
        const float2 e = make_float2(ex2(d.x), ex2(d.y));
        s2 = __fadd2_rn(s2, e);
        if constexpr (ENT) w2 = __ffma2_rn(e, make_float2(fmaxf(d.x, -1e30f), fmaxf(d.y, -1e30f)), w2);
      }
    } else {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float2 x = word_pair<T>(w_, i);
        // without the polynomial: both forms in one unrolled loop cost more than they save
        const float2 y = CAP ? make_float2(squash_far<CAP>(x.x, q), squash_far<CAP>(x.y, q)) : x;
        const float2 d = make_float2(exponent(y.x, r, q), exponent(y.y, r, q));
        const float2 e = make_float2(ex2(d.x), ex2(d.y));
        s2 = __fadd2_rn(s2, e);
        if constexpr (ENT) w2 = __ffma2_rn(e, make_float2(fmaxf(d.x, -1e30f), fmaxf(d.y, -1e30f)), w2);
      }
    }
    s = s2.x + s2.y;
    if constexpr (ENT) w = w2.x + w2.y;
  }

  // Adds the statistics of another set.
  __device__ __forceinline__ void merge(RowStats o, const Squash& q) {
    m = fmaxf(m, o.m);
    if (!o.unset()) {
      if (unset() || ref_diff(o.r, r, q) > 0.f) {
        rebase(o.r, q);
        lim = o.lim;
      } else {
        o.rebase(r, q);
      }
    }
    s += o.s;
    if constexpr (ENT) w += o.w;
  }

  // Joins the sets of the warp's lanes; the same result on every lane.
  __device__ __forceinline__ void warp_merge(const Squash& q) {
    m = redux_max(m);
    if (__any_sync(0xffffffffu, r.sh != 0.f)) {
#pragma unroll 1
      for (int o = 16; o > 0; o >>= 1) {
        RowStats t;
        t.m = m;
        t.lim = __shfl_xor_sync(0xffffffffu, lim, o);
        t.s = __shfl_xor_sync(0xffffffffu, s, o);
        t.w = ENT ? __shfl_xor_sync(0xffffffffu, w, o) : 0.f;
        t.r.sh = __shfl_xor_sync(0xffffffffu, r.sh, o);
        t.r.k = __shfl_xor_sync(0xffffffffu, r.k, o);
        merge(t, q);
      }
      return;
    }
    const int top = __reduce_max_sync(0xffffffffu, unset() ? INT_MIN : (int)r.k);
    if (top != INT_MIN) {
      rebase(Ref{0.f, (float)top}, q);
      lim = (r.k + kSlack) * q.rkl;
    }
    s = warp_sum(s);
    if constexpr (ENT) w = warp_sum(w);
  }

  // Brings S into [1, 2) by moving the reference (exactly), so that log S is small next to it.
  __device__ __forceinline__ void center() {
    if (!(s > 0.f && s < INFINITY)) return;
    const int e = (int)(__float_as_uint(s) >> 23) - 127;
    const float f = __int_as_float((127 - e) << 23);
    if constexpr (ENT) w = (w - (float)e * s) * f;
    s *= f;
    r.k += (float)e;
  }
};

// log-probability of the logit y given a centred reference and log S.
__device__ __forceinline__ float log_prob(float y, const Ref& r, float logs, const Squash& q) {
  const float d = exponent(y, r, q);
  // a logit at the type's lowest value: only its product with kl overflows
  if (d == -INFINITY) return (y - (r.sh + r.k * q.rkl)) * q.inv_t - logs;
  return fmaf(d, kLn2, -logs);
}
// log sum exp.
__device__ __forceinline__ float ref_lse(const Ref& r, float logs, const Squash& q) {
  return fmaf(r.k, kLn2, logs) + r.sh * q.inv_t;
}

// ---------------------------------------------------------------------------
// Thread-block clusters: CTAs of one row
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t row_cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void row_cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
// For a CTA that leaves once the others have read its shared memory: arrive after the last read of
// theirs, without ordering any memory, and wait before the end.
__device__ __forceinline__ void row_cluster_arrive_relaxed() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
}
__device__ __forceinline__ void row_cluster_wait() { asm volatile("barrier.cluster.wait;" ::: "memory"); }
// A word at the same shared-memory offset in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t ld_cluster_u32(const void* p, uint32_t rank) {
  uint32_t a, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t ld_cluster_u64(const void* p, uint32_t rank) {
  uint32_t a;
  uint64_t v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}

// Clusters of `cs` CTAs of a persistent kernel that the device holds at once.
template <typename... KArgs>
inline cudaError_t resident_clusters(void (*kern)(KArgs...), int threads, int cs, size_t smem, int* n) {
  if (cs == 1) {
    int per_sm = 0;
    const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, smem);
    *n = std::max(1, per_sm) * sm_count();
    return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(cs * sm_count()));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cs;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaOccupancyMaxActiveClusters(n, kern, &cfg);
  *n = std::max(1, *n);
  return e;
}

// Launches `kern` with clusters of `cs` CTAs (none for 1).
template <typename... KArgs, typename... Args>
inline cudaError_t launch_rows(void (*kern)(KArgs...), int64_t grid, int threads, int cs, size_t smem,
                               cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cs;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cs > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

}  // namespace ak
