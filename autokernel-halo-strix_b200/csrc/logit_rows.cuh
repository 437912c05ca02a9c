// Device helpers shared by the operators over rows of logits (token log-probabilities,
// distillation): addressing of strided rows, 32-byte groups, running softmax statistics.
#pragma once

#include "ak_common.cuh"

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
struct Squash {
  float cap, inv_cap, inv_t, kl;
  float kc;  // -2 log2(e) / cap
};

inline Squash make_squash(float temperature, float softcap) {
  Squash q;
  q.cap = softcap > 0.f ? softcap : 0.f;
  q.inv_cap = softcap > 0.f ? 1.f / softcap : 0.f;
  q.kc = softcap > 0.f ? (float)(-2.0 * 1.4426950408889634 / (double)softcap) : 0.f;
  q.inv_t = 1.f / temperature;
  q.kl = (float)(1.4426950408889634 / (double)temperature);
  return q;
}

// cap tanh(x / cap) = cap (1 - E) / (1 + E) with E = e^(-2 |x| / cap) and x's sign: two special-unit
// operations.  With u = 2^-24, E's argument is off by 2 u relative and the hardware's exponential
// by 4 u, which reaches tanh as 2 E / (1 + E)^2 (4 |x / cap| + 4) u <= 2.4 u; the difference, the sum
// and the quick division add 6 u of tanh itself: at most 8 u absolute.
template <bool CAP>
__device__ __forceinline__ float squash(float x, const Squash& q) {
  if constexpr (!CAP) return x;
  const float e = ex2(fabsf(x) * q.kc);
  const float y = copysignf(q.cap * __fdividef(1.f - e, 1.f + e), x);
  return x == -INFINITY ? x : y;
}

// Derivative of squash at its output y.
template <bool CAP>
__device__ __forceinline__ float squash_slope(float y, const Squash& q) {
  if constexpr (!CAP) return 1.f;
  const float t = y * q.inv_cap;
  return y == -INFINITY ? 0.f : 1.f - t * t;
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

// Where a product of e = 2^(kl (x - mu)) with x - mu is formed, -inf has to be raised to a finite
// value whose e is still 0: to `floor`, which the type represents.  Holds where mu lies far enough
// above it (and below what a difference could overflow from); elsewhere the terms are cut off one
// by one.
template <typename T>
__device__ __forceinline__ float raise_floor() {
  return sizeof(T) == 2 && !std::is_same<T, __nv_bfloat16>::value ? -65504.f : -1.0e30f;
}
template <typename T>
__device__ __forceinline__ bool can_raise(float mu, const Squash& q) {
  return (mu - raise_floor<T>()) * q.kl > 200.f && mu < 1e30f;
}
template <typename T>
__device__ __forceinline__ uint32_t floor_word() {
  if constexpr (sizeof(T) == 4) return __float_as_uint(raise_floor<T>());
  else return pack2(raise_floor<T>(), raise_floor<T>(), (const T*)nullptr);
}

// ---------------------------------------------------------------------------
// Running softmax statistics of a set of logits
// ---------------------------------------------------------------------------
//   m   largest x (before squash; -inf for an empty set, NaN is passed over)
//   mu  what exponents are taken against: squash(m), or 0 where m is -inf
//   s   sum of e = 2^(kl (y - mu))
//   w   sum of e * (y - mu)    (entropy only)
// y - mu is formed before the scaling: the product with kl of a number near the type's lowest
// value would overflow, and a fused x * kl - mu * kl would turn that into NaN (and rounds mu * kl,
// an error that every term shares).  A -inf logit adds nothing; a NaN reaches s.
template <bool CAP, bool ENT>
struct RowStats {
  float m, mu, s, w;

  __device__ __forceinline__ void init() {
    m = -INFINITY;
    mu = 0.f;
    s = 0.f;
    w = 0.f;
  }

  // Moves the statistics to the larger maximum mn.
  __device__ __forceinline__ void rebase(float mn, const Squash& q) {
    const float nu = CAP ? squash<CAP>(mn, q) : mn;
    if (m != -INFINITY) {  // there s is 0 or NaN
      const float d = fmaxf(mu - nu, -1e30f);
      const float f = ex2(d * q.kl);
      if constexpr (ENT) w = f * fmaf(d, s, w);
      s *= f;
    }
    m = mn;
    mu = nu;
  }

  template <int N>
  __device__ __forceinline__ void add(const float (&x)[N], const Squash& q) {
    float lm = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) lm = fmaxf(lm, x[i]);
    add(x, lm, q);
  }

  // lm: the largest of x
  template <int N>
  __device__ __forceinline__ void add(const float (&x)[N], float lm, const Squash& q) {
    static_assert(N % 2 == 0 || N == 1, "pairs");
    if (lm > m) rebase(lm, q);
    if constexpr (N == 1) {
      const float d = squash<CAP>(x[0], q) - mu;
      const float e = ex2(d * q.kl);
      s += e;
      if constexpr (ENT) w = fmaf(e, fmaxf(d, -1e30f), w);
    } else {
      const float2 nmu = make_float2(-mu, -mu), kl = make_float2(q.kl, q.kl);
      float2 s2 = make_float2(s, 0.f), w2 = make_float2(w, 0.f);
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const float2 y = make_float2(squash<CAP>(x[i], q), squash<CAP>(x[i + 1], q));
        const float2 d = __fadd2_rn(y, nmu);
        const float2 a = __fmul2_rn(d, kl);
        const float2 e = make_float2(ex2(a.x), ex2(a.y));
        s2 = __fadd2_rn(s2, e);
        if constexpr (ENT) w2 = __ffma2_rn(e, make_float2(fmaxf(d.x, -1e30f), fmaxf(d.y, -1e30f)), w2);
      }
      s = s2.x + s2.y;
      if constexpr (ENT) w = w2.x + w2.y;
    }
  }

  // NW words as they lie in memory, lm their largest value.  Two elements at a time: 4 (with the
  // entropy 5) instructions an element for 16-bit types.
  template <typename T, int NW>
  __device__ __forceinline__ void add_words(const uint32_t (&w_)[NW], float lm, const Squash& q) {
    constexpr int P = NW * elems_per_word<T>() / 2;
    if (CAP || (ENT && !can_raise<T>(fmaxf(m, lm), q))) {
      float x[2 * P];
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float2 v = word_pair<T>(w_, i);
        x[2 * i] = v.x;
        x[2 * i + 1] = v.y;
      }
      add(x, lm, q);
      return;
    }
    if (lm > m) rebase(lm, q);
    const float2 nmu = make_float2(-mu, -mu), kl = make_float2(q.kl, q.kl);
    float2 s2 = make_float2(s, 0.f), w2 = make_float2(w, 0.f);
    uint32_t x[NW];
#pragma unroll
    for (int i = 0; i < NW; ++i) x[i] = ENT ? word_max_nan(w_[i], floor_word<T>(), (const T*)nullptr) : w_[i];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float2 d = __fadd2_rn(word_pair<T>(x, i), nmu);
      const float2 a = __fmul2_rn(d, kl);
      const float2 e = make_float2(ex2(a.x), ex2(a.y));
      s2 = __fadd2_rn(s2, e);
      if constexpr (ENT) w2 = __ffma2_rn(e, d, w2);
    }
    s = s2.x + s2.y;
    if constexpr (ENT) w = w2.x + w2.y;
  }

  // Adds the statistics of another set.
  __device__ __forceinline__ void merge(RowStats o, const Squash& q) {
    if (o.m > m) rebase(o.m, q);
    else if (m > o.m) o.rebase(m, q);
    s += o.s;
    if constexpr (ENT) w += o.w;
  }

  // Sums over the warp, the same on every lane.
  __device__ __forceinline__ void warp_merge(const Squash& q) {
    const float M = warp_max(m);
    if (M > m) rebase(M, q);
    s = warp_sum(s);
    if constexpr (ENT) w = warp_sum(w);
  }
};

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
