// Distillation from a teacher's top-K log-probabilities, sm_100a.
//
// Per row, y = softcap(x) / T, p = softmax(y), teacher entries (i_k, t_k), k < K:
//   renormalised: q = softmax of t over the K entries
//                 L = sum_k q_k (log q_k - log p_{i_k})
//                 T dL/dx_i = p_i - q_i
//   tail:         q_k = exp(t_k), r = max(0, 1 - sum q), p_r = sum of p outside the K tokens
//                 L = sum_k q_k (log q_k - log p_{i_k}) + r (log r - log p_r)
//                 T dL/dx_i = p_i - q_i at the teacher's tokens, p_i (1 - r / p_r) elsewhere
// (q_i: the teacher's mass on token i, entries of one token added up; times the softcap's slope).
//
// p_r = 1 - sum_k p_{i_k} would cancel where the student agrees with the teacher, so the rest is
// summed by itself, with a maximum of its own: the teacher's tokens are taken out of the row as it
// lies in shared memory (-inf), and join with the statistics of those K logits afterwards.
// A gradient outside the K tokens is e c with e = 2^(kl (y - mu_rest)) and the row's
// c = (share of p) / S - r / S_rest, which neither over- nor underflows where p_r does.
//
// One read of the logits: a CTA, or the CTAs of a cluster, bring the row into shared memory by
// bulk copies, form the statistics, and write the gradient from shared memory.
#include "logit_rows.cuh"

#include <algorithm>

namespace ak {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxK = 128;       // teacher entries
constexpr int kMaxCluster = 8;   // the portable cluster size
constexpr int kShareWanted = 56 * 1024;  // row bytes per CTA: four CTAs on an SM
constexpr int kShareMost = 216 * 1024;
constexpr float kMasked = 30000.f;
constexpr uint32_t kCopyBytes = 8192;    // of one bulk copy

struct DistillArgs {
  float* losses;        // [rows]
  void* grad;           // GRAD: [rows][V]
  float2* rest;         // !GRAD, nullable: (mu_rest, c) of each row, for the backward
  float* gk;            // !GRAD, nullable: [rows][K] T dL/dx at the teacher's tokens
  const int64_t* idx;   // [rows][K]
  const float* tlp;     // [rows][K]
  const uint8_t* mask;  // nullable [rows]
  const float* inv_n;   // GRAD, nullable: 1 / rows that count (host value in scale otherwise)
  RowAddr addr;
  float scale;          // GRAD: T, times 1 / rows without inv_n
  int V, K, cs, tail;
  Squash q;
  int* status;
};

// The gradient at a logit outside the teacher's tokens.  c = 0 gives 0 whatever x is.
template <bool CAP>
__device__ __forceinline__ float rest_grad(float x, float mu, float c, const Squash& q) {
  if (c == 0.f) return 0.f;
  const float y = squash<CAP>(x, q);
  return ex2((y - mu) * q.kl) * c * squash_slope<CAP>(y, q);
}

// The same for the values of NW words, two at a time without softcap.
template <typename T, bool CAP, int NW>
__device__ __forceinline__ void rest_grads(float* x, const uint32_t (&w)[NW], float mu, float c, const Squash& q) {
  constexpr int P = NW * elems_per_word<T>() / 2;
  const float2 nmu = make_float2(-mu, -mu), kl = make_float2(q.kl, q.kl), c2 = make_float2(c, c);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const float2 v = word_pair<T>(w, i);
    float2 o;
    if constexpr (CAP) {
      o = make_float2(rest_grad<CAP>(v.x, mu, c, q), rest_grad<CAP>(v.y, mu, c, q));
    } else if (c == 0.f) {
      o = make_float2(0.f, 0.f);
    } else {
      const float2 d = __fmul2_rn(__fadd2_rn(v, nmu), kl);
      o = __fmul2_rn(make_float2(ex2(d.x), ex2(d.y)), c2);
    }
    x[2 * i] = o.x;
    x[2 * i + 1] = o.y;
  }
}

template <typename T, bool CAP, bool GRAD>
__global__ void __launch_bounds__(kThreads)
distill_fwd_kernel(const T* __restrict__ logits, const DistillArgs a) {
  using Stats = RowStats<CAP, false>;
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ __align__(128) unsigned char s_row_raw[];  // this CTA's share of the row's groups
  T* s_row = reinterpret_cast<T*>(s_row_raw);
  __shared__ __align__(8) uint64_t s_bar;
  __shared__ Stats s_warp[kWarps];
  __shared__ float s_share[2];     // this CTA's statistics, read by the others of the cluster
  __shared__ float s_out[2];       // (mu_rest, c * scale) for the gradient
  __shared__ float s_edge[2][32];  // head and tail of the row
  __shared__ int s_idx[kMaxK];
  __shared__ float s_q[kMaxK];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cs = a.cs;
  const int64_t r = cs > 1 ? blockIdx.x / cs : blockIdx.x;
  const int rank = cs > 1 ? (int)row_cluster_rank() : 0;
  const Squash q = a.q;
  const T* row = logits + a.addr.off(r);
  const RowCut cut = cut_row(row, a.V);
  const int g0 = (int)((int64_t)cut.groups * rank / cs);
  const int n = ((int)((int64_t)cut.groups * (rank + 1) / cs) - g0) * kGroup;  // elements in s_row
  const int body0 = cut.head + g0 * kGroup;                                   // the first of them
  const int tail0 = cut.head + cut.groups * kGroup;
  const int head_here = rank == 0 ? cut.head : 0, tail_here = rank == cs - 1 ? cut.tail : 0;
  T* grow = GRAD ? reinterpret_cast<T*>(a.grad) + r * a.V : nullptr;
  const bool vec = GRAD && (reinterpret_cast<uintptr_t>(grow + body0) & 15u) == 0;
  const bool live = a.mask == nullptr || a.mask[r] != 0;

  if (!live) {  // the same in every CTA of the row; what the row holds is not looked at
    if constexpr (GRAD) {
      const float zero[VEC] = {};
      for (int v = tid; v < n / VEC; v += kThreads) {
        if (vec) store_frag<T, VEC>(grow + body0 + v * VEC, zero);
        else
          for (int i = 0; i < VEC; ++i) grow[body0 + v * VEC + i] = from_f<T>(0.f);
      }
      if (tid < head_here) grow[tid] = from_f<T>(0.f);
      if (tid < tail_here) grow[tail0 + tid] = from_f<T>(0.f);
    }
    if (rank == 0) {
      if (tid == 0) {
        a.losses[r] = 0.f;
        if (!GRAD && a.rest) a.rest[r] = make_float2(0.f, 0.f);
      }
      if (!GRAD && a.gk && tid < a.K) a.gk[r * a.K + tid] = 0.f;
    }
    return;
  }

  // ---- the row on its way into shared memory
  if (tid == 0) {
    mbar_init(&s_bar, 1);
    mbar_fence_init();
    const uint32_t bytes = (uint32_t)(n * sizeof(T));
    mbar_arrive_expect_tx(&s_bar, bytes);
    const char* src = reinterpret_cast<const char*>(row + body0);
    for (uint32_t o = 0; o < bytes; o += kCopyBytes)
      bulk_g2s(s_row_raw + o, src + o, min(kCopyBytes, bytes - o), &s_bar);
  }
  if (warp == 1 && lane < head_here) s_edge[0][lane] = to_f<T>(row[lane]);
  if (warp == 2 && lane < tail_here) s_edge[1][lane] = to_f<T>(row[tail0 + lane]);
  __syncthreads();

  // ---- the teacher's entries, all on the first warp: entry 32 j + lane in slot j.  A negative
  // index is padding.
  constexpr int S = kMaxK / 32;
  int idx[S];
  float yk[S], qk[S], logq[S], mass[S];
  Stats top;  // the teacher's tokens
  top.init();
  bool bad = false, none = false;
  float rest = 0.f;
  if (warp == 0) {
    float t[S], xk[S];
    bool any = false;
#pragma unroll
    for (int j = 0; j < S; ++j) {
      const int k = 32 * j + lane;
      idx[j] = -1;
      t[j] = yk[j] = xk[j] = -INFINITY;
      if (k < a.K) {
        const int64_t i = a.idx[r * a.K + k];
        bad |= i >= a.V;
        if (i >= 0 && i < a.V) {
          idx[j] = (int)i;
          t[j] = a.tlp[r * a.K + k];
          xk[j] = to_f<T>(row[i]);
          yk[j] = squash<CAP>(xk[j], q);
          any = true;
        }
      }
    }
    bad = __any_sync(0xffffffffu, bad);
    any = __any_sync(0xffffffffu, any);
    float qsum = 0.f;
    if (a.tail) {
#pragma unroll
      for (int j = 0; j < S; ++j) {
        qk[j] = idx[j] >= 0 ? expf(t[j]) : 0.f;
        logq[j] = t[j];
        qsum += qk[j];
      }
      qsum = warp_sum(qsum);
    } else {
      float tm = t[0], z = 0.f;
#pragma unroll
      for (int j = 1; j < S; ++j) tm = fmaxf(tm, t[j]);
      tm = warp_max(tm);
#pragma unroll
      for (int j = 0; j < S; ++j) {
        qk[j] = (idx[j] >= 0 && tm != -INFINITY) ? expf(t[j] - tm) : 0.f;
        z += qk[j];
      }
      z = warp_sum(z);
      const float logz = logf(z);
#pragma unroll
      for (int j = 0; j < S; ++j) {
        qk[j] = z == 0.f ? 0.f : qk[j] / z;  // z: 0 without entries, NaN kept
        logq[j] = t[j] - tm - logz;
        qsum += qk[j];
      }
      qsum = warp_sum(qsum);
    }
    none = a.tail ? !any : qsum == 0.f;  // no teacher: loss 0, no gradient
    rest = a.tail ? fmaxf(1.f - qsum, 0.f) : 0.f;
#pragma unroll
    for (int j = 0; j < S; ++j) {
      mass[j] = 0.f;
      s_idx[32 * j + lane] = idx[j];
      s_q[32 * j + lane] = qk[j];
    }
    __syncwarp();
    // entries of one token: its logit counts once, at the first of them; their masses add up
    uint32_t later = 0;
    for (int m = 0; m < a.K; ++m) {
      const int im = s_idx[m];
      const float qm = s_q[m];
#pragma unroll
      for (int j = 0; j < S; ++j) {
        if (32 * j < a.K && idx[j] == im) {
          mass[j] += qm;
          if (m < 32 * j + lane) later |= 1u << j;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < S; ++j) {
      if (idx[j] >= 0 && !(later >> j & 1u)) {
        const float x[1] = {xk[j]};
        top.add(x, q);
      }
    }
    top.warp_merge(q);
    // out of the row, once it is here
    mbar_wait_bounded(&s_bar, 0u, a.status);
#pragma unroll
    for (int j = 0; j < S; ++j) {
      const int i = idx[j];
      if (i < 0) continue;
      if (i >= body0 && i < body0 + n) s_row[i - body0] = from_f<T>(-INFINITY);
      else if (i < head_here) s_edge[0][i] = -INFINITY;
      else if (i >= tail0 && i - tail0 < tail_here) s_edge[1][i - tail0] = -INFINITY;
    }
  }
  __syncthreads();

  // ---- the rest of the row
  mbar_wait_bounded(&s_bar, 0u, a.status);  // complete: makes the copies visible to each thread
  Stats st;
  st.init();
  constexpr int U = 2;  // 16-byte pieces at a time
  const int nv = n / VEC;
  const uint4* s_vec = reinterpret_cast<const uint4*>(s_row_raw);
  int v = tid;
  for (; v + (U - 1) * kThreads < nv; v += U * kThreads) {
    uint32_t w[4 * U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint4 f = s_vec[v + u * kThreads];
      w[4 * u] = f.x; w[4 * u + 1] = f.y; w[4 * u + 2] = f.z; w[4 * u + 3] = f.w;
    }
    st.template add_words<T>(w, words_max<T>(w), q);
  }
  for (; v < nv; v += kThreads) {
    const uint4 f = s_vec[v];
    const uint32_t w[4] = {f.x, f.y, f.z, f.w};
    st.template add_words<T>(w, words_max<T>(w), q);
  }
  if (warp < 2 && lane < (warp == 0 ? head_here : tail_here)) {
    const float x[1] = {s_edge[warp][lane]};
    st.add(x, q);
  }
  st.warp_merge(q);
  if (lane == 0) s_warp[warp] = st;
  __syncthreads();
  if (warp == 0) {
    st.init();
    if (lane < kWarps) st = s_warp[lane];
    st.warp_merge(q);
    if (lane == 0) { s_share[0] = st.m; s_share[1] = st.s; }
  }
  if (cs > 1) {
    row_cluster_sync();
    if (warp == 0) {
      st.init();
      if (lane < cs) {  // every CTA joins them in the same way
        const float m = __uint_as_float(ld_cluster_u32(&s_share[0], lane));
        st.s = __uint_as_float(ld_cluster_u32(&s_share[1], lane));
        if (m != -INFINITY) { st.m = m; st.mu = squash<CAP>(m, q); }
      }
      st.warp_merge(q);
    }
  }

  // ---- loss and coefficients
  const float scale = GRAD ? (a.inv_n ? a.scale * *a.inv_n : a.scale) : 1.f;
  float gk[S];
  if (warp == 0) {
    Stats all = st;
    all.merge(top, q);
    const float logs = logf(all.s);
    const bool empty = all.s == 0.f;  // every logit is -inf: no distribution, no gradient
    float loss = 0.f;
#pragma unroll
    for (int j = 0; j < S; ++j) {
      const float lpk = (empty || yk[j] == -INFINITY) ? -INFINITY : (yk[j] - all.mu) * q.inv_t - logs;
      if (idx[j] >= 0 && qk[j] != 0.f) loss += qk[j] * (logq[j] - lpk);
      gk[j] = 0.f;
      if (idx[j] >= 0 && !none && !empty) gk[j] = (expf(lpk) - mass[j]) * squash_slope<CAP>(yk[j], q);
      if (bad) gk[j] = NAN;
    }
    loss = warp_sum(loss);
    // the scale of p in units of e: p = e 2^(kl (mu_rest - mu)) / S
    float c = (none || st.s == 0.f) ? 0.f : ex2((st.mu - all.mu) * q.kl) / all.s;
    // The rest is left out where the student has masked it: no logit outside the teacher's tokens
    // above -inf, or none within kMasked of the largest (a mask of the type's lowest value).
    if (rest > 0.f && st.s != 0.f && !none && !(st.mu - all.mu < -kMasked)) {
      loss += rest * (logf(rest) - ((st.mu - all.mu) * q.inv_t + logf(st.s) - logs));
      c -= rest / st.s;
    }
    if (bad) { loss = NAN; c = NAN; }
    if (lane == 0) {
      if (rank == 0) a.losses[r] = loss;
      s_out[0] = st.mu;
      s_out[1] = c * scale;
      if (!GRAD && rank == 0 && a.rest) a.rest[r] = make_float2(st.mu, c);
    }
    if (!GRAD && rank == 0 && a.gk) {
#pragma unroll
      for (int j = 0; j < S; ++j)
        if (32 * j + lane < a.K) a.gk[r * a.K + 32 * j + lane] = gk[j];
    }
  }

  if constexpr (GRAD) {
    __syncthreads();
    if (cs > 1) row_cluster_arrive_relaxed();  // this CTA has read the others' statistics
    const float mu = s_out[0], cg = s_out[1];
    for (int u = tid; u < nv; u += kThreads) {
      const uint4 f = s_vec[u];
      const uint32_t w[4] = {f.x, f.y, f.z, f.w};
      float x[VEC];
      rest_grads<T, CAP>(x, w, mu, cg, q);
      T* out = grow + body0 + u * VEC;
      if (vec) store_frag<T, VEC>(out, x);
      else
        for (int i = 0; i < VEC; ++i) out[i] = from_f<T>(x[i]);
    }
    if (warp < 2 && lane < (warp == 0 ? head_here : tail_here))
      grow[(warp == 0 ? 0 : tail0) + lane] = from_f<T>(rest_grad<CAP>(s_edge[warp][lane], mu, cg, q));
    __syncthreads();  // the teacher's tokens over what was written for them
    if (warp == 0) {
#pragma unroll
      for (int j = 0; j < S; ++j) {
        const int i = idx[j];
        if (i >= 0 && ((i >= body0 && i < body0 + n) || i < head_here || (i >= tail0 && i - tail0 < tail_here)))
          grow[i] = from_f<T>(gk[j] * scale);
      }
    }
  } else if (cs > 1) {
    row_cluster_arrive_relaxed();
  }
  if (cs > 1) row_cluster_wait();  // the others have read this one's
}

struct DistillBwdArgs {
  const float2* rest;
  const float* gk;
  const int64_t* idx;
  const uint8_t* mask;
  const float* inv_n;
  const float* g_loss;
  RowAddr addr;
  float scale;
  int V, K, segs;
  Squash q;
};

constexpr int kBwdBatch = 2;
constexpr int kBwdGroups = kThreads * kBwdBatch;

// The gradient from the forward's (mu_rest, c) and K numbers a row: each CTA takes one segment of a
// row, then writes those of the teacher's tokens that lie in it.
template <typename T, bool CAP>
__global__ void __launch_bounds__(kThreads)
distill_bwd_kernel(T* __restrict__ grad, const T* __restrict__ logits, const DistillBwdArgs a) {
  const int tid = threadIdx.x;
  const uint32_t r32 = blockIdx.x / (uint32_t)a.segs;
  const int64_t r = r32;
  const int seg = (int)(blockIdx.x - r32 * (uint32_t)a.segs);
  const Squash q = a.q;
  const T* row = logits + a.addr.off(r);
  T* grow = grad + r * a.V;
  const RowCut cut = cut_row(row, a.V);
  const bool vec = (reinterpret_cast<uintptr_t>(grow + cut.head) & 31u) == 0;
  const bool live = a.mask == nullptr || a.mask[r] != 0;
  const float scale = a.scale * (a.inv_n ? *a.inv_n : 1.f) * *a.g_loss;
  const float2 rc = a.rest[r];
  const float mu = rc.x, c = live ? rc.y * scale : 0.f;  // c = 0: zeros, whatever the row holds
  const int gbeg = seg * kBwdGroups;
  const T* body = row + cut.head;
  T* gbody = grow + cut.head;
  RawGroup<T> raw[kBwdBatch];
#pragma unroll
  for (int u = 0; u < kBwdBatch; ++u) {
    const int g = gbeg + u * kThreads + tid;
    if (g < cut.groups) raw[u] = load_group<T>(body + (int64_t)g * kGroup);
  }
#pragma unroll
  for (int u = 0; u < kBwdBatch; ++u) {
    const int g = gbeg + u * kThreads + tid;
    if (g < cut.groups) {
      float x[kGroup];
#pragma unroll
      for (int h = 0; h < (int)sizeof(T) / 2; ++h)
        rest_grads<T, CAP>(x + h * 16 / ((int)sizeof(T) / 2), raw[u].r[h].w, mu, c, q);
      store_group<T>(gbody + (int64_t)g * kGroup, x, vec);
    }
  }
  const int tail0 = cut.head + cut.groups * kGroup;
  const bool first = seg == 0, last = seg == a.segs - 1;
  if (first && tid < cut.head) grow[tid] = from_f<T>(rest_grad<CAP>(to_f<T>(row[tid]), mu, c, q));
  if (last && tid < cut.tail)
    grow[tail0 + tid] = from_f<T>(rest_grad<CAP>(to_f<T>(row[tail0 + tid]), mu, c, q));
  if (!live) return;
  __syncthreads();
  if (tid < a.K) {
    const int64_t i = a.idx[r * a.K + tid];
    const int64_t lo = first ? 0 : cut.head + (int64_t)gbeg * kGroup;
    const int64_t hi = last ? a.V : cut.head + (int64_t)(gbeg + kBwdGroups) * kGroup;
    if (i >= lo && i < hi && i < a.V) grow[i] = from_f<T>(a.gk[r * a.K + tid] * scale);
  }
}

// inv_n[0] = 1 / max(1, rows whose mask is set).
__global__ void __launch_bounds__(1024)
distill_inv_rows(float* __restrict__ inv_n, const uint8_t* __restrict__ mask, int64_t rows) {
  __shared__ int s[32];
  int c = 0;
  for (int64_t i = threadIdx.x; i < rows; i += blockDim.x) c += mask[i] != 0;
  c = __reduce_add_sync(0xffffffffu, c);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    int t = 0;
    for (int i = 0; i < 32; ++i) t += s[i];
    inv_n[0] = 1.f / (float)max(t, 1);
  }
}

// loss[0] = mult * inv_n * sum of the rows' losses, in a fixed order.
__global__ void __launch_bounds__(1024)
distill_mean(float* __restrict__ loss, const float* __restrict__ losses, const float* __restrict__ inv_n,
             float mult, int64_t rows) {
  __shared__ float s[32];
  float v = 0.f;
  for (int64_t i = threadIdx.x; i < rows; i += blockDim.x) v += losses[i];
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = 0.f;
    for (int i = 0; i < 32; ++i) t += s[i];
    loss[0] = t * mult * (inv_n ? *inv_n : 1.f);
  }
}

int64_t share_bytes(int64_t V, int cs, int es) { return ((V / kGroup + cs - 1) / cs) * kGroup * es; }

// CTAs per row: as many as bring the share to kShareWanted, and more while the rows leave SMs
// without a CTA and each CTA keeps half a group per thread.
int cluster_for(int64_t rows, int64_t V, int es) {
  int cs = 1;
  while (cs < kMaxCluster && share_bytes(V, cs, es) > kShareWanted) cs *= 2;
  while (cs < kMaxCluster && rows * cs * 2 <= sm_count() * 2 && V / (2 * cs) >= kThreads * kGroup / 2) cs *= 2;
  return cs;
}

int check_args(const char* what, const void* logits, int64_t rows, int64_t inner, int64_t V, int64_t K,
               float temperature, float softcap, int dt) {
  AK_REQUIRE(valid_dtype(dt), AK_ERR_DTYPE, "%s: unsupported dtype %d", what, dt);
  AK_REQUIRE(rows >= 0 && rows < (1LL << 27) && inner > 0 && V > 0 && V < (1LL << 30), AK_ERR_SHAPE,
             "%s: bad shape: %lld rows of %lld", what, (long long)rows, (long long)V);
  AK_REQUIRE(K >= 1 && K <= kMaxK, AK_ERR_SHAPE, "%s: teacher entries per row must be in 1..%d, got %lld", what, kMaxK,
             (long long)K);
  AK_REQUIRE(share_bytes(V, kMaxCluster, elem_size(dt)) <= kShareMost, AK_ERR_SHAPE,
             "%s: a row of %lld elements does not fit the shared memory of %d CTAs", what, (long long)V, kMaxCluster);
  AK_REQUIRE(temperature > 0.f && temperature < INFINITY, AK_ERR_ARG, "%s: temperature must be positive and finite",
             what);
  AK_REQUIRE(softcap >= 0.f && softcap < INFINITY, AK_ERR_ARG, "%s: softcap must be >= 0 and finite", what);
  AK_REQUIRE(rows == 0 || logits, AK_ERR_ARG, "%s: null pointer", what);
  AK_REQUIRE((reinterpret_cast<uintptr_t>(logits) % elem_size(dt)) == 0, AK_ERR_ARG,
             "%s: logits not aligned to their type", what);
  return AK_OK;
}

template <typename T>
int launch_fwd(const T* logits, const DistillArgs& a, int64_t rows, cudaStream_t st) {
  const bool cap = a.q.cap > 0.f;
  auto kern = a.grad ? (cap ? distill_fwd_kernel<T, true, true> : distill_fwd_kernel<T, false, true>)
                     : (cap ? distill_fwd_kernel<T, true, false> : distill_fwd_kernel<T, false, false>);
  const size_t smem = (size_t)share_bytes(a.V, a.cs, sizeof(T)) + 16;
  AK_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
              "ak_distill_topk_fwd: shared memory");
  AK_CUDA_TRY(launch_rows(kern, rows * a.cs, kThreads, a.cs, smem, st, logits, a), "ak_distill_topk_fwd");
  return AK_OK;
}

}  // namespace
}  // namespace ak

using namespace ak;

extern "C" int ak_distill_topk_fwd(float* loss, float* losses, float* inv_n, void* grad, float* rest_stats, float* gk,
                                   const void* logits, const int64_t* teacher_idx, const float* teacher_lp,
                                   const uint8_t* mask, int64_t rows, int64_t inner, int64_t stride_outer,
                                   int64_t stride_inner, int64_t V, int64_t K, float temperature, float softcap,
                                   int tail, int dt, int* status, void* stream) {
  clear_error();
  int rc = check_args("ak_distill_topk_fwd", logits, rows, inner, V, K, temperature, softcap, dt);
  if (rc) return rc;
  AK_REQUIRE(loss, AK_ERR_ARG, "ak_distill_topk_fwd: null pointer");
  AK_REQUIRE(rows == 0 || (losses && teacher_idx && teacher_lp && (!mask || inv_n)), AK_ERR_ARG,
             "ak_distill_topk_fwd: null pointer");
  AK_REQUIRE(!grad || (!rest_stats && !gk), AK_ERR_ARG,
             "ak_distill_topk_fwd: the gradient, or what its kernel needs, not both");
  AK_REQUIRE((reinterpret_cast<uintptr_t>(grad) % elem_size(dt)) == 0, AK_ERR_ARG,
             "ak_distill_topk_fwd: grad not aligned to its type");
  cudaStream_t st = (cudaStream_t)stream;
  if (rows > 0) {
    if (mask) {
      distill_inv_rows<<<1, 1024, 0, st>>>(inv_n, mask, rows);
      AK_CHECK_LAUNCH("ak_distill_topk_fwd");
    }
    DistillArgs a{};
    a.losses = losses; a.grad = grad;
    a.rest = reinterpret_cast<float2*>(rest_stats);
    a.gk = gk; a.idx = teacher_idx; a.tlp = teacher_lp; a.mask = mask;
    a.inv_n = mask ? inv_n : nullptr;
    a.addr = RowAddr{inner, stride_outer, stride_inner};
    a.scale = mask ? temperature : temperature / (float)rows;
    a.V = (int)V; a.K = (int)K; a.cs = cluster_for(rows, V, elem_size(dt)); a.tail = tail != 0;
    a.q = make_squash(temperature, softcap);
    a.status = status;
    AK_DISPATCH_DTYPE(dt, T, rc = launch_fwd<T>((const T*)logits, a, rows, st));
    if (rc) return rc;
  }
  distill_mean<<<1, 1024, 0, st>>>(loss, losses, (mask && rows > 0) ? inv_n : nullptr,
                                   temperature * temperature / ((mask || rows == 0) ? 1.f : (float)rows), rows);
  AK_CHECK_LAUNCH("ak_distill_topk_fwd");
  return AK_OK;
}

extern "C" int ak_distill_topk_bwd(void* grad, const void* logits, const int64_t* teacher_idx,
                                   const float* rest_stats, const float* gk, const uint8_t* mask, const float* inv_n,
                                   const float* g_loss, int64_t rows, int64_t inner, int64_t stride_outer,
                                   int64_t stride_inner, int64_t V, int64_t K, float temperature, float softcap,
                                   int dt, void* stream) {
  clear_error();
  int rc = check_args("ak_distill_topk_bwd", logits, rows, inner, V, K, temperature, softcap, dt);
  if (rc) return rc;
  if (rows == 0) return AK_OK;
  AK_REQUIRE(grad && teacher_idx && rest_stats && gk && g_loss && (!mask || inv_n), AK_ERR_ARG,
             "ak_distill_topk_bwd: null pointer");
  AK_REQUIRE((reinterpret_cast<uintptr_t>(grad) % elem_size(dt)) == 0, AK_ERR_ARG,
             "ak_distill_topk_bwd: grad not aligned to its type");
  DistillBwdArgs a{};
  a.rest = reinterpret_cast<const float2*>(rest_stats);
  a.gk = gk; a.idx = teacher_idx; a.mask = mask; a.inv_n = mask ? inv_n : nullptr; a.g_loss = g_loss;
  a.addr = RowAddr{inner, stride_outer, stride_inner};
  a.scale = mask ? temperature : temperature / (float)rows;
  a.V = (int)V; a.K = (int)K;
  a.segs = (int)std::max<int64_t>(1, (V / kGroup + kBwdGroups - 1) / kBwdGroups);
  a.q = make_squash(temperature, softcap);
  AK_REQUIRE(rows * a.segs < (1LL << 31), AK_ERR_SHAPE, "ak_distill_topk_bwd: too many rows");
  const bool cap = a.q.cap > 0.f;
  AK_DISPATCH_DTYPE(dt, T, {
    auto kern = cap ? distill_bwd_kernel<T, true> : distill_bwd_kernel<T, false>;
    kern<<<(unsigned)(rows * a.segs), kThreads, 0, (cudaStream_t)stream>>>((T*)grad, (const T*)logits, a);
  });
  AK_CHECK_LAUNCH("ak_distill_topk_bwd");
  return AK_OK;
}
