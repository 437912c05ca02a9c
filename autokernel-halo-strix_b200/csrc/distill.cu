// Distillation from a teacher's top-K log-probabilities, sm_100a.
//
// Per row, y = softcap(x) / T, p = softmax(y), teacher entries (i_k, t_k), k < K:
//   renormalised: q = softmax of t over the K entries
//                 L = sum_k q_k (log q_k - log p_{i_k})
//                 T dL/dx_i = p_i - q_i
//   tail:         q_k = exp(t_k), r = max(0, 1 - sum q), p_r = sum of p outside the K tokens
//                 L = sum_k q_k (log q_k - log p_{i_k}) + r (log r - log p_r)
//                 T dL/dx_i = Q p_i - q_i at the teacher's tokens, Q p_i - r p_i / p_r elsewhere
// (q_i: the teacher's mass on token i, entries of one token added up; Q: the mass of all terms of L,
// sum q + r; times the softcap's slope).  Where the rest has no term (the student has masked it, or
// sum q > 1) Q is sum q.
//
// p_r = 1 - sum_k p_{i_k} would cancel where the student agrees with the teacher, so the rest is
// summed by itself, with a maximum of its own: the teacher's tokens are taken out of the row as it
// lies in shared memory (-inf), and join with the statistics of those K logits afterwards.
// A gradient outside the K tokens is e c with e = 2^d against the rest's reference and the row's
// c = (share of p) / S - r / S_rest, which neither over- nor underflows where p_r does.
//
// One read of the logits: a CTA, or the CTAs of a cluster, bring the row into shared memory by
// bulk copies, form the statistics, and write the gradient from shared memory.  The kernel is
// persistent and its warps have roles, so that a row's long chain of small steps (its indices, the
// K logits they point at, the masses of repeated tokens) runs while the row before it is worked on:
//   loader    copies the next row piece by piece, each as soon as compute has left that piece
//   teacher   the K entries of the next row; takes their tokens out of it when it has arrived
//   compute   statistics of the rest, then the gradient from them
//   finisher  the row's loss, and the gradient at the teacher's tokens over what compute wrote
// Rows of up to 8 KB take one warp each instead: their fixed steps overlap across many rows.
//
// What it measured (loss and gradient, GPU time, floors at the measured 6551 GB/s):
//   8192 x 50304 bf16, K 64       381 us, floor 253: no unit is saturated (issue slots 48 % active,
//                                 special units 48 %, 40 % of the warps): it waits.  Two CTAs an SM
//                                 hold one row each, so nothing is left to load during a row's
//                                 statistics.  Leaving out the stores changes nothing, leaving out
//                                 either pass's exponentials 10 %
//   the same, softcap 30          711 us: issue slots 56 %, twice the instructions
//   3000 x 50257 fp32, K 20       252 us, floor 184
//   16000 x 20000 bf16, K 100     450 us, floor 195: the teacher's warp
//   60000 x 4000 bf16, K 32       220 us, floor 146 (a warp each)
//   100000 x 1500 bf16, K 8       240 us, floor 92 (a warp each)
//   1023 x 50257 fp16, K 33       38 us forward + 37 us backward, floors 16 + 31
// Tried and dropped: one CTA with two row buffers (405 us), no roles (398 us), two teacher warps
// (423 us), four CTAs of half rows (480 us).
#include "logit_rows.cuh"

#include <algorithm>

namespace ak {
namespace {

constexpr int kThreads = 256;    // of the backward kernel
constexpr int kRoles = 3;        // loader, teacher, finisher
// Compute warps: kWide of them with two CTAs on an SM, which a long row (100 KB of shared memory)
// allows anyhow; kNarrow with four CTAs for shares up to kShareNarrow, where what counts is how many
// rows are under way at once.
constexpr int kWide = 11, kNarrow = 5;
constexpr int kShareNarrow = 44 * 1024;
constexpr int kMaxK = 128;       // teacher entries
constexpr int kSlots = kMaxK / 32;
constexpr int kMaxCluster = 8;   // the portable cluster size
constexpr int kShareWanted = 101 * 1024;  // bytes of one row in one CTA: two CTAs fit an SM
constexpr int kShareMost = 208 * 1024;    // of a row too long for that in eight CTAs
constexpr int kPieces = 8;                // a buffer is handed back in pieces
constexpr float kMasked = 30000.f;
constexpr int64_t kCountRows = 1024;      // rows up to which every warp counts the mask

struct DistillArgs {
  float* losses;        // [rows]
  void* grad;           // GRAD: [rows][V]
  float4* rest;         // !GRAD, nullable: (reference, c) of each row's rest, for the backward
  float* gk;            // !GRAD, nullable: [rows][K] T dL/dx at the teacher's tokens
  const int64_t* idx;   // [rows][K]
  const float* tlp;     // [rows][K]
  const uint8_t* mask;  // nullable [rows]
  const float* inv_n;   // GRAD, nullable: 1 / rows that count (else each warp counts the mask itself)
  RowAddr addr;
  int64_t rows;
  float scale;          // GRAD: T, times 1 / rows without a mask
  int V, K, log_cs, tail;
  uint32_t piece;       // bytes of a piece of the row buffer
  Squash q;
  int* status;
};

// 1 / max(1, rows whose mask is set), counted by one warp.
__device__ __forceinline__ float count_rows(const uint8_t* mask, int64_t rows) {
  int c = 0;
  for (int64_t i = threadIdx.x & 31; i < rows; i += 32) c += mask[i] != 0;
  return 1.f / (float)max(__reduce_add_sync(0xffffffffu, c), 1);
}
__device__ __forceinline__ float grad_scale(const DistillArgs& a) {
  if (a.mask == nullptr) return a.scale;
  return a.scale * (a.inv_n ? *a.inv_n : count_rows(a.mask, a.rows));
}

// The gradient at a logit outside the teacher's tokens.  c = 0 gives 0 whatever x is.
template <int CAP>
__device__ __forceinline__ float rest_grad_at(float y, const Ref& ref, float c, const Squash& q) {  // y: squashed
  if (c == 0.f) return 0.f;
  return ex2(exponent(y, ref, q)) * c * squash_slope<CAP>(y, q);
}
template <int CAP>
__device__ __forceinline__ float rest_grad(float x, const Ref& ref, float c, const Squash& q) {
  return rest_grad_at<CAP>(squash<CAP>(x, q), ref, c, q);
}

// The same for the values of NW words, two at a time where it can.
template <typename T, int CAP, int NW>
__device__ __forceinline__ void rest_grads(float* x, const uint32_t (&w)[NW], const Ref& ref, float c, const Squash& q) {
  constexpr int P = NW * elems_per_word<T>() / 2;
  const float2 kl = both(q.kl), nk = both(-ref.k), c2 = both(c);
  if (!CAP && ref.sh == 0.f && c != 0.f) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float2 d = __ffma2_rn(word_pair<T>(w, i), kl, nk);
      const float2 o = __fmul2_rn(make_float2(ex2(d.x), ex2(d.y)), c2);
      x[2 * i] = o.x;
      x[2 * i + 1] = o.y;
    }
  } else if (CAP && ref.sh == 0.f && c != 0.f && all_near<T>(w, words_max<T>(w), q)) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float2 y = squash_near(word_pair<T>(w, i), q);
      const float2 d = __ffma2_rn(y, kl, nk);
      const float2 o = __fmul2_rn(__fmul2_rn(make_float2(ex2(d.x), ex2(d.y)), c2), squash_slope_near(y, q));
      x[2 * i] = o.x;
      x[2 * i + 1] = o.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const float2 v = word_pair<T>(w, i);
      x[2 * i] = rest_grad_at<CAP>(CAP ? squash_far<CAP>(v.x, q) : v.x, ref, c, q);
      x[2 * i + 1] = rest_grad_at<CAP>(CAP ? squash_far<CAP>(v.y, q) : v.y, ref, c, q);
    }
  }
}

// The gradients of one 16-byte vector, rounded to T and stored.
template <typename T, int CAP>
__device__ __forceinline__ void store_grads(T* out, const uint4& f, const Ref& ref, float c, const Squash& q, bool vec) {
  constexpr int VEC = 16 / sizeof(T);
  const uint32_t w[4] = {f.x, f.y, f.z, f.w};
  float x[VEC];
  rest_grads<T, CAP>(x, w, ref, c, q);
  if (vec) {
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) o[i] = __float_as_uint(x[i]);
      else o[i] = pack2(x[2 * i], x[2 * i + 1], (const T*)nullptr);
    }
    *reinterpret_cast<uint4*>(out) = make_uint4(o[0], o[1], o[2], o[3]);
  } else {
    for (int i = 0; i < VEC; ++i) out[i] = from_f<T>(x[i]);
  }
}

// One CTA's share of a row: n elements from body0 in its buffer, and the row's head (first CTA) or
// tail (last CTA) as loose elements.
template <typename T>
struct Share {
  const T* row;
  int body0, n, tail0, head_here, tail_here;
  __device__ __forceinline__ Share(const T* row_, int V, int rank, int log_cs) : row(row_) {
    const RowCut cut = cut_row(row_, V);
    const int g0 = (int)(((int64_t)cut.groups * rank) >> log_cs);
    n = ((int)(((int64_t)cut.groups * (rank + 1)) >> log_cs) - g0) * kGroup;
    body0 = cut.head + g0 * kGroup;
    tail0 = cut.head + cut.groups * kGroup;
    head_here = rank == 0 ? cut.head : 0;
    tail_here = rank == (1 << log_cs) - 1 ? cut.tail : 0;
  }
  __device__ __forceinline__ bool has(int i) const {
    return (i >= body0 && i < body0 + n) || i < head_here || (i >= tail0 && i - tail0 < tail_here);
  }
};

// What the teacher's warp hands on with a row.
struct TeacherRow {
  float m, lim, s;  // statistics of the teacher's tokens, each once
  Ref r;
  float rest;      // r
  float total;     // sum q
  int none, bad;
  int idx[kMaxK];  // -1: no entry
  float q[kMaxK], logq[kMaxK], y[kMaxK], mass[kMaxK];
};

// What compute hands to the finisher.
struct FinishRow {
  Ref all, rest;
  float logs, tail_loss, c, mass;  // mass: Q
  int empty;
};

// Bounded waits.  The first that runs out reports AK_ERR_TIMEOUT and raises the CTA's abort flag;
// the later ones return at once, so the kernel runs to its end without waiting and its outputs are
// invalid.  Roles hand over to one another by these waits alone: one role may then run any number of
// rows ahead of another, which a barrier that counts threads would not survive.  The only barriers
// of that kind are among the compute warps (each passes one a live row, in step or not at all) and
// at the kernel's end.
struct Waits {
  int* status;
  volatile int* abort;
  template <bool kCluster>
  __device__ __forceinline__ void operator()(uint64_t* bar, uint32_t parity) const {
    if (*abort) return;
    for (uint32_t i = 0; i < kMaxSpins; ++i) {
      uint32_t ok;
      if constexpr (kCluster) {
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
            " selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
      } else {
        ok = mbar_try_wait(bar, parity);
      }
      if (ok) return;
      if (i > 1) __nanosleep(100);  // three of the roles wait most of the time
      if ((i & 255u) == 255u && *abort) return;
    }
    *abort = 1;
    report_status(status, (int)AK_ERR_TIMEOUT);
  }
};

__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// The compute warps' barrier; the warp is whole again first, after waits that its lanes left one by one.
__device__ __forceinline__ void compute_sync(int threads) {
  __syncwarp();
  asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
}

// A row's K entries as they lie in memory, entry 32 j + lane in slot j of the teacher's warp.
struct Entries {
  int64_t i[kSlots];
  float t[kSlots];
  __device__ __forceinline__ void load(const DistillArgs& a, int64_t r) {
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      const int k = 32 * j + (int)(threadIdx.x & 31);
      i[j] = k < a.K ? a.idx[r * a.K + k] : -1;
      t[j] = k < a.K ? a.tlp[r * a.K + k] : 0.f;
    }
  }
};

// The valid entries: token (or -1), log-probability and the student's logit.
struct Picked {
  int idx[kSlots];
  float t[kSlots], x[kSlots];
  bool any, bad;
  // logit(i): the student's logit of token i
  template <typename F>
  __device__ __forceinline__ void pick(const Entries& e, const DistillArgs& a, F logit) {
    any = bad = false;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      idx[j] = -1;
      t[j] = x[j] = -INFINITY;
      if (32 * j < a.K) {
        bad |= e.i[j] >= a.V;
        if (e.i[j] >= 0 && e.i[j] < a.V) {
          any = true;
          idx[j] = (int)e.i[j];
          t[j] = e.t[j];
          x[j] = logit(idx[j]);
        }
      }
    }
  }
};

constexpr int kTags = 2048;
__device__ __forceinline__ int mix_bits(int i) { return (int)(((uint32_t)i * 2654435761u) >> 21); }  // 11 bits

// Whether a token may come twice: two tables of who holds a place that its low and its mixed bits
// name.  Which of several entries holds it is not known (lanes of one store go in any order), but it
// is one of them: where the holder has the same token, that comes twice; where both places are held
// by other tokens it may, which costs a comparison of all with all.  A token that comes twice meets
// one of the two at an entry that does not hold its place.
__device__ __forceinline__ bool maybe_twice(const Picked& p, uint8_t (*tag)[kTags], int* s_idx) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < kSlots; ++j) {
    s_idx[32 * j + lane] = p.idx[j];
    if (p.idx[j] >= 0) {
      tag[0][p.idx[j] & (kTags - 1)] = (uint8_t)(32 * j + lane);
      tag[1][mix_bits(p.idx[j])] = (uint8_t)(32 * j + lane);
    }
  }
  __syncwarp();
  bool twice = false;
#pragma unroll
  for (int j = 0; j < kSlots; ++j) {
    if (p.idx[j] < 0) continue;
    const int a = tag[0][p.idx[j] & (kTags - 1)], b = tag[1][mix_bits(p.idx[j])], me = 32 * j + lane;
    twice |= (a != me && (b != me || s_idx[a] == p.idx[j])) || (b != me && s_idx[b] == p.idx[j]);
  }
  return __any_sync(0xffffffffu, twice);
}

// What a row's teacher says, on one warp.  s_idx and s_q are its scratch (twice only).
struct Teacher {
  float q[kSlots], logq[kSlots], y[kSlots], mass[kSlots];
  float rest, total;
  bool none, bad;
  template <int CAP>
  __device__ __forceinline__ void work(RowStats<CAP, false>& top, Picked& p, bool twice, const DistillArgs& a, int* s_idx,
                                       float* s_q);
};

template <int CAP>
__device__ __forceinline__ void Teacher::work(RowStats<CAP, false>& top, Picked& p, bool twice, const DistillArgs& a,
                                              int* s_idx, float* s_q) {
  const int lane = threadIdx.x & 31;
  const Squash sq = a.q;
  bad = __any_sync(0xffffffffu, p.bad);
  const bool any = __any_sync(0xffffffffu, p.any);
  // 1 - sum q would cancel in 32 bits: a teacher's 64 entries may leave 1e-5, of which their
  // exponentials' roundings are a tenth.  So the masses and their sum are formed in 64.
  if (a.tail) {
    double all = 0.0;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      q[j] = 0.f;
      logq[j] = p.t[j];
      if (32 * j < a.K) {
        const double e = p.idx[j] >= 0 ? exp((double)p.t[j]) : 0.0;
        q[j] = (float)e;
        all += e;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    none = !any;
    rest = (float)fmax(1.0 - all, 0.0);
    total = (float)all;
  } else {
    float tm = p.t[0], z = 0.f, qsum = 0.f;
#pragma unroll
    for (int j = 1; j < kSlots; ++j) tm = fmaxf(tm, p.t[j]);
    tm = redux_max(tm);
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      q[j] = 0.f;
      if (32 * j < a.K) z += q[j] = (p.idx[j] >= 0 && tm != -INFINITY) ? expf(p.t[j] - tm) : 0.f;
    }
    z = warp_sum(z);
    const float logz = logf(z);
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      q[j] = z == 0.f ? 0.f : q[j] / z;  // z: 0 without entries, NaN kept
      logq[j] = p.t[j] - tm - logz;
      qsum += q[j];
    }
    none = warp_sum(qsum) == 0.f;  // no teacher: loss 0, no gradient
    rest = 0.f;
    total = 1.f;
  }
  // entries of one token: its logit counts once, at the first of them; their masses add up
  uint32_t later = 0;
#pragma unroll
  for (int j = 0; j < kSlots; ++j) mass[j] = twice ? 0.f : q[j];
  if (twice) {
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      s_idx[32 * j + lane] = p.idx[j];
      s_q[32 * j + lane] = q[j];
    }
    __syncwarp();
    for (int m = 0; m < a.K; ++m) {
      const int im = s_idx[m];
      const float qm = s_q[m];
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        if (p.idx[j] == im) {
          mass[j] += qm;
          if (m < 32 * j + lane) later |= 1u << j;
        }
      }
    }
    __syncwarp();  // the scratch is free for the next row
  }
  top.init();
  uint32_t w[kSlots];
#pragma unroll
  for (int j = 0; j < kSlots; ++j) {
    y[j] = squash<CAP>(p.x[j], sq);
    w[j] = __float_as_uint((p.idx[j] < 0 || (later >> j & 1u)) ? -INFINITY : p.x[j]);
  }
  top.template add_words<float>(w, words_max<float>(w), sq);
  top.warp_merge(sq);
}

// A row's coefficients from the statistics of the rest and of the teacher's tokens.
template <int CAP>
__device__ __forceinline__ FinishRow coefficients(const RowStats<CAP, false>& st, const RowStats<CAP, false>& top,
                                                  float rest, float total, bool none, bool bad, const Squash& q) {
  RowStats<CAP, false> all = st;
  all.merge(top, q);
  all.center();
  FinishRow f;
  f.all = all.r;
  f.rest = st.r;
  f.logs = logf(all.s);
  f.empty = all.s == 0.f;  // every logit is -inf: no distribution, no gradient
  f.tail_loss = 0.f;
  // the scale of p in units of e: p = e 2^(rest's reference - the row's) / S
  const float below = ref_diff(st.r, all.r, q);
  // The rest is left out where the student has masked it: no logit outside the teacher's tokens
  // above -inf, or none within kMasked of the largest (a mask of the type's lowest value).
  const bool counts =
      rest > 0.f && st.s != 0.f && !none && !(squash<CAP>(st.m, q) - squash<CAP>(all.m, q) < -kMasked);
  f.mass = counts ? 1.f : total;
  f.c = (none || st.s == 0.f) ? 0.f : f.mass * ex2(below) / all.s;
  if (counts) {
    f.tail_loss = rest * (logf(rest) - (fmaf(below, kLn2, logf(st.s)) - f.logs));
    f.c -= rest / st.s;
  }
  if (bad) f.c = NAN;
  return f;
}

// One entry's term of the loss, added to it, and its token's gradient before the scale.
template <int CAP>
__device__ __forceinline__ float entry_grad(float& loss, int idx, float qk, float logq, float y, float mass,
                                            const FinishRow& f, bool none, bool bad, const Squash& q) {
  const float lpk = (f.empty || y == -INFINITY) ? -INFINITY : log_prob(y, f.all, f.logs, q);
  if (idx >= 0 && qk != 0.f) loss += qk * (logq - lpk);
  if (bad) return NAN;
  return (idx >= 0 && !none && !f.empty) ? fmaf(f.mass, expf(lpk), -mass) * squash_slope<CAP>(y, q) : 0.f;
}

template <typename T, int CAP, bool GRAD, int W>
__global__ void __launch_bounds__(32 * (W + kRoles), W == kWide ? 2 : 4)
distill_fwd_kernel(const T* __restrict__ logits, const DistillArgs a) {
  using Stats = RowStats<CAP, false>;
  constexpr int VEC = 16 / sizeof(T), kCompute = 32 * W;
  constexpr int U = W == kWide ? 4 : 2;  // 16-byte vectors that a compute thread works on at a time
  extern __shared__ __align__(128) unsigned char s_row[];  // this CTA's share of a row
  __shared__ __align__(8) uint64_t full;                   // the row has arrived
  __shared__ __align__(8) uint64_t left[kPieces];          // compute has left the piece
  __shared__ __align__(8) uint64_t ready[2], done[2];      // s_teacher, s_edge: written, read
  __shared__ __align__(8) uint64_t stored[2];              // compute is done with the row
  __shared__ __align__(8) uint64_t joined[2];
  __shared__ TeacherRow s_teacher[2];
  __shared__ FinishRow s_fin[2];
  __shared__ Stats s_warp[2][W];
  __shared__ __align__(16) float4 s_joined[2][kMaxCluster];  // statistics of the cluster's CTAs
  __shared__ float s_edge[2][2][32];                         // head and tail of the row
  __shared__ int s_idx[kMaxK];
  __shared__ float s_q[kMaxK];
  __shared__ uint8_t s_tag[2][kTags];
  __shared__ int s_abort;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cs = 1 << a.log_cs;
  const int64_t first = blockIdx.x >> a.log_cs, step = gridDim.x >> a.log_cs;
  const int rank = cs > 1 ? (int)row_cluster_rank() : 0;
  const Squash q = a.q;
  const Waits wait{a.status, &s_abort};
  if (tid == 0) {
    s_abort = 0;
    mbar_init(&full, 1);
    for (int c = 0; c < kPieces; ++c) mbar_init(&left[c], W);
    for (int b = 0; b < 2; ++b) {
      mbar_init(&ready[b], 1);
      mbar_init(&done[b], 1);
      mbar_init(&stored[b], W);
      mbar_init(&joined[b], cs);
    }
    mbar_fence_init();
  }
  __syncthreads();
  if (cs > 1) row_cluster_sync();  // the barriers of every CTA are initialised

  if (warp == 0) {
    // ---------------- loader
    if (lane == 0) {
      uint32_t ph = 0;
      for (int64_t r = first; r < a.rows; r += step, ph ^= 1u) {
        const bool live = a.mask == nullptr || a.mask[r] != 0;
        const Share<T> sh(logits + a.addr.off(r), a.V, rank, a.log_cs);
        const uint32_t bytes = live ? (uint32_t)(sh.n * sizeof(T)) : 0u;
        const char* src = reinterpret_cast<const char*>(sh.row + sh.body0);
        for (int c = 0; c < kPieces; ++c) {
          wait.operator()<false>(&left[c], ph ^ 1u);
          if (*wait.abort) break;
          if (c == 0) mbar_expect_tx(&full, bytes);
          // the generic accesses to the piece (the teacher's writes among them) before the copy
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          const uint32_t o = c * a.piece;
          if (o < bytes) bulk_g2s(s_row + o, src + o, min(a.piece, bytes - o), &full);
        }
        // last: until now the row is not complete, so nobody can leave a piece for the second time
        // before this warp has seen the first
        if (!*wait.abort) mbar_arrive(&full);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- teacher
    Entries entries;  // of the next row, on their way while this one is worked on
    if (first < a.rows) entries.load(a, first);
    int it = 0;
    for (int64_t r = first; r < a.rows; r += step, ++it) {
      const int b = it & 1;
      const bool live = a.mask == nullptr || a.mask[r] != 0;
      const Share<T> sh(logits + a.addr.off(r), a.V, rank, a.log_cs);
      TeacherRow& out = s_teacher[b];
      Picked p;
      Teacher te;
      Stats top;
      float e0 = 0.f, e1 = 0.f;
      const Entries now = entries;
      if (r + step < a.rows) entries.load(a, r + step);
      if (live) {  // all that needs no shared row
        if (lane < sh.head_here) e0 = to_f<T>(sh.row[lane]);
        if (lane < sh.tail_here) e1 = to_f<T>(sh.row[sh.tail0 + lane]);
        p.pick(now, a, [&](int i) { return to_f<T>(sh.row[i]); });
        const bool twice = maybe_twice(p, s_tag, s_idx);
        te.template work<CAP>(top, p, twice, a, s_idx, s_q);
      }
      wait.operator()<false>(&done[b], ((uint32_t)(it >> 1) & 1u) ^ 1u);
      wait.operator()<false>(&full, (uint32_t)it & 1u);
      if (live) {
        s_edge[b][0][lane] = e0;
        s_edge[b][1][lane] = e1;
        __syncwarp();
        T* buf = reinterpret_cast<T*>(s_row);
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
          if (32 * j >= a.K) break;
          const int k = 32 * j + lane, i = p.idx[j];
          out.idx[k] = i;
          out.q[k] = te.q[j];
          out.logq[k] = te.logq[j];
          out.y[k] = te.y[j];
          out.mass[k] = te.mass[j];
          if (i < 0) continue;
          if (i >= sh.body0 && i < sh.body0 + sh.n) buf[i - sh.body0] = from_f<T>(-INFINITY);
          else if (i < sh.head_here) s_edge[b][0][i] = -INFINITY;
          else if (i >= sh.tail0 && i - sh.tail0 < sh.tail_here) s_edge[b][1][i - sh.tail0] = -INFINITY;
        }
        if (lane == 0) {
          out.m = top.m;
          out.lim = top.lim;
          out.s = top.s;
          out.r = top.r;
          out.rest = te.rest;
          out.total = te.total;
          out.none = te.none;
          out.bad = te.bad;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ready[b]);
    }
  } else if (warp == 2) {
    // ---------------- finisher
    const float scale = GRAD ? grad_scale(a) : 1.f;
    int it = 0;
    for (int64_t r = first; r < a.rows; r += step, ++it) {
      const int b = it & 1;
      const bool live = a.mask == nullptr || a.mask[r] != 0;
      // of every row, masked or not, so that no phase of the two is passed over
      wait.operator()<false>(&ready[b], (uint32_t)(it >> 1) & 1u);
      wait.operator()<false>(&stored[b], (uint32_t)(it >> 1) & 1u);
      if (live) {
        const TeacherRow& tr = s_teacher[b];
        const FinishRow fin = s_fin[b];
        const Share<T> sh(logits + a.addr.off(r), a.V, rank, a.log_cs);
        T* grow = GRAD ? reinterpret_cast<T*>(a.grad) + r * a.V : nullptr;
        float loss = 0.f;
        for (int k = lane; k < a.K; k += 32) {
          const int i = tr.idx[k];
          const float gk = entry_grad<CAP>(loss, i, tr.q[k], tr.logq[k], tr.y[k], tr.mass[k], fin, tr.none, tr.bad, q);
          if constexpr (GRAD) {
            if (i >= 0 && sh.has(i)) grow[i] = from_f<T>(gk * scale);
          } else {
            if (rank == 0 && a.gk) a.gk[r * a.K + k] = gk;
          }
        }
        loss = warp_sum(loss) + fin.tail_loss;
        if (rank == 0 && lane == 0) {
          a.losses[r] = tr.bad ? NAN : loss;
          if (!GRAD && a.rest) a.rest[r] = make_float4(fin.rest.sh, fin.rest.k, fin.c, 0.f);
        }
      } else if (rank == 0) {
        if (lane == 0) {
          a.losses[r] = 0.f;
          if (!GRAD && a.rest) a.rest[r] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        if (!GRAD && a.gk)
          for (int k = lane; k < a.K; k += 32) a.gk[r * a.K + k] = 0.f;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&done[b]);
    }
  } else {
    // ---------------- compute
    const int cw = warp - kRoles, ct = tid - 32 * kRoles;
    const float scale = GRAD ? grad_scale(a) : 1.f;
    const uint4* s_vec = reinterpret_cast<const uint4*>(s_row);
    const int pv = (int)(a.piece / 16);
    int it = 0, nlive = 0;
    for (int64_t r = first; r < a.rows; r += step, ++it) {
      const int b = it & 1;
      const bool live = a.mask == nullptr || a.mask[r] != 0;
      const Share<T> sh(logits + a.addr.off(r), a.V, rank, a.log_cs);
      const int nv = sh.n / VEC;
      T* grow = GRAD ? reinterpret_cast<T*>(a.grad) + r * a.V : nullptr;
      const bool vec = GRAD && (reinterpret_cast<uintptr_t>(grow + sh.body0) & 15u) == 0;
      // hands back the pieces before this warp's next 16 bytes, v (of its first lane)
      int piece = 0;
      auto leave = [&](int v) {
        while (piece < kPieces && v >= (piece + 1) * pv) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&left[piece]);
          ++piece;
        }
      };
      Ref rest_ref{0.f, 0.f};
      float cg = 0.f;  // a masked row: zeros, whatever it holds
      wait.operator()<false>(&ready[b], (uint32_t)(it >> 1) & 1u);
      if (live) {
        wait.operator()<false>(&full, (uint32_t)it & 1u);  // complete: makes the copies visible to this thread
        const int lb = nlive & 1;
        const uint32_t lph = (uint32_t)(nlive >> 1) & 1u;
        ++nlive;
        Stats st;
        st.init();
        int v = ct;
        for (; v + (U - 1) * kCompute < nv; v += U * kCompute) {
          uint32_t w[4 * U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const uint4 f = s_vec[v + u * kCompute];
            w[4 * u] = f.x; w[4 * u + 1] = f.y; w[4 * u + 2] = f.z; w[4 * u + 3] = f.w;
          }
          st.template add_words<T>(w, words_max<T>(w), q);
          if constexpr (!GRAD) leave(v - lane + U * kCompute);
        }
        for (; v < nv; v += kCompute) {
          const uint4 f = s_vec[v];
          const uint32_t w[4] = {f.x, f.y, f.z, f.w};
          st.template add_words<T>(w, words_max<T>(w), q);
        }
        if constexpr (!GRAD) leave(kPieces * pv);
        const int e = cw * 32 + lane;  // head and tail: loose elements 0 .. 31, 32 .. 63
        for (int i = e; i < 64; i += kCompute)
          if ((i & 31) < (i < 32 ? sh.head_here : sh.tail_here)) st.add1(s_edge[b][i >> 5][i & 31], q);
        st.warp_merge(q);
        if (lane == 0) s_warp[lb][cw] = st;
        compute_sync(kCompute);
        st.init();
        if (lane < W) st = s_warp[lb][lane];
        st.warp_merge(q);
        if (cs > 1) {
          if (cw == 0 && lane < cs) {  // to every CTA of the cluster
            uint32_t at, bar;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(&s_joined[lb][rank])), "r"(lane));
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(smem_u32(&joined[lb])), "r"(lane));
            asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(st.m), "f"(st.r.sh),
                         "f"(st.r.k), "f"(st.s)
                         : "memory");
            asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
          }
          wait.operator()<true>(&joined[lb], lph);
          st.init();
          if (lane < cs) {  // every warp of every CTA joins them in the same way
            const float4 o = s_joined[lb][lane];
            st.m = o.x;
            st.r = Ref{o.y, o.z};
            st.s = o.w;
            if (o.w > 0.f) st.lim = 0.f;  // something was seen
          }
          st.warp_merge(q);
        }
        const TeacherRow& tr = s_teacher[b];
        Stats top;
        top.m = tr.m;
        top.lim = tr.lim;
        top.s = tr.s;
        top.r = tr.r;
        const FinishRow f = coefficients<CAP>(st, top, tr.rest, tr.total, tr.none, tr.bad, q);
        if (cw == 0 && lane == 0) s_fin[b] = f;
        rest_ref = f.rest;
        cg = f.c * scale;
      }
      if constexpr (GRAD) {
        T* gbody = grow + sh.body0;
        int u = ct;
        for (; u + (U - 1) * kCompute < nv; u += U * kCompute) {
          uint4 f[U];
#pragma unroll
          for (int j = 0; j < U; ++j) f[j] = s_vec[u + j * kCompute];
#pragma unroll
          for (int j = 0; j < U; ++j)
            store_grads<T, CAP>(gbody + (u + j * kCompute) * VEC, f[j], rest_ref, cg, q, vec);
          leave(u - lane + U * kCompute);
        }
        for (; u < nv; u += kCompute) store_grads<T, CAP>(gbody + u * VEC, s_vec[u], rest_ref, cg, q, vec);
        const int e = cw * 32 + lane;
        for (int i = e; i < 64; i += kCompute)
          if ((i & 31) < (i < 32 ? sh.head_here : sh.tail_here))
            grow[(i < 32 ? 0 : sh.tail0) + (i & 31)] =
                from_f<T>(rest_grad<CAP>(s_edge[b][i >> 5][i & 31], rest_ref, cg, q));
      }
      leave(kPieces * pv);
      // The finisher writes over what was stored here, and hands the row back to the teacher.  Row
      // it + 2 arrives on the same barrier: its ready[b] waits for done[b], so for the finisher.
      __syncwarp();
      if (lane == 0) mbar_arrive(&stored[b]);
    }
  }
  __syncthreads();
  if (s_abort) {  // a copy may still be on its way into this CTA's shared memory
    for (int i = 0; i < 1000; ++i) __nanosleep(1000);
  }
  if (cs > 1) row_cluster_sync();  // no more statistics from the other CTAs
}

// Short rows: one warp a row does it all, so that the steps of many rows overlap.
constexpr int kShortBytes = 8192;  // of a row at most
constexpr int kRowWarps = 8;

__host__ __device__ constexpr int warp_row_bytes(int bytes) { return (bytes + 15) / 16 * 16; }

template <typename T, int CAP, bool GRAD>
__global__ void __launch_bounds__(32 * kRowWarps, 3)
distill_warp_kernel(const T* __restrict__ logits, const DistillArgs a) {
  using Stats = RowStats<CAP, false>;
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ __align__(128) unsigned char s_rows[];
  __shared__ float s_edges[kRowWarps][2][32];
  __shared__ int s_idxs[kRowWarps][kMaxK];
  __shared__ float s_qs[kRowWarps][kMaxK];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t r = (int64_t)blockIdx.x * kRowWarps + warp;
  if (r >= a.rows) return;
  const Squash q = a.q;
  const Share<T> sh(logits + a.addr.off(r), a.V, 0, 0);
  const int nv = sh.n / VEC;
  T* buf = reinterpret_cast<T*>(s_rows + warp * warp_row_bytes(a.V * (int)sizeof(T)));
  float (*edge)[32] = s_edges[warp];
  T* grow = GRAD ? reinterpret_cast<T*>(a.grad) + r * a.V : nullptr;
  const bool vec = GRAD && (reinterpret_cast<uintptr_t>(grow + sh.body0) & 15u) == 0;
  const bool live = a.mask == nullptr || a.mask[r] != 0;
  const uint4* s_vec = reinterpret_cast<const uint4*>(buf);
  Ref rest_ref{0.f, 0.f};
  float cg = 0.f;
  if (live) {
    Entries e;
    e.load(a, r);
    for (int v = lane; v < nv; v += 32)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(buf + v * VEC)), "l"(sh.row + sh.body0 + v * VEC)
                   : "memory");
    if (lane < sh.head_here) edge[0][lane] = to_f<T>(sh.row[lane]);
    if (lane < sh.tail_here) edge[1][lane] = to_f<T>(sh.row[sh.tail0 + lane]);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    Picked p;
    p.pick(e, a, [&](int i) {
      return i < sh.body0 ? edge[0][i] : (i < sh.tail0 ? to_f<T>(buf[i - sh.body0]) : edge[1][i - sh.tail0]);
    });
    __syncwarp();
    // the row itself tells whether a token comes twice: each entry leaves its number there
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      const int i = p.idx[j];
      if (i < 0) continue;
      if (i < sh.body0) edge[0][i] = (float)(32 * j + lane);
      else if (i < sh.tail0) buf[i - sh.body0] = from_f<T>((float)(32 * j + lane));
      else edge[1][i - sh.tail0] = (float)(32 * j + lane);
    }
    __syncwarp();
    bool twice = false;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      const int i = p.idx[j];
      if (i < 0) continue;
      const float who = i < sh.body0 ? edge[0][i] : (i < sh.tail0 ? to_f<T>(buf[i - sh.body0]) : edge[1][i - sh.tail0]);
      twice |= who != (float)(32 * j + lane);
    }
    twice = __any_sync(0xffffffffu, twice);
    // ... and gives way to a logit without probability
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      const int i = p.idx[j];
      if (i < 0) continue;
      if (i < sh.body0) edge[0][i] = -INFINITY;
      else if (i < sh.tail0) buf[i - sh.body0] = from_f<T>(-INFINITY);
      else edge[1][i - sh.tail0] = -INFINITY;
    }
    __syncwarp();
    Teacher te;
    Stats top, st;
    te.template work<CAP>(top, p, twice, a, s_idxs[warp], s_qs[warp]);
    st.init();
    int v = lane;
    for (; v + 32 < nv; v += 64) {
      const uint4 f = s_vec[v], h = s_vec[v + 32];
      const uint32_t w[8] = {f.x, f.y, f.z, f.w, h.x, h.y, h.z, h.w};
      st.template add_words<T>(w, words_max<T>(w), q);
    }
    if (v < nv) {
      const uint4 f = s_vec[v];
      const uint32_t w[4] = {f.x, f.y, f.z, f.w};
      st.template add_words<T>(w, words_max<T>(w), q);
    }
    if (lane < sh.head_here) st.add1(edge[0][lane], q);
    if (lane < sh.tail_here) st.add1(edge[1][lane], q);
    st.warp_merge(q);
    const FinishRow f = coefficients<CAP>(st, top, te.rest, te.total, te.none, te.bad, q);
    const float scale = GRAD ? grad_scale(a) : 1.f;
    float loss = 0.f, gk[kSlots];
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      gk[j] = 0.f;
      if (32 * j < a.K)
        gk[j] = entry_grad<CAP>(loss, p.idx[j], te.q[j], te.logq[j], te.y[j], te.mass[j], f, te.none, te.bad, q);
    }
    loss = warp_sum(loss) + f.tail_loss;
    if (lane == 0) a.losses[r] = te.bad ? NAN : loss;
    if constexpr (GRAD) {
      rest_ref = f.rest;
      cg = f.c * scale;
      for (int u = lane; u < nv; u += 32) store_grads<T, CAP>(grow + sh.body0 + u * VEC, s_vec[u], rest_ref, cg, q, vec);
      if (lane < sh.head_here) grow[lane] = from_f<T>(rest_grad<CAP>(edge[0][lane], rest_ref, cg, q));
      if (lane < sh.tail_here) grow[sh.tail0 + lane] = from_f<T>(rest_grad<CAP>(edge[1][lane], rest_ref, cg, q));
      __syncwarp();  // the teacher's tokens over what was written for them
#pragma unroll
      for (int j = 0; j < kSlots; ++j)
        if (p.idx[j] >= 0) grow[p.idx[j]] = from_f<T>(gk[j] * scale);
    } else {
      if (lane == 0 && a.rest) a.rest[r] = make_float4(f.rest.sh, f.rest.k, f.c, 0.f);
      if (a.gk) {
#pragma unroll
        for (int j = 0; j < kSlots; ++j)
          if (32 * j + lane < a.K) a.gk[r * a.K + 32 * j + lane] = gk[j];
      }
    }
  } else {  // what the row holds is not looked at
    if (lane == 0) a.losses[r] = 0.f;
    if constexpr (GRAD) {
      const uint4 none = make_uint4(0u, 0u, 0u, 0u);
      for (int u = lane; u < nv; u += 32) store_grads<T, CAP>(grow + sh.body0 + u * VEC, none, rest_ref, 0.f, q, vec);
      if (lane < sh.head_here) grow[lane] = from_f<T>(0.f);
      if (lane < sh.tail_here) grow[sh.tail0 + lane] = from_f<T>(0.f);
    } else {
      if (lane == 0 && a.rest) a.rest[r] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (a.gk)
        for (int k = lane; k < a.K; k += 32) a.gk[r * a.K + k] = 0.f;
    }
  }
}

struct DistillBwdArgs {
  const float4* rest;
  const float* gk;
  const int64_t* idx;
  const uint8_t* mask;
  const float* inv_n;
  const float* g_loss;
  RowAddr addr;
  int64_t rows;
  float scale;
  int V, K, segs;
  Squash q;
};

constexpr int kBwdBatch = 4;
constexpr int kBwdGroups = 32 * kBwdBatch;  // groups of one warp

// The gradient from the forward's reference, c and K numbers a row: each warp takes one segment of a
// row, then writes those of the teacher's tokens that lie in it.
template <typename T, int CAP>
__global__ void __launch_bounds__(kThreads)
distill_bwd_kernel(T* __restrict__ grad, const T* __restrict__ logits, const DistillBwdArgs a) {
  const int tid = threadIdx.x & 31;
  const uint32_t at = blockIdx.x * (uint32_t)(kThreads / 32) + (threadIdx.x >> 5), r32 = at / (uint32_t)a.segs;
  const int64_t r = r32;
  const int seg = (int)(at - r32 * (uint32_t)a.segs);
  if (r >= a.rows) return;
  const Squash q = a.q;
  const T* row = logits + a.addr.off(r);
  T* grow = grad + r * a.V;
  const RowCut cut = cut_row(row, a.V);
  const bool vec = (reinterpret_cast<uintptr_t>(grow + cut.head) & 31u) == 0;
  const bool live = a.mask == nullptr || a.mask[r] != 0;
  const float scale = a.scale * (a.inv_n ? *a.inv_n : 1.f) * *a.g_loss;
  const float4 rc = a.rest[r];
  const Ref ref{rc.x, rc.y};
  const float c = live ? rc.z * scale : 0.f;  // c = 0: zeros, whatever the row holds
  const int gbeg = seg * kBwdGroups;
  const T* body = row + cut.head;
  T* gbody = grow + cut.head;
  RawGroup<T> raw[kBwdBatch];
#pragma unroll
  for (int u = 0; u < kBwdBatch; ++u) {
    const int g = gbeg + u * 32 + tid;
    if (g < cut.groups) raw[u] = load_group<T>(body + (int64_t)g * kGroup);
  }
#pragma unroll
  for (int u = 0; u < kBwdBatch; ++u) {
    const int g = gbeg + u * 32 + tid;
    if (g < cut.groups) {
      float x[kGroup];
#pragma unroll
      for (int h = 0; h < (int)sizeof(T) / 2; ++h)
        rest_grads<T, CAP>(x + h * 16 / ((int)sizeof(T) / 2), raw[u].r[h].w, ref, c, q);
      store_group<T>(gbody + (int64_t)g * kGroup, x, vec);
    }
  }
  const int tail0 = cut.head + cut.groups * kGroup;
  const bool first = seg == 0, last = seg == a.segs - 1;
  if (first && tid < cut.head) grow[tid] = from_f<T>(rest_grad<CAP>(to_f<T>(row[tid]), ref, c, q));
  if (last && tid < cut.tail)
    grow[tail0 + tid] = from_f<T>(rest_grad<CAP>(to_f<T>(row[tail0 + tid]), ref, c, q));
  if (!live) return;
  __syncwarp();
  for (int k = tid; k < a.K; k += 32) {
    const int64_t i = a.idx[r * a.K + k];
    const int64_t lo = first ? 0 : cut.head + (int64_t)gbeg * kGroup;
    const int64_t hi = last ? a.V : cut.head + (int64_t)(gbeg + kBwdGroups) * kGroup;
    if (i >= lo && i < hi && i < a.V) grow[i] = from_f<T>(a.gk[r * a.K + k] * scale);
  }
}

// inv_n[0] = 1 / max(1, rows whose mask is set).
__global__ void __launch_bounds__(1024)
distill_inv_rows(float* __restrict__ inv_n, const uint8_t* __restrict__ mask, int64_t rows) {
  __shared__ int s[32];
  int c = 0;
#pragma unroll 8
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

// loss[0] = mult / rows that count * sum of the rows' losses, in a fixed order; inv_n (with a mask)
// receives that quotient of 1.
__global__ void __launch_bounds__(1024)
distill_mean(float* __restrict__ loss, float* __restrict__ inv_n, const float* __restrict__ losses,
             const uint8_t* __restrict__ mask, float mult, int64_t rows) {
  __shared__ float s[32];
  __shared__ int n[32];
  float v = 0.f;
  int c = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < rows; i += blockDim.x) {
    v += losses[i];
    if (mask) c += mask[i] != 0;
  }
  v = warp_sum(v);
  c = __reduce_add_sync(0xffffffffu, c);
  if ((threadIdx.x & 31) == 0) { s[threadIdx.x >> 5] = v; n[threadIdx.x >> 5] = c; }
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = 0.f;
    int k = 0;
    for (int i = 0; i < 32; ++i) { t += s[i]; k += n[i]; }
    const float inv = mask ? 1.f / (float)max(k, 1) : 1.f;
    loss[0] = t * mult * inv;
    if (inv_n) inv_n[0] = inv;
  }
}

int64_t share_bytes(int64_t V, int cs, int es) { return ((V / kGroup + cs - 1) / cs) * kGroup * es; }

// log2 of the CTAs per row: as many as let two CTAs' shares fit an SM, and more while the rows leave
// SMs without a CTA and each CTA keeps half a group per thread.
int log_cluster_for(int64_t rows, int64_t V, int es) {
  int l = 0;
  while ((1 << l) < kMaxCluster && share_bytes(V, 1 << l, es) > kShareWanted) ++l;
  while ((1 << l) < kMaxCluster && (rows << (l + 1)) <= sm_count() && (V >> (l + 1)) >= 32 * kWide * kGroup / 2) ++l;
  return l;
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
  AK_REQUIRE(temperature >= kLowestTemperature && temperature < INFINITY, AK_ERR_ARG,
             "%s: temperature must be at least 2^-100 and finite", what);
  AK_REQUIRE(softcap == 0.f || (softcap >= kLowestSoftcap && softcap < INFINITY), AK_ERR_ARG,
             "%s: softcap must be 0, or at least 2^-100 and finite", what);
  AK_REQUIRE(rows == 0 || logits, AK_ERR_ARG, "%s: null pointer", what);
  AK_REQUIRE((reinterpret_cast<uintptr_t>(logits) % elem_size(dt)) == 0, AK_ERR_ARG,
             "%s: logits not aligned to their type", what);
  return AK_OK;
}

template <typename T, int W>
int launch_width(const T* logits, DistillArgs& a, int64_t share, cudaStream_t st) {
  auto kern = distill_fwd_kernel<T, kNoCap, true, W>;
  AK_DISPATCH_CAP(a.q, CAP, kern = a.grad ? distill_fwd_kernel<T, CAP, true, W> : distill_fwd_kernel<T, CAP, false, W>);
  const int cs = 1 << a.log_cs;
  a.piece = (uint32_t)((share + kPieces * 16 - 1) / (kPieces * 16) * 16);
  const size_t smem = (size_t)std::max<int64_t>(share, 16);
  // the most that this instance is launched with, not this call's: the attribute is the kernel's, and
  // another thread may launch it for a longer row between here and the launch
  AK_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   W == kWide ? kShareMost : kShareNarrow),
              "ak_distill_topk_fwd: shared memory");
  int64_t grid = a.rows * cs;
  if (grid > sm_count()) {  // fewer have an SM each
    int clusters = 0;
    AK_CUDA_TRY(resident_clusters(kern, 32 * (W + kRoles), cs, smem, &clusters), "ak_distill_topk_fwd: occupancy");
    grid = std::min<int64_t>(a.rows, clusters) * cs;
  }
  AK_CUDA_TRY(launch_rows(kern, grid, 32 * (W + kRoles), cs, smem, st, logits, (const DistillArgs&)a),
              "ak_distill_topk_fwd");
  return AK_OK;
}

template <typename T>
int launch_fwd(const T* logits, DistillArgs& a, cudaStream_t st) {
  if ((int64_t)a.V * (int64_t)sizeof(T) <= kShortBytes && a.rows >= 4 * sm_count()) {
    auto kern = distill_warp_kernel<T, kNoCap, true>;
    AK_DISPATCH_CAP(a.q, CAP, kern = a.grad ? distill_warp_kernel<T, CAP, true> : distill_warp_kernel<T, CAP, false>);
    const size_t smem = (size_t)kRowWarps * warp_row_bytes(a.V * (int)sizeof(T));
    AK_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowWarps * kShortBytes),
                "ak_distill_topk_fwd: shared memory");
    AK_CUDA_TRY(launch_rows(kern, (a.rows + kRowWarps - 1) / kRowWarps, 32 * kRowWarps, 1, smem, st, logits,
                            (const DistillArgs&)a),
                "ak_distill_topk_fwd");
    return AK_OK;
  }
  const int64_t share = share_bytes(a.V, 1 << a.log_cs, sizeof(T));
  return share <= kShareNarrow ? launch_width<T, kNarrow>(logits, a, share, st)
                               : launch_width<T, kWide>(logits, a, share, st);
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
  AK_REQUIRE(aligned16(rest_stats), AK_ERR_ARG, "ak_distill_topk_fwd: rest_stats not 16-byte aligned");
  AK_REQUIRE(!grad || (!rest_stats && !gk), AK_ERR_ARG,
             "ak_distill_topk_fwd: the gradient, or what its kernel needs, not both");
  AK_REQUIRE((reinterpret_cast<uintptr_t>(grad) % elem_size(dt)) == 0, AK_ERR_ARG,
             "ak_distill_topk_fwd: grad not aligned to its type");
  cudaStream_t st = (cudaStream_t)stream;
  if (rows > 0) {
    // few rows: each warp counts them, which costs less than a launch
    const bool count = mask && grad && rows > kCountRows;
    if (count) {
      distill_inv_rows<<<1, 1024, 0, st>>>(inv_n, mask, rows);
      AK_CHECK_LAUNCH("ak_distill_topk_fwd");
    }
    DistillArgs a{};
    a.losses = losses; a.grad = grad;
    a.rest = reinterpret_cast<float4*>(rest_stats);
    a.gk = gk; a.idx = teacher_idx; a.tlp = teacher_lp; a.mask = mask;
    a.inv_n = count ? inv_n : nullptr;
    a.addr = RowAddr{inner, stride_outer, stride_inner};
    a.scale = mask ? temperature : temperature / (float)rows;
    a.rows = rows; a.V = (int)V; a.K = (int)K; a.log_cs = log_cluster_for(rows, V, elem_size(dt)); a.tail = tail != 0;
    a.q = make_squash(temperature, softcap);
    a.status = status;
    AK_DISPATCH_DTYPE(dt, T, rc = launch_fwd<T>((const T*)logits, a, st));
    if (rc) return rc;
  }
  distill_mean<<<1, 1024, 0, st>>>(loss, rows > 0 ? inv_n : nullptr, losses, mask,
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
  AK_REQUIRE(grad && teacher_idx && rest_stats && aligned16(rest_stats) && gk && g_loss && (!mask || inv_n), AK_ERR_ARG,
             "ak_distill_topk_bwd: null pointer, or rest_stats not 16-byte aligned");
  AK_REQUIRE((reinterpret_cast<uintptr_t>(grad) % elem_size(dt)) == 0, AK_ERR_ARG,
             "ak_distill_topk_bwd: grad not aligned to its type");
  DistillBwdArgs a{};
  a.rest = reinterpret_cast<const float4*>(rest_stats);
  a.gk = gk; a.idx = teacher_idx; a.mask = mask; a.inv_n = mask ? inv_n : nullptr; a.g_loss = g_loss;
  a.addr = RowAddr{inner, stride_outer, stride_inner};
  a.scale = mask ? temperature : temperature / (float)rows;
  a.rows = rows; a.V = (int)V; a.K = (int)K;
  a.segs = (int)std::max<int64_t>(1, (V / kGroup + kBwdGroups - 1) / kBwdGroups);
  a.q = make_squash(temperature, softcap);
  AK_REQUIRE(rows * a.segs < (1LL << 32) - 8, AK_ERR_SHAPE, "ak_distill_topk_bwd: too many rows");
  AK_DISPATCH_DTYPE(dt, T, {
    auto kern = distill_bwd_kernel<T, kNoCap>;
    AK_DISPATCH_CAP(a.q, CAP, kern = distill_bwd_kernel<T, CAP>);
    kern<<<(unsigned)((rows * a.segs + kThreads / 32 - 1) / (kThreads / 32)), kThreads, 0, (cudaStream_t)stream>>>(
        (T*)grad, (const T*)logits, a);
  });
  AK_CHECK_LAUNCH("ak_distill_topk_bwd");
  return AK_OK;
}
