// Log-probabilities of given tokens from logit rows, with each row's entropy and its most
// likely alternatives; sm_100a.
//
//   y = softcap(x) / T,  lse = log sum exp y,  logprob = y_t - lse
//   H = lse - sum p y,   p = exp(y - lse)
//   dx_i = [ g_lp (1[i = t] - p_i) - g_H p_i (log p_i + H) ] dy_i/dx_i
//
// Forward: one pass over the row with the running maximum and the two sums of RowStats, by one
// CTA per row, or by a cluster of CTAs whose shares are joined through distributed shared memory
// where there are few rows.
//
// Alternatives, without a second pass over the row: a thread writes the maximum of each group of
// 16 adjacent elements it reads to shared memory.  Order groups by (maximum, lowest position) and
// elements by (value, lowest position): an element outside the first k groups is preceded by the k
// largest elements of those groups, so the k groups hold the k best elements, ties included.  Only
// they are read again, from L2.
//
// What bounds it and what it measured (GPU time; 6551 GB/s is the measured copy rate):
//   8192 x 50304 bf16, entropy   129-133 us = 6.2-6.4 TB/s: HBM; one exponential an element keeps the special
//                                units at 2/3
//   4096 x 32768 fp16, entropy   48.2 us = 5.6 TB/s
//   8192 x 50304 bf16, top 64    163 us: the selection costs 35 us (its barriers and a few hundred
//                                instructions a warp; ranking by counting among the ~75 candidates)
//   64 x 131072 fp32, softcap    17 us, floor 5.1 us (18.4 with the softcap by special units alone)
//   1 x 50304 bf16, top 20       9.8 us: latency of one cluster (load, two reductions, selection, join)
//   backward 8192 x 50304 bf16   238 us = 6.9 TB/s: HBM
#include "logit_rows.cuh"

#include <algorithm>

namespace ak {
namespace {

constexpr int kThreads = 256;       // of a CTA; kFew where a row has no work for that many
constexpr int kFew = 128;
constexpr int kMaxTop = 128;         // alternatives
constexpr int kMaxCluster = 8;       // the portable cluster size
constexpr int kMaxGroupMax = 8194;  // group maxima of one CTA's share (32 KB), head and tail included
constexpr int kCandGroups = 512;     // candidates of the short way through the selection
constexpr int kCandElems = 768;
constexpr int kBisect = 16;          // steps towards the bound at most

// Unsigned keys in the order of the values: -0 and +0 are equal, NaN is below every number, 0 is
// no value at all.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 1u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b >> 31) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k <= 1u) return __uint_as_float(0x7fffffffu);
  return __uint_as_float((k >> 31) ? (k & 0x7fffffffu) : ~k);
}

// One CTA's share of a row as the selection sees it: local group 0 is the row's head (first CTA
// only), 1 .. n are whole groups, n + 1 is the tail (last CTA only).
template <typename T>
struct Share {
  const T* row;
  int head, tail, g0, n, body_end;  // body_end: first element of the tail
  int head_here, tail_here;
  __device__ __forceinline__ int start(int j) const {
    return j == 0 ? 0 : (j <= n ? head + (g0 + j - 1) * kGroup : body_end);
  }
  __device__ __forceinline__ int size(int j) const { return j == 0 ? head_here : (j <= n ? kGroup : tail_here); }
  __device__ __forceinline__ int elems() const { return head_here + n * kGroup + tail_here; }
};

template <int NT>
struct SelectScratch {
  union {
    struct {
      uint32_t groups[kCandGroups];
      uint64_t elems[kCandElems];
    } cand;
    uint32_t keys[kMaxTop * kGroup];  // the exact way: elements of the chosen groups
    struct {                          // clusters: the lists of all CTAs, and places in the joined one
      uint64_t lists[kMaxTop * kMaxCluster];
      int place[kMaxTop];
    };
  };
  uint32_t chosen[kMaxTop];  // groups, then elements, in order of position
  uint32_t warp_n[2][NT / 32];
  uint32_t ngroups, nelems;
};

// The first k of the n keys key(0 .. n - 1) in the order (key descending, position ascending):
// their positions, ascending, in out.  Needs n >= k.  A binary search over the key's bits for the k-th largest,
// then everything above it and the first of those equal to it.
template <int NT, typename Key>
__device__ void select_exact(Key key_at, int n, int k, uint32_t* out, SelectScratch<NT>& sc) {
  constexpr int kWarps = NT / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t t = 0;
  int above = 0;  // number of keys > t, known at the end
  for (int bit = 31; bit >= -1; --bit) {
    const uint32_t probe = bit >= 0 ? (t | (1u << bit)) : t;
    int c = 0;
    for (int i = tid; i < n; i += NT) c += bit >= 0 ? (key_at(i) >= probe) : (key_at(i) > probe);
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0) sc.warp_n[0][warp] = (uint32_t)c;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) total += (int)sc.warp_n[0][i];
    __syncthreads();
    if (bit < 0) above = total;
    else if (total >= k) t = probe;
  }
  const int equal_wanted = k - above;
  int taken = 0, equal_seen = 0;
  for (int i0 = 0; i0 < n; i0 += NT) {
    const int i = i0 + tid;
    const uint32_t key = i < n ? key_at(i) : 0u;
    const bool eq = i < n && key == t;
    const uint32_t eq_ballot = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) sc.warp_n[0][warp] = __popc(eq_ballot);
    __syncthreads();
    int eq_before = equal_seen, eq_total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) eq_before += (int)sc.warp_n[0][w];
      eq_total += (int)sc.warp_n[0][w];
    }
    eq_before += __popc(eq_ballot & ((1u << lane) - 1u));
    const bool take = i < n && (key > t || (eq && eq_before < equal_wanted));
    const uint32_t ballot = __ballot_sync(0xffffffffu, take);
    if (lane == 0) sc.warp_n[1][warp] = __popc(ballot);
    __syncthreads();
    int before = taken, total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += (int)sc.warp_n[1][w];
      total += (int)sc.warp_n[1][w];
    }
    if (take) out[before + __popc(ballot & ((1u << lane) - 1u))] = (uint32_t)i;
    taken += total;
    equal_seen += eq_total;
    __syncthreads();
  }
}

// Entry of the sorted list: larger is better.
__device__ __forceinline__ uint64_t entry(uint32_t key, int index) {
  return ((uint64_t)key << 32) | (uint32_t)(~(uint32_t)index);
}

// The k best elements of the share, best first, in top[0 .. k).  gmax holds the n + 2 group maxima
// (a barrier has passed since they were written), mine the largest element this thread has seen.
template <typename T, int NT>
__device__ void select_top(uint64_t* top, const Share<T>& sh, const float* gmax, float mine, int k,
                           SelectScratch<NT>& sc) {
  constexpr int kWarps = NT / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // A lower bound of the k-th best element: a key that at least k threads' largest elements reach,
  // found by bisection between the smallest and the largest of those; it ends early where not many
  // more than k do.
  const uint32_t key = order_key(mine);
  uint32_t lo = __reduce_min_sync(0xffffffffu, key), hi = __reduce_max_sync(0xffffffffu, key);
  if (lane == 0) { sc.warp_n[0][warp] = lo; sc.warp_n[1][warp] = hi; }
  if (tid == 0) { sc.ngroups = 0; sc.nelems = 0; }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    lo = min(lo, sc.warp_n[0][w]);
    hi = max(hi, sc.warp_n[1][w]);
  }
  for (int i = 0; i < kBisect && lo < hi; ++i) {
    const uint32_t probe = lo + (hi - lo + 1) / 2;
    const int c = __syncthreads_count(key >= probe);
    if (c < k) {
      hi = probe - 1;
    } else {
      lo = probe;
      if (c <= k + k / 8 + 2) break;
    }
  }
  // -inf is also what a thread has that saw no number: then every element is a candidate
  const bool all = lo <= order_key(-INFINITY);
  const float bound = key_value(lo);
  // candidates: the groups that reach the bound (four maxima at a time), then their elements
  const int ng = sh.n + 2;
  for (int i = 4 * tid; i < ng; i += 4 * NT) {
    const float4 m = *reinterpret_cast<const float4*>(gmax + i);  // past the end: padding of the buffer
    const bool c0 = m.x >= bound || all, c1 = (m.y >= bound || all) && i + 1 < ng,
               c2 = (m.z >= bound || all) && i + 2 < ng, c3 = (m.w >= bound || all) && i + 3 < ng;
    if (c0 || c1 || c2 || c3) {
      uint32_t at = atomicAdd(&sc.ngroups, (uint32_t)(c0 + c1 + c2 + c3));
      if (at + 4 <= kCandGroups) {
        if (c0) sc.cand.groups[at++] = (uint32_t)i;
        if (c1) sc.cand.groups[at++] = (uint32_t)i + 1;
        if (c2) sc.cand.groups[at++] = (uint32_t)i + 2;
        if (c3) sc.cand.groups[at] = (uint32_t)i + 3;
      }
    }
  }
  __syncthreads();
  const uint32_t ncg = sc.ngroups;
  bool exact = ncg > kCandGroups - 4;
  if (!exact) {
    for (int i = tid; i < (int)ncg; i += NT) {
      const int g = (int)sc.cand.groups[i], first = sh.start(g), size = sh.size(g);
      float x[kGroup];
      if (g >= 1 && g <= sh.n) {
        unpack_group<T>(x, load_group<T>(sh.row + first));
      } else {
#pragma unroll
        for (int e = 0; e < kGroup; ++e) x[e] = e < size ? to_f<T>(sh.row[first + e]) : 0.f;
      }
      uint32_t take = 0;
#pragma unroll
      for (int e = 0; e < kGroup; ++e) take |= (x[e] >= bound || all) ? 1u << e : 0u;
      take &= (1u << size) - 1u;
      uint32_t at = atomicAdd(&sc.nelems, (uint32_t)__popc(take));
      if (at + kGroup <= kCandElems) {
#pragma unroll
        for (int e = 0; e < kGroup; ++e)
          if (take >> e & 1u) sc.cand.elems[at++] = entry(order_key(x[e]), first + e);
      }
    }
    __syncthreads();
    exact = sc.nelems > kCandElems - kGroup;
  }
  if (!exact) {
    // the position of each candidate is the number of better ones
    const int ne = (int)sc.nelems;
    for (int i = tid; i < ne; i += NT) {
      const uint64_t e = sc.cand.elems[i];
      int rank = 0, o = 0;
      for (; o + 4 <= ne; o += 4) {
        const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(sc.cand.elems + o);
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(sc.cand.elems + o + 2);
        rank += (a.x > e) + (a.y > e) + (b.x > e) + (b.y > e);
      }
      for (; o < ne; ++o) rank += sc.cand.elems[o] > e;
      if (rank < k) top[rank] = e;
    }
    __syncthreads();
    return;
  }
  // Many equal values (masked or constant rows): choose the k groups, then the k elements, exactly.
  __syncthreads();
  const int kg = min(k, ng);
  select_exact<NT>([&](int i) { return sh.size(i) ? order_key(gmax[i]) : 0u; }, ng, kg, sc.chosen, sc);
  for (int i = tid; i < kg * kGroup; i += NT) {
    const int g = (int)sc.chosen[i / kGroup], e = i % kGroup;
    sc.keys[i] = e < sh.size(g) ? order_key(to_f<T>(sh.row[sh.start(g) + e])) : 0u;
  }
  __syncthreads();
  // positions in the list of chosen groups ascend with the position in the row
  __shared__ uint32_t groups[kMaxTop];
  for (int i = tid; i < kg; i += NT) groups[i] = sc.chosen[i];
  __syncthreads();
  select_exact<NT>([&](int i) { return sc.keys[i]; }, kg * kGroup, k, sc.chosen, sc);
  uint64_t e = 0;
  if (tid < k) {
    const int at = (int)sc.chosen[tid], g = (int)groups[at / kGroup];
    e = entry(sc.keys[at], sh.start(g) + at % kGroup);
  }
  __syncthreads();
  uint64_t* list = sc.cand.elems;  // the keys have been read
  if (tid < k) list[tid] = e;
  __syncthreads();
  if (tid < k) {
    int rank = 0;
    for (int o = 0; o < k; ++o) rank += list[o] > e;
    top[rank] = e;
  }
  __syncthreads();
}

struct FwdArgs {
  float* logprobs;      // nullable
  float* entropy;       // nullable
  float* lse;           // nullable
  float4* stats;        // nullable: (reference, log S, entropy) for the backward
  float* top_lp;        // nullable with top_idx
  int64_t* top_idx;
  const int64_t* targets;  // nullable
  RowAddr addr;
  int64_t ignore_index;
  int V, k, cs;
  Squash q;
};

constexpr int kBatch = 2;  // groups of a thread in flight
// CTAs on an SM: 16-bit groups take 32 registers a thread with two in flight, which hides the
// row's start and end behind seven other rows; fp32 groups are twice as large
template <typename T, int CAP, int NT>
constexpr int resident() { return (sizeof(T) == 4 ? 4 : (CAP ? 5 : 8)) * (kThreads / NT); }

// A row's results from its joined and centred statistics.
template <typename T, int CAP, bool ENT>
__device__ __forceinline__ void write_row(const FwdArgs& a, int64_t r, const T* row, const RowStats<CAP, ENT>& st,
                                          float logs) {
  const int64_t t = a.targets ? a.targets[r] : 0;
  const bool ignored = a.targets && t == a.ignore_index;
  if (a.logprobs) {
    float lp = 0.f;
    if (!ignored) {
      if (t < 0 || t >= a.V) lp = NAN;  // not a token
      else if (st.s == 0.f) lp = -INFINITY;
      else lp = log_prob(squash<CAP>(to_f<T>(row[t]), a.q), st.r, logs, a.q);
    }
    a.logprobs[r] = lp;
  }
  float H = 0.f;
  if constexpr (ENT) {
    if (!ignored && st.s != 0.f) H = fmaf(-kLn2, st.w / st.s, logs);
    a.entropy[r] = H;
  }
  if (a.lse) a.lse[r] = ref_lse(st.r, logs, a.q);
  if (a.stats) a.stats[r] = make_float4(st.r.sh, st.r.k, logs, H);
}

template <typename T, int CAP, bool ENT, bool TOP, int NT>
__global__ void __launch_bounds__(NT, (resident<T, CAP, NT>()))
token_logprobs_fwd_kernel(const T* __restrict__ logits, const FwdArgs a) {
  constexpr int kWarps = NT / 32;
  using Stats = RowStats<CAP, ENT>;
  extern __shared__ __align__(16) float gmax[];  // TOP: group maxima
  __shared__ Stats s_warp[kWarps];
  __shared__ Stats s_cta;
  __shared__ float s_share[6];         // this CTA's statistics, read by the others of the cluster
  __shared__ uint64_t s_top[TOP ? kMaxTop : 1];
  __shared__ __align__(16) unsigned char s_scratch[TOP ? sizeof(SelectScratch<NT>) : 8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cs = a.cs;
  const int64_t r = cs > 1 ? blockIdx.x / cs : blockIdx.x;
  const int rank = cs > 1 ? (int)row_cluster_rank() : 0;
  const Squash q = a.q;
  const T* row = logits + a.addr.off(r);
  const RowCut cut = cut_row(row, a.V);
  Share<T> sh;
  sh.row = row;
  sh.head = cut.head;
  sh.tail = cut.tail;
  sh.g0 = (int)((int64_t)cut.groups * rank / cs);
  sh.n = (int)((int64_t)cut.groups * (rank + 1) / cs) - sh.g0;
  sh.body_end = cut.head + cut.groups * kGroup;
  sh.head_here = rank == 0 ? cut.head : 0;
  sh.tail_here = rank == cs - 1 ? cut.tail : 0;

  Stats st;
  st.init();
  const T* body = row + cut.head + (int64_t)sh.g0 * kGroup;
  auto group = [&](const RawGroup<T>& raw, int g) {
    float lm = words_max<T>(raw.r[0].w);
    if constexpr (sizeof(T) == 4) lm = fmaxf(lm, words_max<T>(raw.r[1].w));
    if constexpr (TOP) gmax[1 + g] = lm;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) st.template add_words<T>(raw.r[i].w, lm, q);
  };
  int g = tid;
  for (; g + (kBatch - 1) * NT < sh.n; g += kBatch * NT) {
    RawGroup<T> raw[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) raw[u] = load_group<T>(body + (int64_t)(g + u * NT) * kGroup);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) group(raw[u], g + u * NT);
  }
  for (; g < sh.n; g += NT) group(load_group<T>(body + (int64_t)g * kGroup), g);
  // head and tail: one element a lane of the first and the last warp
  if (warp == 0 || warp == kWarps - 1) {
    const bool first = warp == 0;
    const int n = first ? sh.head_here : sh.tail_here;
    uint32_t key = 0;
    if (lane < n) {
      const float x = to_f<T>(row[(first ? 0 : sh.body_end) + lane]);
      st.add1(x, q);
      key = order_key(x);
    }
    if constexpr (TOP) {
      const uint32_t best = __reduce_max_sync(0xffffffffu, key);
      if (lane == 0) gmax[first ? 0 : sh.n + 1] = key_value(best);
    }
  }
  const float mine = st.m;
  st.warp_merge(q);
  if (lane == 0) s_warp[warp] = st;
  __syncthreads();
  if (warp == 0) {
    st.init();
    if (lane < kWarps) st = s_warp[lane];
    st.warp_merge(q);
    if (lane == 0) s_cta = st;
  }
  if (TOP || cs > 1) {
    __syncthreads();
    st = s_cta;
  }
  const int kl = TOP ? min(a.k, sh.elems()) : 0;
  if constexpr (TOP)
    if (kl > 0) select_top<T>(s_top, sh, gmax, mine, kl, *reinterpret_cast<SelectScratch<NT>*>(s_scratch));
  if (cs > 1) {
    if (tid == 0) {
      s_share[0] = st.lim;
      s_share[1] = st.s;
      s_share[2] = ENT ? st.w : 0.f;
      s_share[3] = __int_as_float(kl);
      s_share[4] = st.r.sh;
      s_share[5] = st.r.k;
    }
    row_cluster_sync();
    st.init();
    if (lane < cs) {  // every warp of every CTA joins them in the same way
      st.lim = __uint_as_float(ld_cluster_u32(&s_share[0], lane));
      st.s = __uint_as_float(ld_cluster_u32(&s_share[1], lane));
      st.w = __uint_as_float(ld_cluster_u32(&s_share[2], lane));
      st.r.sh = __uint_as_float(ld_cluster_u32(&s_share[4], lane));
      st.r.k = __uint_as_float(ld_cluster_u32(&s_share[5], lane));
    }
    st.warp_merge(q);
  }
  st.center();
  // S = 0: every logit is -inf and the row has no distribution: log-probabilities -inf, entropy 0
  const float logs = logf(st.s);
  if constexpr (TOP) {
    // An entry's position in the row's list: its own in this CTA's list and the number of better
    // entries in each other list, all sorted.  The other lists are copied here first.
    SelectScratch<NT>& sc = *reinterpret_cast<SelectScratch<NT>*>(s_scratch);
    if (cs > 1) {
      __syncthreads();  // the selection is done with its scratch
      for (int i = tid; i < cs * a.k; i += NT) {  // 0 from the end of a shorter list on
        const int c = i / a.k, o = i - c * a.k;
        sc.lists[i] = o < (int)ld_cluster_u32(&s_share[3], c) ? ld_cluster_u64(&s_top[o], c) : 0ull;
      }
      for (int i = tid; i < kl; i += NT) sc.place[i] = i;
      __syncthreads();
      for (int i = tid; i < cs * kl; i += NT) {
        const int c = i / kl, o = i - c * kl;
        if (c == rank) continue;
        const uint64_t e = s_top[o];
        int lo = 0, hi = a.k;
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (sc.lists[c * a.k + mid] > e) lo = mid + 1;
          else hi = mid;
        }
        if (lo) atomicAdd(&sc.place[o], lo);
      }
      __syncthreads();
    }
    for (int i = tid; i < kl; i += NT) {
      const uint64_t e = s_top[i];
      const int pos = cs > 1 ? sc.place[i] : i;
      if (pos < a.k) {
        const float x = key_value((uint32_t)(e >> 32));
        a.top_idx[r * a.k + pos] = (int64_t)(uint32_t)~(uint32_t)e;
        a.top_lp[r * a.k + pos] = st.s == 0.f ? -INFINITY : log_prob(squash<CAP>(x, q), st.r, logs, q);
      }
    }
  }
  if (rank == 0 && tid == 0) write_row<T, CAP, ENT>(a, r, row, st, logs);
  if (cs > 1) {  // the other CTAs have read this one's shared memory
    row_cluster_arrive_relaxed();
    row_cluster_wait();
  }
}

// Many short rows: one warp a row, nothing shared.
template <typename T, int CAP, bool ENT>
__global__ void __launch_bounds__(kThreads)
token_logprobs_warp_kernel(const T* __restrict__ logits, const FwdArgs a, int64_t rows) {
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (r >= rows) return;
  const Squash q = a.q;
  const T* row = logits + a.addr.off(r);
  const RowCut cut = cut_row(row, a.V);
  RowStats<CAP, ENT> st;
  st.init();
  const T* body = row + cut.head;
  auto group = [&](const RawGroup<T>& raw) {
    float lm = words_max<T>(raw.r[0].w);
    if constexpr (sizeof(T) == 4) lm = fmaxf(lm, words_max<T>(raw.r[1].w));
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) st.template add_words<T>(raw.r[i].w, lm, q);
  };
  int g = lane;
  for (; g + (kBatch - 1) * 32 < cut.groups; g += kBatch * 32) {
    RawGroup<T> raw[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) raw[u] = load_group<T>(body + (int64_t)(g + u * 32) * kGroup);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) group(raw[u]);
  }
  for (; g < cut.groups; g += 32) group(load_group<T>(body + (int64_t)g * kGroup));
  if (lane < cut.head) st.add1(to_f<T>(row[lane]), q);
  if (lane < cut.tail) st.add1(to_f<T>(row[cut.head + cut.groups * kGroup + lane]), q);
  st.warp_merge(q);
  st.center();
  const float logs = logf(st.s);
  if (lane == 0) write_row<T, CAP, ENT>(a, r, row, st, logs);
}

struct BwdArgs {
  const float4* stats;
  const float* g_lp;       // nullable
  const float* g_ent;      // nullable
  const int64_t* targets;  // nullable
  RowAddr addr;
  int64_t rows, ignore_index;
  int V, segs;
  Squash q;
};

constexpr int kBwdBatch = 4;
constexpr int kBwdGroups = 32 * kBwdBatch;  // groups of one warp

// Elementwise from the forward's numbers: each warp takes one segment of a row.
template <typename T, int CAP, bool ENT>
__global__ void __launch_bounds__(kThreads)
token_logprobs_bwd_kernel(T* __restrict__ grad, const T* __restrict__ logits, const BwdArgs a) {
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
  const int64_t t = a.targets ? a.targets[r] : -1;
  const float4 st = a.stats[r];
  const Ref ref{st.x, st.y};
  const float logs = st.z, H = st.w;
  // rows without a gradient: ignored ones, and those whose every logit is -inf (S = 0)
  const bool none = (a.targets && t == a.ignore_index) || logs == -INFINITY;
  float gl = (a.targets && a.g_lp) ? a.g_lp[r] : 0.f;
  if (a.targets && !none && (t < 0 || t >= a.V)) gl = NAN;
  const float ge = ENT ? a.g_ent[r] : 0.f;
  // e = 2^d, p = e / S, log p = d ln 2 - log S:
  // dx = e (c0 + c1 d) (+ gl / T at the target), times the softcap's slope
  const float f = q.inv_t * expf(-logs);
  const float c0 = (ge * (logs - H) - gl) * f, c1 = -ge * kLn2 * f, ct = gl * q.inv_t;
  const int ti = (a.targets && t >= 0 && t < a.V) ? (int)t : -1;

  auto one_at = [&](float y, int i) {  // y: squashed
    const float d = exponent(y, ref, q);
    float o = ex2(d);
    o *= ENT ? fmaf(c1, fmaxf(d, kNoTerm), c0) : c0;
    if (i == ti) o += ct;
    return o * squash_slope<CAP>(y, q);
  };
  auto one = [&](float x, int i) { return one_at(squash<CAP>(x, q), i); };
  [[maybe_unused]] uint32_t floor = 0;
  bool quick = ref.sh == 0.f;
  if constexpr (ENT && !CAP) {
    float f;
    quick = raise_to<T>(f, ref, q);
    floor = floor_word<T>(f);
  }
  const float2 kl = both(q.kl), nk = both(-ref.k), c02 = both(c0), c12 = both(c1);

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
      if (none) {
#pragma unroll
        for (int i = 0; i < kGroup; ++i) x[i] = 0.f;
      } else if (quick) {
        constexpr int W = 8, P = W * elems_per_word<T>() / 2;  // pairs of one 32-byte piece
#pragma unroll
        for (int h = 0; h < (int)sizeof(T) / 2; ++h) {
          uint32_t w[W];
#pragma unroll
          for (int i = 0; i < W; ++i)
            w[i] = ENT && !CAP ? word_max_nan(raw[u].r[h].w[i], floor, (const T*)nullptr) : raw[u].r[h].w[i];
          if (CAP && !all_near<T>(w, words_max<T>(w), q)) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
              const float2 v = word_pair<T>(w, i);
              x[h * 2 * P + 2 * i] = one_at(squash_far<CAP>(v.x, q), -2);  // the target's part follows
              x[h * 2 * P + 2 * i + 1] = one_at(squash_far<CAP>(v.y, q), -2);
            }
            continue;
          }
#pragma unroll
          for (int i = 0; i < P; ++i) {
            float2 y = word_pair<T>(w, i);
            if constexpr (CAP) y = squash_near(y, q);
            float2 d = __ffma2_rn(y, kl, nk);
            if constexpr (CAP && ENT) d = make_float2(fmaxf(d.x, kNoTerm), fmaxf(d.y, kNoTerm));
            float2 o = __fmul2_rn(make_float2(ex2(d.x), ex2(d.y)), ENT ? __ffma2_rn(c12, d, c02) : c02);
            if constexpr (CAP) o = __fmul2_rn(o, squash_slope_near(y, q));
            x[h * 2 * P + 2 * i] = o.x;
            x[h * 2 * P + 2 * i + 1] = o.y;
          }
        }
        const int ta = ti - (cut.head + g * kGroup);
        if ((unsigned)ta < (unsigned)kGroup) {
          const float add = CAP ? ct * squash_slope<CAP>(squash<CAP>(to_f<T>(row[ti]), q), q) : ct;
#pragma unroll
          for (int i = 0; i < kGroup; ++i)
            if (i == ta) x[i] += add;
        }
      } else {
        unpack_group<T>(x, raw[u]);
#pragma unroll
        for (int i = 0; i < kGroup; ++i) x[i] = one(x[i], cut.head + g * kGroup + i);
      }
      store_group<T>(gbody + (int64_t)g * kGroup, x, vec);
    }
  }
  if (seg == 0 && tid < cut.head) grow[tid] = from_f<T>(none ? 0.f : one(to_f<T>(row[tid]), tid));
  const int tail0 = cut.head + cut.groups * kGroup;
  if (seg == a.segs - 1 && tid < cut.tail)
    grow[tail0 + tid] = from_f<T>(none ? 0.f : one(to_f<T>(row[tail0 + tid]), tail0 + tid));
}

// CTAs per row: one where the rows fill the GPU, else as many (2, 4, 8) as give every SM a CTA and
// each CTA at least half a group per thread; more where one CTA's group maxima would not fit.
int cluster_for(int64_t rows, int64_t V, bool top) {
  int cs = 1;
  while (cs < kMaxCluster && rows * cs * 2 <= sm_count() * 2 && V / (2 * cs) >= kThreads * kGroup / 2) cs *= 2;
  if (top)
    while (cs < kMaxCluster && (V / kGroup) / cs + 2 > kMaxGroupMax - 2) cs *= 2;
  return cs;
}

int check_rows(const char* what, const void* logits, int64_t rows, int64_t inner, int64_t V, float temperature,
               float softcap, int dt) {
  AK_REQUIRE(valid_dtype(dt), AK_ERR_DTYPE, "%s: unsupported dtype %d", what, dt);
  AK_REQUIRE(rows >= 0 && inner > 0 && V > 0 && V < (1LL << 30) && rows < (1LL << 27), AK_ERR_SHAPE,
             "%s: bad shape: %lld rows of %lld", what, (long long)rows, (long long)V);
  AK_REQUIRE(temperature >= kLowestTemperature && temperature < INFINITY, AK_ERR_ARG,
             "%s: temperature must be at least 2^-100 and finite", what);
  AK_REQUIRE(softcap == 0.f || (softcap >= kLowestSoftcap && softcap < INFINITY), AK_ERR_ARG,
             "%s: softcap must be 0, or at least 2^-100 and finite", what);
  AK_REQUIRE(rows == 0 || logits, AK_ERR_ARG, "%s: null pointer", what);
  AK_REQUIRE((reinterpret_cast<uintptr_t>(logits) % elem_size(dt)) == 0, AK_ERR_ARG,
             "%s: logits not aligned to their type", what);
  return AK_OK;
}

// Rows up to kShortRow elements: a warp each where there are enough of them to fill the GPU with
// warps (100000 rows of 1500 bf16 values: 77 us, a CTA each 262 us), else, and where alternatives
// are wanted, a CTA of 128 threads.
constexpr int64_t kShortRow = 4096, kSmallRow = 8192;

template <typename T, int NT>
void (*pick_fwd(const Squash& q, bool ent, bool top))(const T*, FwdArgs) {
  AK_DISPATCH_CAP(q, CAP, return ent ? (top ? token_logprobs_fwd_kernel<T, CAP, true, true, NT>
                                            : token_logprobs_fwd_kernel<T, CAP, true, false, NT>)
                                     : (top ? token_logprobs_fwd_kernel<T, CAP, false, true, NT>
                                            : token_logprobs_fwd_kernel<T, CAP, false, false, NT>));
}

template <typename T>
int launch_fwd(const T* logits, const FwdArgs& a, int64_t rows, cudaStream_t st) {
  const bool ent = a.entropy != nullptr, top = a.k > 0;
  if (!top && a.V <= kShortRow && rows >= 4 * sm_count()) {
    auto kern = token_logprobs_warp_kernel<T, kNoCap, true>;
    AK_DISPATCH_CAP(a.q, CAP, kern = ent ? token_logprobs_warp_kernel<T, CAP, true>
                                         : token_logprobs_warp_kernel<T, CAP, false>);
    const int64_t grid = (rows + kThreads / 32 - 1) / (kThreads / 32);
    AK_CUDA_TRY(launch_rows(kern, grid, kThreads, 1, 0, st, logits, a, rows), "ak_token_logprobs_fwd");
    return AK_OK;
  }
  const bool few = a.V <= kSmallRow && a.cs == 1;
  const int nt = few ? kFew : kThreads;
  auto kern = few ? pick_fwd<T, kFew>(a.q, ent, top) : pick_fwd<T, kThreads>(a.q, ent, top);
  const size_t smem = top ? ((size_t)(a.V / kGroup) / a.cs + 3 + 4) * 4 : 0;  // read four at a time
  AK_CUDA_TRY(launch_rows(kern, rows * a.cs, nt, a.cs, smem, st, logits, a), "ak_token_logprobs_fwd");
  return AK_OK;
}

}  // namespace
}  // namespace ak

using namespace ak;

extern "C" int ak_token_logprobs_fwd(float* logprobs, float* entropy, float* lse, float* row_stats, float* top_lp,
                                     int64_t* top_idx, const void* logits, const int64_t* targets, int64_t rows,
                                     int64_t inner, int64_t stride_outer, int64_t stride_inner, int64_t V, int64_t k,
                                     float temperature, float softcap, int64_t ignore_index, int dt, void* stream) {
  clear_error();
  int rc = check_rows("ak_token_logprobs_fwd", logits, rows, inner, V, temperature, softcap, dt);
  if (rc) return rc;
  AK_REQUIRE(k >= 0 && k <= kMaxTop && k <= V, AK_ERR_SHAPE,
             "ak_token_logprobs_fwd: top_k %lld must be at most %d and at most the vocabulary", (long long)k, kMaxTop);
  AK_REQUIRE(k == 0 || V <= (int64_t)kMaxCluster * kGroup * (kMaxGroupMax - 4), AK_ERR_SHAPE,
             "ak_token_logprobs_fwd: vocabulary of %lld too large for top_k", (long long)V);
  if (rows == 0) return AK_OK;
  AK_REQUIRE((k == 0) || (top_lp && top_idx), AK_ERR_ARG, "ak_token_logprobs_fwd: null top_lp or top_idx");
  AK_REQUIRE(!logprobs || targets, AK_ERR_ARG, "ak_token_logprobs_fwd: logprobs need targets");
  AK_REQUIRE(aligned16(row_stats), AK_ERR_ARG, "ak_token_logprobs_fwd: row_stats not 16-byte aligned");
  FwdArgs a{};
  a.logprobs = logprobs; a.entropy = entropy; a.lse = lse;
  a.stats = reinterpret_cast<float4*>(row_stats);
  a.top_lp = top_lp; a.top_idx = top_idx; a.targets = targets;
  a.addr = RowAddr{inner, stride_outer, stride_inner};
  a.ignore_index = ignore_index;
  a.V = (int)V; a.k = (int)k; a.cs = cluster_for(rows, V, k > 0);
  a.q = make_squash(temperature, softcap);
  AK_DISPATCH_DTYPE(dt, T, return launch_fwd<T>((const T*)logits, a, rows, (cudaStream_t)stream));
  return AK_OK;
}

extern "C" int ak_token_logprobs_bwd(void* grad, const void* logits, const int64_t* targets, const float* row_stats,
                                     const float* g_logprobs, const float* g_entropy, int64_t rows, int64_t inner,
                                     int64_t stride_outer, int64_t stride_inner, int64_t V, float temperature,
                                     float softcap, int64_t ignore_index, int dt, void* stream) {
  clear_error();
  int rc = check_rows("ak_token_logprobs_bwd", logits, rows, inner, V, temperature, softcap, dt);
  if (rc) return rc;
  if (rows == 0) return AK_OK;
  AK_REQUIRE(grad && row_stats && aligned16(row_stats), AK_ERR_ARG,
             "ak_token_logprobs_bwd: null pointer, or row_stats not 16-byte aligned");
  AK_REQUIRE(!g_logprobs || targets, AK_ERR_ARG, "ak_token_logprobs_bwd: a gradient of logprobs needs targets");
  AK_REQUIRE((reinterpret_cast<uintptr_t>(grad) % elem_size(dt)) == 0, AK_ERR_ARG,
             "ak_token_logprobs_bwd: grad not aligned to its type");
  BwdArgs a{};
  a.stats = reinterpret_cast<const float4*>(row_stats);
  a.g_lp = g_logprobs; a.g_ent = g_entropy; a.targets = targets;
  a.addr = RowAddr{inner, stride_outer, stride_inner};
  a.ignore_index = ignore_index;
  a.rows = rows;
  a.V = (int)V;
  a.segs = (int)std::max<int64_t>(1, (V / kGroup + kBwdGroups - 1) / kBwdGroups);
  a.q = make_squash(temperature, softcap);
  AK_REQUIRE(rows * a.segs < (1LL << 32) - 8, AK_ERR_SHAPE, "ak_token_logprobs_bwd: too many rows");
  const bool ent = g_entropy != nullptr;
  AK_DISPATCH_DTYPE(dt, T, {
    auto kern = token_logprobs_bwd_kernel<T, kNoCap, true>;
    AK_DISPATCH_CAP(a.q, CAP, kern = ent ? token_logprobs_bwd_kernel<T, CAP, true> : token_logprobs_bwd_kernel<T, CAP, false>);
    kern<<<(unsigned)((rows * a.segs + kThreads / 32 - 1) / (kThreads / 32)), kThreads, 0, (cudaStream_t)stream>>>(
        (T*)grad, (const T*)logits, a);
  });
  AK_CHECK_LAUNCH("ak_token_logprobs_bwd");
  return AK_OK;
}
