// Chapters (or experts) chosen from router logits z [rows, C], the first S of which are shared and not chosen from:
//
//   s = softmax(z[S:]) or sigmoid(z[S:]);  sel = s + b (balance bias; without one sel = z, whose order is that of s)
//   groups: the N = C - S chapters in G runs; a group is worth its largest sel, or the sum of its two largest; the `keep` best stay
//   the k largest sel in order (sel descending, id ascending), then  w = s / max(sum s, 1e-12)  or  w = s
//   joint list: shared first with u = 1, then u = rho w;  u / max(sum u, 1e-12) where S > 0
//
// A logit at or below the lowest finite bfloat16 (-inf too) is masked: score 0, never before an unmasked one.  A row that runs out
// of candidates is filled up with the lowest ids left, weight 0.  The bias counts in the selection alone.
//
// The order is that of exact arithmetic.  With a bias, or sums of two, fp32 keys carry errors of the exponential and the
// quotient; where neighbours in the order are closer than those errors allow (a row in some hundreds), the few candidates
// concerned are ranked again by 64-bit keys.  Rows that this does not settle (NaN, more keys that are equal or infinite than the lists
// hold) run through the same selection in 64 bits as a whole.  Bare logits need no arithmetic and are always sure.
//
// Bound by HBM for many rows (4 bytes a logit read) by right, by issuing in fact, and by latency for a few.  Up to 512 candidates and
// k < 32 a warp has a row in registers (257 chapters, k = 8, sigmoid, bias, groups: 1 row 8 us, 1,000 rows 12, 8,192 rows 31; by a CTA
// a row 10, 27 and 107; 513 chapters, k = 31, softmax, bias: 12, 18.5 and 105 against 10, 29 and 119), beyond that a CTA, or a warp
// that streams it where there are many.  Either way the k + 1 largest lie among the values above a bound that at least k + 1 of
// the threads' own maxima reach, found by bisection; what lies above it is ranked.  (Where fewer threads have a candidate, or fewer
// candidates are there than k + 1, all of them are: 8,192 rows of 64 chapters in 8 groups, 2 kept, k = 16: 29 us; in 64 bits 124.)
#include <algorithm>
#include <cfloat>

#include "moc_common.cuh"

namespace moc {
namespace {

constexpr float kMaskedLogit = -3.3895313892515355e38f;      // lowest finite bfloat16
constexpr int kMostK = 128, kWarpMostK = 31, kWarpMostN = 512, kMostN = 16384, kMostGroups = 64;
constexpr int kSelCand = 512;
constexpr int kWarpRows = 4;                 // rows (warps) of a CTA
// Keys order like the numbers (larger first), with what may not be chosen below: distinct, the lowest id on top.
constexpr uint32_t kFiller = 0x00400000u;

struct SelectParams {
  const void* logits;
  const float* bias;              // [C] or NULL
  long long* idx;
  float* weights;
  int* comb_idx;
  float* comb_w;
  float* row_stats;               // [rows, 4] = largest logit, sum of exponentials, sum of chosen scores, sum of u
  int* load;                      // [C] or NULL
  long long ld;
  int rows, N, S, k, groups, keep, per;
  int need;                       // values that a bound has to leave: k + 1, or all there can be (of the groups that stay)
  FastDiv per_group;
  int sigmoid, top2, renorm;
  int count_here;                 // the launch is one CTA, which counts as well (`load` from zero)
  float rho;
};

__device__ __forceinline__ float logit_of(const float* z, long long i) { return z[i]; }
__device__ __forceinline__ float logit_of(const __nv_bfloat16* z, long long i) { return __bfloat162float(z[i]); }
__device__ __forceinline__ void store_logit(float* z, long long i, float v) { z[i] = v; }
__device__ __forceinline__ void store_logit(__nv_bfloat16* z, long long i, float v) { z[i] = __float2bfloat16(v); }
__device__ __forceinline__ bool masked(float z) { return z <= kMaskedLogit; }

__device__ __forceinline__ uint32_t to_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);             // (-0 and 0 are one)
  return v != v ? 0xFFFFFFFFu : (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t to_key(double v) {
  const uint64_t u = __double_as_longlong(v + 0.0);
  return v != v ? ~0ull : (u >> 63) ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float((k >> 31) ? k & 0x7FFFFFFFu : ~k); }
__device__ __forceinline__ double of_key(uint64_t k) {
  return __longlong_as_double((k >> 63) ? k & ~(1ull << 63) : ~k);
}
template <typename K> struct KeyOf;
template <> struct KeyOf<float> { using type = uint32_t; };
template <> struct KeyOf<double> { using type = uint64_t; };

__device__ __forceinline__ uint64_t warp_most(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { const uint64_t t = __shfl_xor_sync(0xffffffffu, v, o); v = t > v ? t : v; }
  return v;
}
template <typename T> __device__ __forceinline__ T warp_total(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
template <typename K> __device__ __forceinline__ K score_of(const SelectParams& p, float z, float m, K total) {
  if (masked(z)) return K(0);
  if (p.sigmoid) return K(1) / (K(1) + exp_of(-static_cast<K>(z)));
  return exp_of(static_cast<K>(z) - static_cast<K>(m)) / total;
}
// key of candidate c; `group`: the value that a group is judged by (scores where no bias and sums of two)
template <typename K>
__device__ __forceinline__ typename KeyOf<K>::type candidate_key(const SelectParams& p, float z, int c, float m, K total, bool group) {
  using U = typename KeyOf<K>::type;
  if (masked(z)) return static_cast<U>(kFiller - c);
  const K sel = p.bias != nullptr ? score_of<K>(p, z, m, total) + static_cast<K>(p.bias[p.S + c])
                : group && p.top2 ? score_of<K>(p, z, m, total) : static_cast<K>(z);
  return sel == -INFINITY ? static_cast<U>(kFiller - c) : to_key(sel);
}
template <typename U> __device__ __forceinline__ bool chosen_from(U key) { return key > static_cast<U>(kFiller); }

// whether candidate ia with key a comes before ib with key b
__device__ __forceinline__ bool ahead(uint64_t a, int ia, uint64_t b, int ib) { return a > b || (a == b && ia < ib); }

// Fast keys of the first pass (softmax: `e` = exp(z - m) and 1 / total): -inf for what may not be chosen, NaN stays.
__device__ __forceinline__ float fast_sigmoid(float z) {
  float e, s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
  return s;
}

// How far fast keys can be off.  Sigmoid: the exponential is off by 2 + 1.2 |z| ulp, which the slope s (1 - s) <= 1/4 brings
// below 4e-8, the sum and the reciprocal by another 3 ulp of at most 1: 2.5e-7.
// Softmax, in units u = 2^-24 of the largest score 1 / total.  The sum of the exponentials: 4 u of a term's exponential (2 ulp); |z - m| u of its
// argument, which averages over the terms by their size: n terms of e^-x against one of 1 make x n e^-x / (1 + n e^-x), 6.8 u at most for
// n = 16,384, 8 u where m is rounded up to a whole number; additions one after another, 16 of a thread's, 5 across a warp, 5 across
// warps.  That is 38 u where a thread has its logits in registers.  Streaming, a lane's sum moves to a larger reference with a factor
// of 4 u each time; references are whole numbers, so what has moved j times is e^(1-j) of the sum or less: the average of j over the 512
// terms of a lane is below 4.7, 19 u; 4 u more across lanes and 6.5 u back to the largest logit, but 5 u of additions alone (16 terms
// by a tree, the rest in 64 bits): 46.5 u = 2.8e-6.  The key's own exponential, argument, quotient and product: 6.5 u, together 3.2e-6.
// The bias's addition: half an ulp of the key.  A sum of two keys adds theirs.
constexpr float kSumError = 3.0e-6f, kKeyError = 3.5e-6f;
__device__ __forceinline__ float key_error(const SelectParams& p, float v, float inv_total) {
  return (p.sigmoid ? 3e-7f : kKeyError * inv_total) + 6.1e-8f * fabsf(v);
}
// whether a > b for certain (NaN: no)
__device__ __forceinline__ bool apart(const SelectParams& p, float a, float b, float inv_total) {
  return a - b > key_error(p, a, inv_total) + key_error(p, b, inv_total);
}

// the two largest keys of a group
template <typename U> struct Best2 { U a, b; };
template <typename U> __device__ __forceinline__ void take(Best2<U>& t, U k) {
  if (k > t.a) { t.b = t.a; t.a = k; }
  else if (k > t.b) t.b = k;
}
template <typename U> __device__ __forceinline__ U group_value(const SelectParams& p, const Best2<U>& t) {
  return p.top2 && chosen_from(t.a) && chosen_from(t.b) ? to_key(of_key(t.a) + of_key(t.b)) : t.a;
}

// One row's lists, by one warp; pick(j, ok, z): candidate of the j-th place, whether it may be chosen at all, and its logit.
template <int EACH, typename Pick>
__device__ __forceinline__ void write_row(const SelectParams& p, long long row, float m, float total, Pick pick) {
  const int lane = threadIdx.x & 31;
  int id[EACH];
  float w[EACH], mass = 0.f;
#pragma unroll
  for (int q = 0; q < EACH; ++q) {
    const int j = lane + 32 * q;
    id[q] = 0;
    w[q] = 0.f;
    if (j < p.k) {
      bool ok;
      float z;
      id[q] = pick(j, ok, z);
      if (ok) w[q] = score_of<float>(p, z, m, total);
      mass += w[q];
      if (p.count_here) atomicAdd(p.load + p.S + id[q], 1);
    }
  }
  mass = warp_total(mass);
  const float floor_mass = max_nan(mass, 1e-12f);          // (divided by, not multiplied with its reciprocal: one rounding)
  float sum = 0.f;
#pragma unroll
  for (int q = 0; q < EACH; ++q) {
    const int j = lane + 32 * q;
    if (j >= p.k) break;
    if (p.renorm) w[q] /= floor_mass;
    sum += p.rho * w[q];
    p.idx[row * p.k + j] = id[q] + p.S;
    p.weights[row * p.k + j] = w[q];
  }
  sum = static_cast<float>(p.S) + warp_total(sum);
  const float joint = max_nan(sum, 1e-12f);
  int* ci = p.comb_idx + row * (p.S + p.k);
  float* cw = p.comb_w + row * (p.S + p.k);
  for (int j = lane; j < p.S; j += 32) { ci[j] = j; cw[j] = 1.f / joint; }
#pragma unroll
  for (int q = 0; q < EACH; ++q) {
    const int j = lane + 32 * q;
    if (j >= p.k) break;
    ci[p.S + j] = id[q] + p.S;
    cw[p.S + j] = p.S > 0 ? p.rho * w[q] / joint : w[q];
  }
  if (lane == 0 && p.row_stats != nullptr) reinterpret_cast<float4*>(p.row_stats)[row] = make_float4(m, total, mass, sum);
}

// 64-bit sum of the exponentials of a row, by `threads` threads of which this is `t`; their parts are still to be added
template <typename LT> __device__ __noinline__ double total64(const LT* z, int n, float m, int t, int threads) {
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 1
  for (int c = t; c < n; c += 4 * threads) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float v = c + u * threads < n ? logit_of(z, c + u * threads) : -INFINITY;
      if (!masked(v)) sum[u] += exp(static_cast<double>(v) - static_cast<double>(m));
    }
  }
  return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}
template <typename LT> __device__ __noinline__ uint64_t key64(const SelectParams& p, const LT* z, int c, float m, double total, bool group) {
  return candidate_key<double>(p, logit_of(z, c), c, m, total, group);
}

// Candidates ranked by 64-bit keys: whether a, the next above b, is before it for certain.  Softmax keys may have been formed with
// the fp32 sum of the exponentials, off by kSumError at most: it scales the difference of the scores, not that of the biases.
__device__ __forceinline__ bool apart64(const SelectParams& p, uint64_t a, int ia, uint64_t b, int ib) {
  if (p.sigmoid || a == b) return p.sigmoid || p.bias[p.S + ia] == p.bias[p.S + ib];
  const double sa = of_key(a), sb = of_key(b);
  const double da = sa - static_cast<double>(p.bias[p.S + ia]), db = sb - static_cast<double>(p.bias[p.S + ib]);
  return sa - sb > kSumError * (1 + kSumError) * fabs(da - db);
}
// Whether fp32 values tell the groups that stay (least of them) from those that go: two keys each, or bare logits.  (Groups without a
// candidate are behind all others, in the order of their ids.)
__device__ __forceinline__ bool groups_apart(const SelectParams& p, float least, float most, float inv_total) {
  return (p.bias == nullptr && !p.top2) || most == -INFINITY ||
         least - most > 2.f * (key_error(p, least, inv_total) + key_error(p, most, inv_total));
}
// Places of candidates (ids in the complements of the low words of `cand`) by their 64-bit keys, by `threads` threads of which this
// is `t0`.  Returns whether this thread has met one that is not for certain before the next.
__device__ __noinline__ bool rank_wide(const SelectParams& p, const unsigned long long* cand, const uint64_t* wide, int n, int t0, int threads,
                                       int* place) {
  bool unclear = false;
  for (int t = t0; t < n; t += threads) {
    const int id = static_cast<int>(~static_cast<uint32_t>(cand[t]));
    const uint64_t mine = wide[t];
    int rank = 0, nid = -1;
    uint64_t next = 0;
    for (int j = 0; j < n; ++j) {
      const int oid = static_cast<int>(~static_cast<uint32_t>(cand[j]));
      const uint64_t o = wide[j];
      rank += ahead(o, oid, mine, id);
      if (ahead(mine, id, o, oid) && (nid < 0 || ahead(o, oid, next, nid))) { next = o; nid = oid; }
    }
    if (rank < p.k) {
      place[rank] = id;
      unclear |= nid >= 0 && !apart64(p, mine, id, next, nid);
    }
  }
  return unclear;
}
// The value of a group by 64-bit keys of the candidates that may be among its best, by one warp.  (Eight loads in flight a lane: one
// row that comes here would otherwise end after all others, 20 us late for groups of 512.)
template <typename LT>
__device__ __noinline__ uint64_t group_value64(const SelectParams& p, const LT* z, int g, float m, float inv_total, double total) {
  constexpr int kFlight = 8;
  const int lane = threadIdx.x & 31, end = (g + 1) * p.per;
  const bool biased = p.bias != nullptr;
  const float* bias = biased ? p.bias + p.S : nullptr;
  auto each = [&](auto go) {                           // go(candidate, its fast key), kFlight of a lane at a time
    for (int c0 = g * p.per + lane; c0 < end; c0 += 32 * kFlight) {
      float v[kFlight], b[kFlight];
#pragma unroll
      for (int i = 0; i < kFlight; ++i) {
        const bool in = c0 + 32 * i < end;
        v[i] = in ? logit_of(z, c0 + 32 * i) : -INFINITY;
        b[i] = in && biased ? bias[c0 + 32 * i] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < kFlight; ++i) {
        const float sc = p.sigmoid ? fast_sigmoid(v[i]) : expf(v[i] - m) * inv_total;
        go(c0 + 32 * i, masked(v[i]) ? -INFINITY : biased ? sc + b[i] : p.top2 ? sc : v[i]);
      }
    }
  };
  float a = -INFINITY, b = -INFINITY;
  each([&](int, float v) {
    b = fmaxf(b, fminf(a, v));
    a = fmaxf(a, v);
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
    b = fmaxf(fminf(a, oa), fmaxf(b, ob));
    a = fmaxf(a, oa);
  }
  const float last = p.top2 ? b : a;
  const float edge = last - 2.f * key_error(p, last, inv_total);
  Best2<uint64_t> t{0, 0};
  each([&](int c, float v) {
    if (c < end && v >= edge) take(t, key64(p, z, c, m, total, true));
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t ka = __shfl_xor_sync(0xffffffffu, t.a, o), kb = __shfl_xor_sync(0xffffffffu, t.b, o);
    take(t, ka);
    take(t, kb);
  }
  return group_value(p, t);
}
// Places n .. k - 1 of a row that has n < k candidates (their ids in place[0 .. n)), by one warp: the lowest other ids, complemented.
// They lie below k, as at most n of those are candidates.
__device__ __forceinline__ void fill_up(int* place, int n, int k) {
  const int lane = threadIdx.x & 31;
  for (int id0 = 0, at = n; at < k; id0 += 32) {
    const int id = id0 + lane;
    bool free = id < k;
    for (int j = 0; j < n; ++j) free &= place[j] != id;
    const uint32_t votes = __ballot_sync(0xffffffffu, free);
    const int pos = at + __popc(votes & ((1u << lane) - 1u));
    if (free && pos < k) place[pos] = ~id;
    at += __popc(votes);
  }
  __syncwarp();
}
// Which groups stay, where fp32 values (of groups lane and lane + 32) close at the border between `least` and `most`: those near it
// again in 64 bits.  The others are ahead of, or behind, all of them in any case.
template <typename LT>
__device__ __noinline__ unsigned long long choose_groups_near(const SelectParams& p, const LT* z, float v0, float v1, float least, float most,
                                                              float m, float inv_total) {
  const int lane = threadIdx.x & 31;
  const double total = p.sigmoid ? 1.0 : warp_total(total64(z, p.N, m, lane, 32));
  const float slack = 2.f * (key_error(p, least, inv_total) + key_error(p, most, inv_total));
  const float value[2] = {v0, v1};
  uint64_t exact[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const bool near = lane + 32 * r < p.groups && value[r] >= most - slack && value[r] <= least + slack;
    exact[r] = to_key(static_cast<double>(value[r]));
    uint32_t todo = __ballot_sync(0xffffffffu, near);
    while (todo != 0) {
      const int g = __ffs(todo) - 1;
      todo &= todo - 1;
      const uint64_t v = group_value64(p, z, g + 32 * r, m, inv_total, total);
      if (lane == g) exact[r] = v;
    }
  }
  int rank[2] = {0, 0};
  for (int g = 0; g < p.groups; ++g) {
    const uint64_t other = __shfl_sync(0xffffffffu, exact[g >> 5], g & 31);
#pragma unroll
    for (int r = 0; r < 2; ++r) rank[r] += other > exact[r] || (other == exact[r] && g < lane + 32 * r);
  }
  const uint32_t lo = __ballot_sync(0xffffffffu, lane < p.groups && rank[0] < p.keep);
  const uint32_t hi = __ballot_sync(0xffffffffu, lane + 32 < p.groups && rank[1] < p.keep);
  return static_cast<unsigned long long>(hi) << 32 | lo;
}

// ---- a warp a row ----------------------------------------------------------------------------
// What a warp keeps of the k best candidates seen so far, largest first.
struct BestList {
  uint64_t key[kMostK];
  int id[kMostK];
};

// The whole selection by 64-bit keys, by one warp: the candidates stream by, those that are before the last place go into the list.
template <typename LT>
__device__ __noinline__ void choose_warp64(const SelectParams& p, const LT* z, float m, BestList& list) {
  const int lane = threadIdx.x & 31;
  double total = 1.0;
  if (!p.sigmoid) total = warp_total(total64(z, p.N, m, lane, 32));
  unsigned long long kept = ~0ull;
  if (p.keep < p.groups) {
    uint64_t value[2] = {0, 0};
    int rank[2] = {0, 0};
    for (int g = 0; g < p.groups; ++g) {
      Best2<uint64_t> t{0, 0};
      for (int c = g * p.per + lane; c < (g + 1) * p.per; c += 32) take(t, key64(p, z, c, m, total, true));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const uint64_t a = __shfl_xor_sync(0xffffffffu, t.a, o), b = __shfl_xor_sync(0xffffffffu, t.b, o);
        take(t, a);
        take(t, b);
      }
      if (lane == (g & 31)) value[g >> 5] = group_value(p, t);
    }
    for (int g = 0; g < p.groups; ++g) {
      const uint64_t other = __shfl_sync(0xffffffffu, value[g >> 5], g & 31);
#pragma unroll
      for (int r = 0; r < 2; ++r) rank[r] += ahead(other, g, value[r], lane + 32 * r);
    }
    const uint32_t lo = __ballot_sync(0xffffffffu, lane < p.groups && rank[0] < p.keep);
    const uint32_t hi = __ballot_sync(0xffffffffu, lane + 32 < p.groups && rank[1] < p.keep);
    kept = static_cast<unsigned long long>(hi) << 32 | lo;
  }
  for (int j = lane; j < p.k; j += 32) { list.key[j] = 0; list.id[j] = 0x7FFFFFFF; }
  __syncwarp();
  for (int c0 = 0; c0 < p.N; c0 += 32) {
    const int c = c0 + lane;
    uint64_t key = 0;
    if (c < p.N) key = kept >> (div_of(c, p.per_group) & 63) & 1 ? key64(p, z, c, m, total, false) : static_cast<uint64_t>(kFiller - c);
    uint32_t todo = __ballot_sync(0xffffffffu, ahead(key, c, list.key[p.k - 1], list.id[p.k - 1]) && c < p.N);
    while (todo != 0) {
      const int from = __ffs(todo) - 1, id = c0 + from;
      todo &= todo - 1;
      const uint64_t mine = __shfl_sync(0xffffffffu, key, from);
      uint64_t k_new[kMostK / 32];
      int i_new[kMostK / 32];
#pragma unroll
      for (int q = 0; q < kMostK / 32; ++q) {
        const int j = lane + 32 * q;
        k_new[q] = 0;
        i_new[q] = 0;
        if (j >= p.k) continue;
        // entries behind the new one move down by one place
        const bool here = !ahead(list.key[j], list.id[j], mine, id);
        const bool above = j > 0 && !ahead(list.key[j - 1], list.id[j - 1], mine, id);
        k_new[q] = above ? list.key[j - 1] : here ? mine : list.key[j];
        i_new[q] = above ? list.id[j - 1] : here ? id : list.id[j];
      }
      __syncwarp();
#pragma unroll
      for (int q = 0; q < kMostK / 32; ++q)
        if (lane + 32 * q < p.k) { list.key[lane + 32 * q] = k_new[q]; list.id[lane + 32 * q] = i_new[q]; }
      __syncwarp();
    }
  }
}

// The groups that stay (bit g), from keys in shared memory (candidate c at c + c / 32), by R groups a lane (2: of more than 32) or
// 1 / lanes of one.
template <int R, typename LT>
__device__ __forceinline__ unsigned long long choose_groups_warp(const SelectParams& p, const float* sk, const LT* z, float m, float inv_total) {
  const int lane = threadIdx.x & 31;
  const int shift = R > 1 || p.groups > 16 ? 0 : p.groups > 8 ? 1 : p.groups > 4 ? 2 : p.groups > 2 ? 3 : 4;     // log2 of a group's lanes
  const int lanes = 1 << shift, sub = lane & (lanes - 1);
  float value[R];
  int rank[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int g = (lane >> shift) + 32 * r;
    float a = -INFINITY, b = -INFINITY;
    if (g < p.groups)
      for (int c = g * p.per + sub; c < (g + 1) * p.per; c += lanes) {
        const float v = sk[c + (c >> 5)];
        b = fmaxf(b, fminf(a, v));
        a = fmaxf(a, v);
      }
    for (int o = lanes >> 1; o > 0; o >>= 1) {
      const float oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
      b = fmaxf(fminf(a, oa), fmaxf(b, ob));
      a = fmaxf(a, oa);
    }
    value[r] = p.top2 && b > -INFINITY ? a + b : a;
    rank[r] = 0;
  }
  for (int g = 0; g < p.groups; ++g) {
    const float other = __shfl_sync(0xffffffffu, R > 1 && g >= 32 ? value[R - 1] : value[0], (g << shift) & 31);
#pragma unroll
    for (int r = 0; r < R; ++r) rank[r] += other > value[r] || (other == value[r] && g < (lane >> shift) + 32 * r);
  }
  float least = INFINITY, most = -INFINITY;            // of those that stay, of those that go
  uint32_t mask[2] = {0, 0};
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int g = (lane >> shift) + 32 * r;
    if (g >= p.groups) continue;
    if (rank[r] < p.keep) {
      mask[r] |= 1u << (g & 31);
      least = fminf(least, value[r]);
    } else {
      most = fmaxf(most, value[r]);
    }
  }
  unsigned long long kept = __reduce_or_sync(0xffffffffu, mask[0]);
  if constexpr (R > 1) kept |= static_cast<unsigned long long>(__reduce_or_sync(0xffffffffu, mask[1])) << 32;
  least = of_key(__reduce_min_sync(0xffffffffu, to_key(least)));
  most = of_key(__reduce_max_sync(0xffffffffu, to_key(most)));
  if (groups_apart(p, least, most, inv_total)) return kept;
  const float v0 = __shfl_sync(0xffffffffu, value[0], (lane << shift) & 31);
  return choose_groups_near(p, z, lane << shift < 32 || R > 1 ? v0 : -INFINITY, R > 1 ? value[R - 1] : -INFINITY, least, most, m, inv_total);
}

template <typename LT, int NV>
__global__ void __launch_bounds__(32 * kWarpRows)
select_warp_kernel(const SelectParams p) {
  // keys of the candidates for the groups, or the list of the 64-bit selection
  constexpr int kWords = NV * 33 * 4 > static_cast<int>(sizeof(BestList)) ? NV * 33 * 4 / 8 + 1 : static_cast<int>(sizeof(BestList) / 8);
  __shared__ uint64_t keys[kWarpRows][kWords];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * kWarpRows + warp;
  if (p.count_here) {
    for (int c = threadIdx.x; c < p.S + p.N; c += 32 * kWarpRows) p.load[c] = 0;
    __syncthreads();
  }
  if (row >= p.rows) return;
  const LT* zr = static_cast<const LT*>(p.logits) + row * p.ld + p.S;
  float z[NV], v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) z[i] = lane + 32 * i < p.N ? logit_of(zr, lane + 32 * i) : -INFINITY;
  if (p.bias != nullptr) {
    const float* b = p.bias + p.S;
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = lane + 32 * i < p.N ? b[lane + 32 * i] : 0.f;
  }
  float m = 0.f, total = 1.f, inv_total = 1.f;
  const bool judged = p.keep < p.groups && p.top2 && p.bias == nullptr;      // groups by scores, picks by logits
  float* sk = reinterpret_cast<float*>(keys[warp]);
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float sc = p.bias != nullptr || judged ? fast_sigmoid(z[i]) : 0.f;
      if (judged) sk[lane + 33 * i] = masked(z[i]) ? -INFINITY : sc;
      v[i] = masked(z[i]) ? -INFINITY : p.bias != nullptr ? sc + v[i] : z[i];
    }
  } else {
    m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i) m = fmaxf(m, z[i]);
    m = of_key(__reduce_max_sync(0xffffffffu, to_key(m)));
    float e[NV];
    total = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) { e[i] = masked(z[i]) ? 0.f : expf(z[i] - m); total += e[i]; }
    total = warp_total(total);
    if (total == 0.f) total = 1.f;                  // (every logit masked)
    inv_total = 1.f / total;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (judged) sk[lane + 33 * i] = masked(z[i]) ? -INFINITY : e[i] * inv_total;
      v[i] = masked(z[i]) ? -INFINITY : p.bias != nullptr ? e[i] * inv_total + v[i] : z[i];
    }
  }
  bool sure = true;
  if (p.keep < p.groups) {
    if (!judged) {
#pragma unroll
      for (int i = 0; i < NV; ++i) sk[lane + 33 * i] = v[i];
    }
    __syncwarp();
    if (p.groups <= 32) {
      const uint32_t k32 = static_cast<uint32_t>(choose_groups_warp<1>(p, sk, zr, m, inv_total));
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (!(k32 >> (div_of(lane + 32 * i, p.per_group) & 31) & 1)) v[i] += -INFINITY;        // (NaN stays)
    } else {
      const unsigned long long kept = choose_groups_warp<2>(p, sk, zr, m, inv_total);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (!(kept >> (div_of(lane + 32 * i, p.per_group) & 63) & 1)) v[i] += -INFINITY;
    }
    __syncwarp();
  }
  // lane j keeps the j-th pick
  int pick = 0;
  bool ok = false;
  float chosen = 0.f;              // its logit
  float best = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) best = max_nan(best, v[i]);
  const uint32_t mine = to_key(best), none = 0x007FFFFFu;          // (the key of -inf)
  uint32_t hi = __reduce_max_sync(0xffffffffu, mine);
  const int some = __popc(__ballot_sync(0xffffffffu, mine > none));
  int need = p.need;
  if (some == 0) {                                           // nothing to choose from: the lowest ids
    pick = lane;
  } else if (hi == 0xFFFFFFFFu) {                            // NaN
    sure = false;
  } else if (sure) {
    uint32_t lo;
    if (some >= need) {
      // count(lanes >= lo) >= need, count(> hi) == 0
      lo = __reduce_min_sync(0xffffffffu, mine > none ? mine : 0xFFFFFFFFu);
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        const int n = __popc(__ballot_sync(0xffffffffu, mine >= mid));
        if (n >= need) {
          lo = mid;
          if (n <= need + 2) break;
        } else {
          hi = mid - 1;
        }
      }
    } else {                                                 // candidates in few lanes (few groups, masks): all of them to begin with
      float least = INFINITY;
      int count = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (v[i] > -INFINITY) { least = fminf(least, v[i]); ++count; }
      lo = __reduce_min_sync(0xffffffffu, to_key(least));
      need = min(need, __reduce_add_sync(0xffffffffu, count));
    }
    hi = 0xFF7FFFFFu;                                        // (the largest finite number's key)
    float edge;
    int n;
    while (true) {
      edge = of_key(lo);
      if (p.bias != nullptr) edge = fmaxf(edge - 2.f * key_error(p, edge, inv_total), -FLT_MAX);        // what may yet turn out to reach the bound
      int count = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) count += v[i] >= edge;
      n = __reduce_add_sync(0xffffffffu, count);
      if (n <= 32) break;
      // too many for a candidate a lane: a higher bound that at least `need` values reach
      int above = 0;
      uint32_t mid = lo;
      while (lo < hi) {
        mid = lo + (hi - lo + 1) / 2;
        const float bound = of_key(mid);
        count = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) count += v[i] >= bound;
        above = __reduce_add_sync(0xffffffffu, count);
        if (above >= need) break;
        hi = mid - 1;
      }
      if (lo >= hi) break;
      lo = mid;
    }
    sure = n <= 32 && n >= need && edge < INFINITY;          // (equal keys, or infinite ones)
    if (sure) {
      // a candidate a lane: id and key through shared memory
      uint32_t* out = reinterpret_cast<uint32_t*>(keys[warp]);
      int at = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const bool in = v[i] >= edge;
        const uint32_t votes = __ballot_sync(0xffffffffu, in);
        if (in) {
          const int pos = at + __popc(votes & ((1u << lane) - 1u));
          out[pos] = lane + 32 * i;
          out[32 + pos] = __float_as_uint(v[i]);
          out[64 + pos] = __float_as_uint(z[i]);
        }
        at += __popc(votes);
      }
      __syncwarp();
      const int id = lane < n ? static_cast<int>(out[lane]) : 0x7FFFFFFF;
      const float key = lane < n ? __uint_as_float(out[32 + lane]) : -INFINITY, logit = lane < n ? __uint_as_float(out[64 + lane]) : 0.f;
      int rank = 0;
      bool close = false;
      // (candidates came in the order of their ids within a slot only)
      for (int j = 0; j < n; ++j) {
        const float other = __shfl_sync(0xffffffffu, key, j);
        const int oid = __shfl_sync(0xffffffffu, id, j);
        rank += other > key || (other == key && oid < id);
        if (p.bias != nullptr) close |= j != lane && lane < n && !apart(p, fmaxf(other, key), fminf(other, key), inv_total);
      }
      if (__any_sync(0xffffffffu, close)) {
        // again by 64-bit keys: all other candidates are certainly behind the first k of these
        double t64 = total;
#pragma unroll 1
        for (int round = 0; round < 2; ++round) {
          const uint64_t wide = lane < n ? key64(p, zr, id, m, t64, false) : 0;
          rank = 0;
          uint64_t next = 0;
          int nid = -1;
          for (int j = 0; j < n; ++j) {
            const uint64_t other = __shfl_sync(0xffffffffu, wide, j);
            const int oid = __shfl_sync(0xffffffffu, id, j);
            rank += ahead(other, oid, wide, id);
            if (ahead(wide, id, other, oid) && (nid < 0 || ahead(other, oid, next, nid))) { next = other; nid = oid; }
          }
          const bool unclear = lane < n && rank < p.k && nid >= 0 && !apart64(p, wide, id, next, nid);
          if (round > 0 || !__any_sync(0xffffffffu, unclear)) break;
          t64 = warp_total(total64(zr, p.N, m, lane, 32));
        }
      }
      __syncwarp();
      if (lane < n) {
        out[rank] = id;
        out[32 + rank] = __float_as_uint(logit);
      }
      __syncwarp();
      if (n < p.k) fill_up(reinterpret_cast<int*>(out), n, p.k);
      if (lane < max(n, p.k)) {
        const int at = static_cast<int>(out[lane]);
        ok = at >= 0;
        pick = ok ? at : ~at;
        chosen = ok ? __uint_as_float(out[32 + lane]) : 0.f;
      }
    }
  }
  if (!sure) {
    BestList& list = *reinterpret_cast<BestList*>(keys[warp]);
    __syncwarp();
    choose_warp64(p, zr, m, list);
    pick = lane < p.k ? list.id[lane] : 0;
    ok = lane < p.k && chosen_from(list.key[lane]);
    chosen = lane < p.k ? logit_of(zr, pick) : 0.f;
  }
  write_row<1>(p, row, m, total, [&](int, bool& good, float& logit) {      // (k <= 32: place j is this lane's)
    good = ok;
    logit = chosen;
    return pick;
  });
}

// ---- a warp a row, many rows of many candidates -----------------------------------------------
// The row streams by (16 loads a lane in flight); what stays of it are the maxima of runs of S candidates a lane, in shared
// memory.  A bound on those that k + 1 of them reach leaves some dozens of runs, which are read again for the candidates.  No
// barrier, a third of the instructions of a CTA a row.  Bound by issuing: 8,192 rows of 4,097 fp32 logits, sigmoid with a bias, 4 of 8
// groups, k = 16: 68 us (2.0 TB/s; 4,840 instructions a row, 0.59 a cycle and scheduler, two rounds of rows).
// Against a CTA a row (4,097 chapters, us): k = 16, sigmoid, bias, groups: 300 rows 20.5 / 20.5 CTA, 600 rows 23 / 26, 1,200 rows 27 / 42,
// 2,400 rows 33 / 66; k = 16, plain softmax: 300 rows 23 / 16, 600 rows 23 / 23, 2,400 rows 33 / 55; k = 64, softmax, bias: 600 rows
// 55 / 39, 1,200 rows 59 / 53, 2,400 rows 74 / 86, 8,192 rows 151 / 184.
constexpr int kStreamMostK = 64, kStreamHits = 256, kStreamCand = 256, kBatch = 16;
constexpr int kStreamRows = 600, kStreamRowsManyPicks = 1500;      // k <= 32, and more
struct StreamShared {
  union {
    struct {
      unsigned long long cand[kStreamCand];
      uint64_t wide[kStreamCand];
    };
    BestList list;
  };
  int place[kMostK];
  uint16_t hits[kStreamHits];
};
// (explicit operations: the same number when a run is read again)
__device__ __forceinline__ float min3(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
template <bool SIG> __device__ __forceinline__ float stream_score(float z, float m, float inv_total) {
  return SIG ? fast_sigmoid(z) : __fmul_rn(expf(__fsub_rn(z, m)), inv_total);
}
template <bool SIG, bool BIAS> __device__ __forceinline__ float stream_key(float z, float b, float m, float inv_total) {
  return masked(z) ? -INFINITY : BIAS ? __fadd_rn(stream_score<SIG>(z, m, inv_total), b) : z;
}

// SIG: sigmoid scores; BIAS: with a balance bias; GROUPS: some groups go.
template <typename LT, int S, bool SIG, bool BIAS, bool GROUPS>
__global__ void __launch_bounds__(32 * kWarpRows, 7)
select_stream_kernel(const SelectParams p, const int chunks, const FastDiv group_batches) {
  extern __shared__ uint32_t tops_all[];               // [kWarpRows][chunks][32] keys of the runs' maxima
  __shared__ StreamShared shared[kWarpRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * kWarpRows + warp;
  if (row >= p.rows) return;
  StreamShared& s = shared[warp];
  uint32_t* tops = tops_all + warp * chunks * 32;
  const LT* zr = static_cast<const LT*>(p.logits) + row * p.ld + p.S;
  const float* bias = BIAS ? p.bias + p.S : nullptr;
  const int groups = GROUPS ? p.groups : 1, per = GROUPS ? p.per : p.N;
  const int batches = group_batches.d;                                 // of a group
  constexpr int kRuns = kBatch / S;                                    // of a batch
  constexpr uint32_t kNone = 0x007FFFFFu;                              // key of -inf
  if (lane == 0) {                                     // the row on its way to L2 as a whole (its 16-byte pieces)
    const uintptr_t first = (reinterpret_cast<uintptr_t>(zr) + 15) & ~uintptr_t{15}, end = reinterpret_cast<uintptr_t>(zr + p.N) & ~uintptr_t{15};
    if (end > first)
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" :: "l"(first), "r"(static_cast<uint32_t>(end - first)) : "memory");
  }

  float m = 0.f, total = 1.f, inv_total = 1.f;
  if (!SIG) {                                          // maximum and sum against it, rounded up to a whole number; a lane's own until the end
    m = -INFINITY;
    float ref = -INFINITY;
    double sums = 0.0;
    for (int c0 = lane; c0 < p.N; c0 += 32 * kBatch) {
      float z[kBatch], most = m;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) z[i] = c0 + 32 * i < p.N ? logit_of(zr, c0 + 32 * i) : -INFINITY;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) most = fmaxf(most, masked(z[i]) ? -INFINITY : z[i]);
      const float up = ceilf(most);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) z[i] = masked(z[i]) ? 0.f : expf(z[i] - up);
#pragma unroll
      for (int n = kBatch / 2; n > 0; n >>= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) z[i] += z[i + n];
      sums = (ref == up || ref == -INFINITY ? sums : sums * static_cast<double>(expf(ref - up))) + static_cast<double>(z[0]);
      m = most;
      ref = up;
    }
    m = of_key(__reduce_max_sync(0xffffffffu, to_key(m)));
    const float up = ceilf(m);
    sums = warp_total(ref == up || ref == -INFINITY ? sums : sums * static_cast<double>(expf(ref - up)));        // (a lane with NaN alone keeps its NaN)
    total = static_cast<float>(m == -INFINITY ? sums : sums * static_cast<double>(expf(up - m)));
    if (total == 0.f) total = 1.f;                     // (every logit masked)
    inv_total = 1.f / total;
  }

  bool sure = true;
  float value[2] = {-INFINITY, -INFINITY};             // of groups lane and lane + 32
  for (int g = 0; g < groups; ++g) {
    float a = -INFINITY, b = -INFINITY;
    for (int bt = 0; bt < batches; ++bt) {
      const int c0 = bt * 32 * kBatch + lane;          // within the group
      const LT* zg = zr + static_cast<long long>(g) * per + c0;
      const float* bg = BIAS ? bias + g * per + c0 : nullptr;
      float z[kBatch], v[kBatch];
      if ((bt + 1) * 32 * kBatch <= per) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) z[i] = logit_of(zg, 32 * i);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) v[i] = BIAS ? bg[32 * i] : 0.f;
      } else {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) z[i] = c0 + 32 * i < per ? logit_of(zg, 32 * i) : -INFINITY;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) v[i] = BIAS && c0 + 32 * i < per ? bg[32 * i] : 0.f;
      }
      float low = z[0];
#pragma unroll
      for (int i = 1; i < kBatch; i += 2) low = i + 1 < kBatch ? min3(low, z[i], z[i + 1]) : fminf(low, z[i]);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) v[i] = BIAS ? __fadd_rn(stream_score<SIG>(z[i], m, inv_total), v[i]) : z[i];
      if (masked(low)) {                               // (as stream_key has it)
#pragma unroll
        for (int i = 0; i < kBatch; ++i) v[i] = masked(z[i]) ? -INFINITY : v[i];
      }
#pragma unroll
      for (int q = 0; q < kRuns; ++q) {
        float top = v[q * S];
#pragma unroll
        for (int i = 1; i < S; i += 2) top = i + 1 < S ? max3_nan(top, v[q * S + i], v[q * S + i + 1]) : max_nan(top, v[q * S + i]);
        tops[((g * batches + bt) * kRuns + q) * 32 + lane] = to_key(top);
      }
      if (GROUPS) {
        if (!BIAS && p.top2) {
#pragma unroll
          for (int i = 0; i < kBatch; ++i) v[i] = masked(z[i]) ? -INFINITY : stream_score<SIG>(z[i], m, inv_total);
        }
#pragma unroll
        for (int i = 0; i < kBatch; i += 2) {          // the two largest of four, two of which are in order
          const float hi = fmaxf(v[i], v[i + 1]), lo = fminf(v[i], v[i + 1]);
          b = max3(b, lo, fminf(a, hi));
          a = fmaxf(a, hi);
        }
      }
    }
    if (GROUPS) {
      // (neither is NaN) the largest, then the largest of what is left: its lane's second, the others' first
      const uint32_t mine = to_key(a), best = __reduce_max_sync(0xffffffffu, mine);
      const uint32_t holders = __ballot_sync(0xffffffffu, mine == best);
      a = of_key(best);
      if (p.top2) b = of_key(__reduce_max_sync(0xffffffffu, lane == __ffs(holders) - 1 ? to_key(b) : mine));
      if (lane == (g & 31)) value[g >> 5] = p.top2 && b > -INFINITY ? a + b : a;
    }
  }
  if (GROUPS) {
    int rank[2] = {0, 0};
    for (int g = 0; g < groups; ++g) {
      const float other = __shfl_sync(0xffffffffu, value[g >> 5], g & 31);
#pragma unroll
      for (int r = 0; r < 2; ++r) rank[r] += other > value[r] || (other == value[r] && g < lane + 32 * r);
    }
    float least = INFINITY, most = -INFINITY;          // of those that stay, of those that go
    uint32_t stays[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const bool real = lane + 32 * r < groups, in = real && rank[r] < p.keep;
      stays[r] = __ballot_sync(0xffffffffu, in);
      if (in) least = fminf(least, value[r]);
      else if (real) most = fmaxf(most, value[r]);
    }
    least = of_key(__reduce_min_sync(0xffffffffu, to_key(least)));
    most = of_key(__reduce_max_sync(0xffffffffu, to_key(most)));
    if (!groups_apart(p, least, most, inv_total)) {
      const unsigned long long kept = choose_groups_near(p, zr, value[0], value[1], least, most, m, inv_total);
      stays[0] = static_cast<uint32_t>(kept);
      stays[1] = static_cast<uint32_t>(kept >> 32);
    }
    for (int i = 0; i < chunks; ++i) {
      const int g = div_of(i / kRuns, group_batches);
      // (NaN stays to be seen)
      if (!((g < 32 ? stays[0] >> g : stays[1] >> (g - 32)) & 1) && tops[i * 32 + lane] != 0xFFFFFFFFu) tops[i * 32 + lane] = kNone;
    }
  }

  // the bound
  uint32_t lo = 0xFFFFFFFFu, hi = 0;
  int some = 0;
  for (int i = 0; i < chunks; ++i) {
    const uint32_t key = tops[i * 32 + lane];
    hi = max(hi, key);
    if (key > kNone) { ++some; lo = min(lo, key); }
  }
  some = __reduce_add_sync(0xffffffffu, some);
  hi = __reduce_max_sync(0xffffffffu, hi);
  lo = __reduce_min_sync(0xffffffffu, lo);
  const int need = p.need;
  int n = 0;
  if (some == 0) {                                     // nothing to choose from: the lowest ids
    for (int j = lane; j < p.k; j += 32) s.place[j] = ~j;
  } else if (hi == 0xFFFFFFFFu) {
    sure = false;                                      // NaN
  } else if (sure) {
    if (some < need) lo = 0x00800000u;                 // candidates in few runs (masks): all of them (the lowest finite number's key)
    while (some >= need && lo < hi) {                  // count(>= lo) >= need, count(> hi) == 0
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      int count = 0;
#pragma unroll 8
      for (int i = 0; i < chunks; ++i) count += tops[i * 32 + lane] >= mid;
      count = __reduce_add_sync(0xffffffffu, count);
      if (count >= need) {
        lo = mid;
        if (count <= need + need / 4 + 2) break;
      } else {
        hi = mid - 1;
      }
    }
    float edge = of_key(lo);
    if (BIAS) edge = fmaxf(edge - 2.f * key_error(p, edge, inv_total), -FLT_MAX);       // what may yet turn out to reach the bound
    const uint32_t from = to_key(edge);
    int runs = 0;
    for (int i = 0; i < chunks; ++i) {
      const bool hit = tops[i * 32 + lane] >= from;
      const uint32_t votes = __ballot_sync(0xffffffffu, hit);
      const int pos = runs + __popc(votes & ((1u << lane) - 1u));
      if (hit && pos < kStreamHits) s.hits[pos] = static_cast<uint16_t>(i * 32 + lane);
      runs += __popc(votes);
    }
    __syncwarp();
    sure = runs <= kStreamHits && edge < INFINITY;
    if (sure) {
      constexpr int kFlight = 4;
      for (int h = 0; h < runs; h += kFlight * 32 / S) {
        float z[kFlight], add[kFlight];
        int id[kFlight];
#pragma unroll
        for (int q = 0; q < kFlight; ++q) {
          const int j = h + q * (32 / S) + lane / S;
          const int run = j < runs ? s.hits[j] : 0, i = run >> 5;
          const int bt = i / kRuns, g = GROUPS ? div_of(bt, group_batches) : 0;
          const int c = ((bt - g * batches) * kBatch + (i - bt * kRuns) * S + lane % S) * 32 + (run & 31);     // within the group
          const bool real = j < runs && c < per;
          id[q] = g * per + c;
          z[q] = real ? logit_of(zr, id[q]) : -INFINITY;
          add[q] = BIAS && real ? bias[id[q]] : 0.f;
        }
#pragma unroll
        for (int q = 0; q < kFlight; ++q) {
          const float v = stream_key<SIG, BIAS>(z[q], add[q], m, inv_total);
          const bool in = v >= edge && v > -INFINITY;
          const uint32_t votes = __ballot_sync(0xffffffffu, in);
          const int pos = n + __popc(votes & ((1u << lane) - 1u));
          if (in && pos < kStreamCand) s.cand[pos] = static_cast<unsigned long long>(to_key(v)) << 32 | ~static_cast<uint32_t>(id[q]);
          n += __popc(votes);
        }
      }
      __syncwarp();
      sure = n <= kStreamCand;
    }
  }
  if (sure && some > 0) {
    if (n > need + 16) {                               // a closer bound, from the candidates themselves
      uint32_t key[kStreamCand / 32];
      uint32_t l = 0xFFFFFFFFu, u = 0;
#pragma unroll
      for (int q = 0; q < kStreamCand / 32; ++q) {
        key[q] = lane + 32 * q < n ? static_cast<uint32_t>(s.cand[lane + 32 * q] >> 32) : 0u;
        u = max(u, key[q]);
        if (key[q] != 0) l = min(l, key[q]);
      }
      u = __reduce_max_sync(0xffffffffu, u);
      l = __reduce_min_sync(0xffffffffu, l);
      while (l < u) {
        const uint32_t mid = l + (u - l + 1) / 2;
        int count = 0;
#pragma unroll
        for (int q = 0; q < kStreamCand / 32; ++q) count += key[q] >= mid;
        count = __reduce_add_sync(0xffffffffu, count);
        if (count >= need) {
          l = mid;
          if (count <= need + 4) break;
        } else {
          u = mid - 1;
        }
      }
      float edge = of_key(l);
      if (BIAS) edge -= 2.f * key_error(p, edge, inv_total);
      const uint32_t from = to_key(edge);
      int left = 0;
#pragma unroll
      for (int q = 0; q < kStreamCand / 32; ++q) {
        const unsigned long long mine = lane + 32 * q < n ? s.cand[lane + 32 * q] : 0;
        const bool in = key[q] >= from;
        const uint32_t votes = __ballot_sync(0xffffffffu, in);        // (every lane has read its entry of this round)
        if (in) s.cand[left + __popc(votes & ((1u << lane) - 1u))] = mine;
        left += __popc(votes);
        __syncwarp();
      }
      n = left;
    }
    for (int t = lane; t < n; t += 32) {
      const unsigned long long mine = s.cand[t];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) rank += s.cand[j] > mine;
      if (BIAS) s.wide[rank] = mine;                   // in order
      if (rank < p.k) s.place[rank] = static_cast<int>(~static_cast<uint32_t>(mine));
    }
    __syncwarp();
    if (n < p.k) fill_up(s.place, n, p.k);
    bool close = false;
    if (BIAS) {
      __syncwarp();
      for (int t = lane; t < p.k && t + 1 < n; t += 32)
        if (!apart(p, of_key(static_cast<uint32_t>(s.wide[t] >> 32)), of_key(static_cast<uint32_t>(s.wide[t + 1] >> 32)), inv_total)) close = true;
      __syncwarp();
    }
    if (BIAS && __any_sync(0xffffffffu, close)) {      // again by 64-bit keys
      double t64 = total;
#pragma unroll 1
      for (int round = 0; round < 2; ++round) {
        for (int t = lane; t < n; t += 32) s.wide[t] = key64(p, zr, static_cast<int>(~static_cast<uint32_t>(s.cand[t])), m, t64, false);
        __syncwarp();
        if (!__any_sync(0xffffffffu, rank_wide(p, s.cand, s.wide, n, lane, 32, s.place)) || round > 0) break;
        t64 = warp_total(total64(zr, p.N, m, lane, 32));
      }
    }
  } else if (!sure) {
    __syncwarp();
    choose_warp64(p, zr, m, s.list);
    for (int j = lane; j < p.k; j += 32) s.place[j] = chosen_from(s.list.key[j]) ? s.list.id[j] : ~s.list.id[j];
  }
  __syncwarp();
  write_row<kStreamMostK / 32>(p, row, m, total, [&](int j, bool& good, float& logit) {
    const int at = s.place[j], id = at >= 0 ? at : ~at;
    good = at >= 0;
    logit = logit_of(zr, id);
    return id;
  });
}

// ---- a CTA a row -----------------------------------------------------------------------------
template <typename K, int TH> __device__ __forceinline__ K cta_total(K v, K* red) {
  v = warp_total(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_total((threadIdx.x & 31) < TH / 32 ? red[threadIdx.x & 31] : K(0));
}
struct CtaShared {
  unsigned long long cand[kSelCand];       // key, then the id's complement: larger is earlier
  int place[kMostK];                       // the picks in order; negative: filled up
  uint64_t group[kMostGroups];
  unsigned long long kept;
  double red[32];
  uint64_t most[32];
  int count, unsure, close;
  float edge;
};

// The groups that stay, from 64-bit keys of all candidates in shared memory.
template <int TH>
__device__ __noinline__ void choose_groups64(const SelectParams& p, CtaShared& s, const uint64_t* keys) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int g = warp; g < p.groups; g += TH / 32) {
    Best2<uint64_t> t{0, 0};
    for (int c = g * p.per + lane; c < (g + 1) * p.per; c += 32) take(t, keys[c]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t a = __shfl_xor_sync(0xffffffffu, t.a, o), b = __shfl_xor_sync(0xffffffffu, t.b, o);
      take(t, a);
      take(t, b);
    }
    if (lane == 0) s.group[g] = group_value(p, t);
  }
  __syncthreads();
  if (warp == 0) {
    uint32_t lo = 0, hi = 0;
    for (int g = lane; g < p.groups; g += 32) {
      const uint64_t mine = s.group[g];
      int rank = 0;
      for (int o = 0; o < p.groups; ++o) rank += s.group[o] > mine || (s.group[o] == mine && o < g);
      if (rank < p.keep) { if (g < 32) lo |= 1u << g; else hi |= 1u << (g - 32); }
    }
    lo = __reduce_or_sync(0xffffffffu, lo);
    hi = __reduce_or_sync(0xffffffffu, hi);
    if (lane == 0) s.kept = static_cast<unsigned long long>(hi) << 32 | lo;
  }
  __syncthreads();
}
// The same from fp32 keys, 64 bits where those close: 0 for a group that stays and -inf for one that goes, behind the values.
template <int TH, typename LT>
__device__ __forceinline__ void choose_groups(const SelectParams& p, CtaShared& s, const float* keys, const LT* z, float m, float inv_total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* values = reinterpret_cast<float*>(s.group);
  for (int g = warp; g < p.groups; g += TH / 32) {
    float a = -INFINITY, b = -INFINITY;
#pragma unroll 4
    for (int c = g * p.per + lane; c < (g + 1) * p.per; c += 32) {
      const float v = keys[c];
      b = fmaxf(b, fminf(a, v));
      a = fmaxf(a, v);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
      b = fmaxf(fminf(a, oa), fmaxf(b, ob));
      a = fmaxf(a, oa);
    }
    if (lane == 0) values[g] = p.top2 && b > -INFINITY ? a + b : a;
  }
  __syncthreads();
  if (warp == 0) {
    float least = INFINITY, most = -INFINITY;
    for (int g = lane; g < p.groups; g += 32) {
      const float mine = values[g];
      int rank = 0;
      for (int o = 0; o < p.groups; ++o) rank += values[o] > mine || (values[o] == mine && o < g);
      values[kMostGroups + g] = rank < p.keep ? 0.f : -INFINITY;
      if (rank < p.keep) least = fminf(least, mine);
      else most = fmaxf(most, mine);
    }
    least = of_key(__reduce_min_sync(0xffffffffu, to_key(least)));
    most = of_key(__reduce_max_sync(0xffffffffu, to_key(most)));
    if (!groups_apart(p, least, most, inv_total)) {
      const unsigned long long kept = choose_groups_near(p, z, lane < p.groups ? values[lane] : -INFINITY,
                                                         lane + 32 < p.groups ? values[lane + 32] : -INFINITY, least, most, m, inv_total);
      for (int g = lane; g < p.groups; g += 32) values[kMostGroups + g] = kept >> g & 1 ? 0.f : -INFINITY;
    }
  }
  __syncthreads();
}

// The whole selection by 64-bit keys in shared memory: any row, at the cost of two barriers a pick.
template <typename LT, int TH>
__device__ __noinline__ void choose_cta64(const SelectParams& p, CtaShared& s, uint64_t* keys, const LT* zr, float m) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double total = 1.0;
  if (!p.sigmoid) total = cta_total<double, TH>(total64(zr, p.N, m, threadIdx.x, TH), s.red);
  __syncthreads();
  unsigned long long kept = ~0ull;
  if (p.keep < p.groups) {
#pragma unroll 1
    for (int c = threadIdx.x; c < p.N; c += TH) keys[c] = key64(p, zr, c, m, total, true);
    __syncthreads();
    choose_groups64<TH>(p, s, keys);
    kept = s.kept;
  }
#pragma unroll 1
  for (int c = threadIdx.x; c < p.N; c += TH)
    keys[c] = kept >> (div_of(c, p.per_group) & 63) & 1 ? key64(p, zr, c, m, total, false) : static_cast<uint64_t>(kFiller - c);
  // (a thread reads and clears its own columns alone)
  uint64_t best = 0;
  int at = 0;
  for (int c = threadIdx.x; c < p.N; c += TH)
    if (keys[c] > best) { best = keys[c]; at = c; }
  for (int t = 0; t < p.k; ++t) {
    const uint64_t top = warp_most(best);
    const uint32_t id = __reduce_min_sync(0xffffffffu, best == top ? static_cast<uint32_t>(at) : 0xFFFFFFFFu);
    if (lane == 0) { s.most[warp] = top; s.cand[warp] = id; }
    __syncthreads();
    uint64_t all = 0;
    uint32_t first = 0xFFFFFFFFu;
    for (int w = 0; w < TH / 32; ++w) {
      const uint64_t v = s.most[w];
      const uint32_t i = static_cast<uint32_t>(s.cand[w]);
      if (v > all || (v == all && i < first)) { all = v; first = i; }
    }
    if (threadIdx.x == 0) s.place[t] = chosen_from(all) ? static_cast<int>(first) : ~static_cast<int>(first);
    if (at == static_cast<int>(first) && best == all) {
      keys[at] = 0;
      best = 0;
      for (int c = threadIdx.x; c < p.N; c += TH)
        if (keys[c] > best) { best = keys[c]; at = c; }
    }
    __syncthreads();
  }
}

template <typename LT, int NV, int TH>
__global__ void __launch_bounds__(TH, TH == 256 ? 5 : 1)
select_cta_kernel(const SelectParams p) {
  extern __shared__ uint64_t keys[];       // [N]: 64-bit keys of an unsure row, or fp32 keys for the groups
  __shared__ CtaShared s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = blockIdx.x;
  if (p.count_here)                        // (many barriers before the first count)
    for (int c = threadIdx.x; c < p.S + p.N; c += TH) p.load[c] = 0;
  const LT* zr = static_cast<const LT*>(p.logits) + row * p.ld + p.S;
  const bool biased = p.bias != nullptr, grouped = p.keep < p.groups, judged = grouped && p.top2 && !biased;
  const float* b = biased ? p.bias + p.S : nullptr;
  float* sk = reinterpret_cast<float*>(keys);
  float v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] = threadIdx.x + TH * i < p.N ? logit_of(zr, threadIdx.x + TH * i) : -INFINITY;
  if (threadIdx.x == 0) { s.count = 0; s.unsure = 0; s.close = 0; }
  float m = 0.f, total = 1.f, inv_total = 1.f;
  if (p.sigmoid) {
    if (biased || judged) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = threadIdx.x + TH * i;
        const float sc = masked(v[i]) ? -INFINITY : fast_sigmoid(v[i]);
        if (judged && c < p.N) sk[c] = sc;
        if (biased && c < p.N) v[i] = sc + b[c];
      }
    }
  } else {
    m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i) m = fmaxf(m, v[i]);
    m = of_key(__reduce_max_sync(0xffffffffu, to_key(m)));
    float* red = reinterpret_cast<float*>(s.most);
    if (lane == 0) red[warp] = m;
    __syncthreads();
    m = of_key(__reduce_max_sync(0xffffffffu, to_key(red[lane < TH / 32 ? lane : 0])));
    total = 0.f;
    if (biased || judged) {                    // the exponentials become the keys
      float e[NV];
#pragma unroll
      for (int i = 0; i < NV; ++i) { e[i] = masked(v[i]) ? 0.f : expf(v[i] - m); total += e[i]; }
      total = cta_total<float, TH>(total, reinterpret_cast<float*>(s.red));
      if (total == 0.f) total = 1.f;
      inv_total = 1.f / total;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = threadIdx.x + TH * i;
        const float sc = masked(v[i]) ? -INFINITY : e[i] * inv_total;
        if (judged && c < p.N) sk[c] = sc;
        if (biased && c < p.N) v[i] = sc + b[c];
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) total += masked(v[i]) ? 0.f : expf(v[i] - m);
      total = cta_total<float, TH>(total, reinterpret_cast<float*>(s.red));
      if (total == 0.f) total = 1.f;
      inv_total = 1.f / total;
    }
  }
  if (!biased) {
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = masked(v[i]) ? -INFINITY : v[i];
  }
  if (grouped) {
    if (!judged) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (threadIdx.x + TH * i < p.N) sk[threadIdx.x + TH * i] = v[i];
    }
    __syncthreads();
    choose_groups<TH>(p, s, sk, zr, m, inv_total);
    const float* off = reinterpret_cast<const float*>(s.group) + kMostGroups;          // 0 where the group stays, else -inf
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (threadIdx.x + TH * i < p.N) v[i] += off[div_of(threadIdx.x + TH * i, p.per_group)];     // (NaN stays)
  }
  // A bound that at least k + 1 of the threads' own maxima reach, and few more.
  float* tops = reinterpret_cast<float*>(s.cand);          // [TH] <= kSelCand * 2
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i) top = max_nan(top, v[i]);
  tops[threadIdx.x] = top;
  __syncthreads();
  const int need = p.need;
  if (warp == 0) {
    uint32_t key[TH / 32], lo = 0xFFFFFFFFu, hi = 0;
    constexpr uint32_t kNone = 0x007FFFFFu;                // of -inf
    int some = 0;
#pragma unroll
    for (int i = 0; i < TH / 32; ++i) {
      key[i] = to_key(tops[lane + 32 * i]);
      hi = max(hi, key[i]);
      if (key[i] > kNone) { ++some; lo = min(lo, key[i]); }
    }
    some = __reduce_add_sync(0xffffffffu, some);
    hi = __reduce_max_sync(0xffffffffu, hi);
    lo = __reduce_min_sync(0xffffffffu, lo);
    if (hi == 0xFFFFFFFFu) {                               // NaN
      if (lane == 0) s.unsure = 1;
    } else if (some < need) {                              // candidates in few threads (masks): all of them (the lowest finite number's key)
      lo = 0x00800000u;
    } else if (some > 0) {
      // count(>= lo) >= need, count(> hi) == 0
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        int n = 0;
#pragma unroll
        for (int i = 0; i < TH / 32; ++i) n += key[i] >= mid;
        n = __reduce_add_sync(0xffffffffu, n);
        if (n >= need) {
          lo = mid;
          if (n <= need + need / 2 + 8) break;
        } else {
          hi = mid - 1;
        }
      }
    }
    // (with a bias: what may yet turn out to reach the bound)
    const float e = some > 0 ? of_key(lo) : INFINITY;
    if (lane == 0) {
      s.edge = biased && some > 0 ? fmaxf(e - 2.f * key_error(p, e, inv_total), -FLT_MAX) : e;
      if (some > 0 && !(s.edge < INFINITY)) s.unsure = 1;          // (more infinite keys than places)
    }
    if (some == 0)
      for (int j = lane; j < p.k; j += 32) s.place[j] = ~j;        // nothing to choose from: the lowest ids
  }
  __syncthreads();
  const float edge = s.edge;
  bool sure = !s.unsure;
  if (sure && edge < INFINITY) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (v[i] >= edge) {
        const int pos = atomicAdd(&s.count, 1);
        if (pos < kSelCand)
          s.cand[pos] = static_cast<unsigned long long>(to_key(v[i])) << 32 | ~static_cast<uint32_t>(threadIdx.x + TH * i);
      }
    }
    __syncthreads();
    const int n = s.count;
    sure = n <= kSelCand;
    if (sure) {
      for (int t = threadIdx.x; t < n; t += TH) {
        const unsigned long long mine = s.cand[t];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank += s.cand[j] > mine;
        if (biased) keys[rank] = mine;              // in order
        if (rank < p.k) s.place[rank] = static_cast<int>(~static_cast<uint32_t>(mine));
      }
      __syncthreads();
      if (biased)
        for (int t = threadIdx.x; t < p.k && t + 1 < n; t += TH)
          if (!apart(p, of_key(static_cast<uint32_t>(keys[t] >> 32)), of_key(static_cast<uint32_t>(keys[t + 1] >> 32)), inv_total)) s.close = 1;
      if (warp == 0 && n < p.k) fill_up(s.place, n, p.k);
      __syncthreads();
      if (s.close) {                                // the candidates again by 64-bit keys
        double t64 = total;
#pragma unroll 1
        for (int round = 0; round < 2; ++round) {
          for (int t = threadIdx.x; t < n; t += TH) keys[t] = key64(p, zr, static_cast<int>(~static_cast<uint32_t>(s.cand[t])), m, t64, false);
          __syncthreads();
          if (!__syncthreads_or(rank_wide(p, s.cand, keys, n, threadIdx.x, TH, s.place)) || round > 0) break;
          t64 = cta_total<double, TH>(total64(zr, p.N, m, threadIdx.x, TH), s.red);
        }
      }
    }
  }
  if (!sure) {                       // (the same for every thread)
    __syncthreads();
    choose_cta64<LT, TH>(p, s, keys, zr, m);
  }
  if (warp == 0) {
    write_row<kMostK / 32>(p, row, m, total, [&](int j, bool& good, float& logit) {
      const int at = s.place[j], id = at >= 0 ? at : ~at;
      good = at >= 0;
      logit = logit_of(zr, id);
      return id;
    });
  }
}

// ---- backward --------------------------------------------------------------------------------
// d_z of a row is zero but at the picks, except where the scores' own sum stays in the weights (softmax scores that are not
// renormalised, or whose sum was clamped): then d_z = p (ds - sum ds p).  Bound by the bytes of d_z.
struct SelectGrads {
  const void* logits;
  const long long* idx;
  const float *weights, *comb_w, *row_stats, *g_weights, *g_comb;
  void* d_logits;
  long long ld;
  int rows, C, S, k, sigmoid, renorm;
  float rho;
};
template <typename LT, int TH>
__global__ void __launch_bounds__(TH == 32 ? 32 * kWarpRows : TH)
select_bwd_kernel(const SelectGrads p) {
  const int tid = TH == 32 ? threadIdx.x & 31 : threadIdx.x, lane = threadIdx.x & 31;
  const long long row = TH == 32 ? static_cast<long long>(blockIdx.x) * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= p.rows) return;
  const LT* z = static_cast<const LT*>(p.logits) + row * p.ld;
  LT* dz = static_cast<LT*>(p.d_logits) + row * p.C;
  const float4 st = reinterpret_cast<const float4*>(p.row_stats)[row];         // largest logit, sum, chosen mass, joint mass
  // every warp forms the row's few sums for itself
  constexpr int kEach = kMostK / 32;
  const float joint = max_nan(st.w, 1e-12f);
  float along = 0.f;                          // sum over the joint list of g * joint weight
  if (p.g_comb != nullptr && p.S > 0)
    for (int j = lane; j < p.S + p.k; j += 32) along = fmaf(p.g_comb[row * (p.S + p.k) + j], p.comb_w[row * (p.S + p.k) + j], along);
  along = warp_total(along);
  float ds[kEach], sc[kEach], dot = 0.f;
  int id[kEach];
#pragma unroll
  for (int q = 0; q < kEach; ++q) {
    const int j = lane + 32 * q;
    ds[q] = sc[q] = 0.f;
    id[q] = 0;
    if (j >= p.k) continue;
    const long long chosen = p.idx[row * p.k + j];
    id[q] = chosen >= p.S && chosen < p.C ? static_cast<int>(chosen) : -1;          // (no chapter: no gradient)
    float g = p.g_weights != nullptr ? p.g_weights[row * p.k + j] : 0.f;
    if (p.g_comb != nullptr) {
      const float gc = p.g_comb[row * (p.S + p.k) + p.S + j];
      g += p.S > 0 ? p.rho * (gc - along) / joint : gc;
    }
    ds[q] = g;
    dot = fmaf(g, p.weights[row * p.k + j], dot);
  }
  dot = warp_total(dot);
  const bool clamped = p.renorm && st.z <= 1e-12f;
  const bool dense = !p.sigmoid && (!p.renorm || clamped);
  float lean = 0.f;
#pragma unroll
  for (int q = 0; q < kEach; ++q) {
    const int j = lane + 32 * q;
    if (j >= p.k) continue;
    // (a place that was filled up has weight 0 and no score; a chosen score that underflowed to 0 has no gradient either)
    const bool live = p.weights[row * p.k + j] != 0.f && id[q] >= 0;
    const float v = logit_of(z, max(id[q], 0));
    sc[q] = !live ? 0.f : p.sigmoid ? 1.f / (1.f + expf(-v)) : expf(v - st.x) / st.y;
    ds[q] = !live ? 0.f : !p.renorm ? ds[q] : clamped ? ds[q] * 1e12f : (ds[q] - dot) / st.z;
    lean = fmaf(ds[q], sc[q], lean);
  }
  lean = dense ? warp_total(lean) : 0.f;
  if (dense) {
#pragma unroll 4
    for (int c = tid; c < p.C; c += TH) {
      const float v = logit_of(z, c);
      store_logit(dz, c, c < p.S || masked(v) ? 0.f : -(expf(v - st.x) / st.y) * lean);
    }
  } else {
#pragma unroll 4
    for (int c = tid; c < p.C; c += TH) store_logit(dz, c, 0.f);
  }
  if constexpr (TH == 32) __syncwarp(); else __syncthreads();
  if (tid >= 32) return;
#pragma unroll
  for (int q = 0; q < kEach; ++q)
    if (lane + 32 * q < p.k && sc[q] != 0.f) {
      // 1 - s of a sigmoid near 1 from the other exponential
      const float v = logit_of(z, id[q]);
      const float slope = p.sigmoid ? sc[q] * (1.f / (1.f + expf(v))) : sc[q];
      store_logit(dz, id[q], p.sigmoid ? ds[q] * slope : slope * (ds[q] - lean));
    }
}

// load[c] = how many of the `n` picks are c (with `weights`: of those whose weight is not 0), by one cluster of kLoadCtas CTAs: each
// counts its share in shared memory, then adds up a share of the chapters over all of them.  (Counted by the selecting CTAs with atomics in global memory, 65,536 picks among 64
// chapters took 30 us: the counters share two cache lines.)
constexpr int kLoadCtas = 8;
__global__ void __launch_bounds__(1024)
select_load_kernel(const long long* __restrict__ idx, const float* __restrict__ weights, long long n, int C, int* __restrict__ load) {
  extern __shared__ int counts[];          // [C]
  const int rank = blockIdx.x;
  for (int c = threadIdx.x; c < C; c += 1024) counts[c] = 0;
  __syncthreads();
#pragma unroll 4
  for (long long i = rank * 1024 + threadIdx.x; i < n; i += kLoadCtas * 1024) {
    const unsigned long long c = static_cast<unsigned long long>(idx[i]);
    if (c >= static_cast<unsigned long long>(C) || (weights != nullptr && weights[i] == 0.f)) continue;
    atomicAdd(counts + static_cast<int>(c), 1);
  }
  cluster_sync();
  const uint32_t base = smem_u32(counts);
  for (int c = rank * 1024 + threadIdx.x; c < C; c += kLoadCtas * 1024) {
    int sum = 0;
#pragma unroll
    for (int r = 0; r < kLoadCtas; ++r) {
      int v;
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(cluster_map(base + c * 4, r)));
      sum += v;
    }
    load[c] = sum;
  }
  cluster_sync();                          // nobody leaves while its counts are read
}

__global__ void balance_bias_kernel(float* __restrict__ bias, const int* __restrict__ load, int C, int S, float rate) {
  __shared__ double red[32];
  double n = 0.0;
  for (int c = S + threadIdx.x; c < C; c += blockDim.x) n += load[c];
  n = warp_total(n);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = n;
  __syncthreads();
  n = 0.0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) n += red[w];
  const double mean = n / (C - S);
  for (int c = S + threadIdx.x; c < C; c += blockDim.x) {
    const double d = mean - load[c];
    bias[c] += d > 0.0 ? rate : d < 0.0 ? -rate : 0.f;
  }
}

int check(const moc_select_shape* s) {
  MOC_REQUIRE(s != nullptr, "NULL selection shape");
  MOC_REQUIRE(s->rows > 0 && s->num_chapters > 0 && s->num_shared >= 0 && s->num_shared < s->num_chapters,
              "rows must be positive and num_shared leave a chapter to choose from");
  const int n = s->num_chapters - s->num_shared;
  MOC_REQUIRE(n <= kMostN && s->num_shared <= kMostN, "at most 16384 chapters to choose from, and as many shared ones");
  MOC_REQUIRE(s->num_groups >= 1 && s->num_groups <= kMostGroups && n % s->num_groups == 0,
              "num_groups must divide the chapters to choose from and be at most 64");
  MOC_REQUIRE(s->top_groups >= 1 && s->top_groups <= s->num_groups, "top_groups must be in 1..num_groups");
  MOC_REQUIRE(s->top_k >= 1 && s->top_k <= kMostK && s->top_k <= s->top_groups * (n / s->num_groups),
              "top_k must be in 1..128 and at most the chapters of top_groups groups");
  MOC_REQUIRE(s->score == MOC_SCORE_SOFTMAX || s->score == MOC_SCORE_SIGMOID, "score must be softmax or sigmoid");
  MOC_REQUIRE(s->dtype == MOC_F32 || s->dtype == MOC_BF16, "logits must be fp32 or bf16");
  MOC_REQUIRE(s->ld >= s->num_chapters, "rows of logits overlap");
  return MOC_OK;
}

template <typename LT, int S> int select_stream(const SelectParams& p, cudaStream_t stream) {
  const bool grouped = p.keep < p.groups, biased = p.bias != nullptr;
  const int per = grouped ? p.per : p.N;
  const int batches = ceil_div(per, 32 * kBatch), chunks = (grouped ? p.groups : 1) * batches * (kBatch / S);
  auto kern = grouped ? (p.sigmoid ? (biased ? select_stream_kernel<LT, S, true, true, true> : select_stream_kernel<LT, S, true, false, true>)
                                   : (biased ? select_stream_kernel<LT, S, false, true, true> : select_stream_kernel<LT, S, false, false, true>))
                      : (p.sigmoid ? (biased ? select_stream_kernel<LT, S, true, true, false> : select_stream_kernel<LT, S, true, false, false>)
                                   : (biased ? select_stream_kernel<LT, S, false, true, false> : select_stream_kernel<LT, S, false, false, false>));
  const size_t bytes = static_cast<size_t>(kWarpRows) * chunks * 128;
  MOC_CUDA_OK(allow_shared(kern, bytes, 128 * 1024));
  kern<<<ceil_div(p.rows, kWarpRows), 32 * kWarpRows, bytes, stream>>>(p, chunks, fast_div(batches));
  MOC_CUDA_OK(cudaGetLastError());
  return MOC_OK;
}
// Runs of `size` candidates of the groups that stay, at least.  Streaming takes its bound from their maxima and needs as many as
// values that are to reach it: 2,000 rows, one of 8 groups of 512 kept (32 runs), sigmoid, bias: k = 28 37 us against 62 by a CTA a row,
// k = 32 (a 33rd is needed) 225 against 62; two kept (64 runs): k = 48 45 against 67, k = 64 336 against 71.
// Runs of 4 up to 2,048 chapters, of 16 beyond (3,000 rows, us, 4 / 16): 1,024 chapters k = 8 20 / 20, k = 64 51 / 63; 2,048 k = 8 plain
// softmax 29 / 25, k = 32 31 / 29, k = 64 sigmoid with a bias 53 / 61; 4,096 k = 8 43 / 35, k = 32 44 / 39, k = 64 64 / 68.
int kept_runs(const SelectParams& p, int size) { return p.keep * 32 * ceil_div(p.per / 32, size); }
template <typename LT> int select_fwd(const SelectParams& p, cudaStream_t stream) {
  const bool grouped = p.keep < p.groups;
  if (p.N <= kWarpMostN && p.k <= kWarpMostK) {
    auto kern = p.N <= 64 ? select_warp_kernel<LT, 2> : p.N <= 128 ? select_warp_kernel<LT, 4>
                : p.N <= 256 ? select_warp_kernel<LT, 8> : select_warp_kernel<LT, 16>;
    kern<<<ceil_div(p.rows, kWarpRows), 32 * kWarpRows, 0, stream>>>(p);
  } else if (p.rows >= (p.k <= 32 ? kStreamRows : kStreamRowsManyPicks) && p.k <= kStreamMostK && p.N > kWarpMostN && (!grouped || p.per >= 256) &&
             kept_runs(p, p.N > 2048 ? 16 : 4) >= p.need) {
    return p.N > 2048 ? select_stream<LT, 16>(p, stream) : select_stream<LT, 4>(p, stream);
  } else {
    // 1,024 threads where 256 with 16 logits each do not hold a row (us, 256 / 1,024 threads, k = 16: 1,024 chapters 1 row 8.3 / 12.4, 500 rows 19 / 45;
    // 4,096 chapters 1 row 10.4 / 12.4, 148 rows 21 / 25, 500 rows 26 / 53).  The 48 registers of five CTAs an SM spill: 170 to 470 bytes a
    // thread, most of it on the way through 64-bit keys.
    const bool big = p.N > 4096;
    auto kern = p.N <= 1024 ? select_cta_kernel<LT, 4, 256> : p.N <= 2048 ? select_cta_kernel<LT, 8, 256>
                : !big ? select_cta_kernel<LT, 16, 256> : p.N <= 8192 ? select_cta_kernel<LT, 8, 1024> : select_cta_kernel<LT, 16, 1024>;
    if (big) MOC_CUDA_OK(allow_shared(kern, static_cast<size_t>(p.N) * 8, kMostN * 8));      // (48 KB need no leave)
    kern<<<p.rows, big ? 1024 : 256, static_cast<size_t>(p.N) * 8, stream>>>(p);
  }
  MOC_CUDA_OK(cudaGetLastError());
  return MOC_OK;
}
int select_load(const long long* idx, const float* weights, long long n, int C, int* load, cudaStream_t stream) {
  const size_t bytes = static_cast<size_t>(C) * sizeof(int32_t);
  if (bytes > 48 * 1024) MOC_CUDA_OK(allow_shared(select_load_kernel, bytes, kSharedMost));
  MOC_CUDA_OK(launch_clustered(select_load_kernel, dim3(kLoadCtas), 1024, static_cast<int>(bytes), kLoadCtas, stream, idx, weights, n, C, load));
  return MOC_OK;
}
template <typename LT> int select_bwd(const SelectGrads& p, cudaStream_t stream) {
  // A warp a row up to 512 chapters, a CTA beyond (us, warp / CTA): 512 chapters 8,192 rows sparse 8 / 26, dense 15 / 33, 500 rows dense 8.3 / 6.2;
  // 1,024 chapters 8,192 rows sparse 10 / 25, dense 26 / 39, but 500 rows dense 12.4 / 6.2 and 1 row dense 12.3 / 4.2; 4,096 chapters 500 rows
  // dense 35 / 9.
  if (p.C <= 512) select_bwd_kernel<LT, 32><<<ceil_div(p.rows, kWarpRows), 32 * kWarpRows, 0, stream>>>(p);
  else select_bwd_kernel<LT, 256><<<p.rows, 256, 0, stream>>>(p);
  MOC_CUDA_OK(cudaGetLastError());
  return MOC_OK;
}

}  // namespace
}  // namespace moc

using namespace moc;

extern "C" int moc_select_fwd(const moc_select_shape* s, const void* logits, const float* balance_bias, int64_t* idx, float* weights,
                              int32_t* comb_idx, float* comb_w, float* row_stats, int32_t* load, void* stream_) {
  const int rc = check(s);
  if (rc != MOC_OK) return rc;
  MOC_REQUIRE(logits && idx && weights && comb_idx && comb_w, "NULL selection buffer");
  MOC_REQUIRE((reinterpret_cast<uintptr_t>(row_stats) & 15) == 0, "row_stats must be 16-byte aligned");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  SelectParams p{};
  p.logits = logits; p.bias = balance_bias; p.idx = reinterpret_cast<long long*>(idx); p.weights = weights;
  p.comb_idx = comb_idx; p.comb_w = comb_w; p.row_stats = row_stats; p.load = load; p.ld = s->ld;
  p.rows = s->rows; p.N = s->num_chapters - s->num_shared; p.S = s->num_shared; p.k = s->top_k;
  p.groups = s->num_groups; p.keep = s->top_groups; p.per = p.N / p.groups;
  p.need = std::min(p.k + 1, p.keep * p.per);
  p.per_group = fast_div(p.per);
  p.sigmoid = s->score == MOC_SCORE_SIGMOID; p.top2 = s->group_top2 != 0; p.renorm = s->renormalize != 0; p.rho = s->routed_scale;
  const bool warps = p.N <= kWarpMostN && p.k <= kWarpMostK;
  p.count_here = load != nullptr && p.rows <= (warps ? kWarpRows : 1);
  const int done = s->dtype == MOC_F32 ? select_fwd<float>(p, stream) : select_fwd<__nv_bfloat16>(p, stream);
  if (done != MOC_OK || load == nullptr || p.count_here) return done;
  return select_load(p.idx, nullptr, static_cast<long long>(p.rows) * p.k, s->num_chapters, load, stream);
}

extern "C" int moc_select_load(const int64_t* idx, const float* weights, int64_t n, int32_t num_chapters, int32_t* load, void* stream) {
  MOC_REQUIRE(idx && load, "NULL selection buffer");
  MOC_REQUIRE(n >= 0 && num_chapters > 0 && num_chapters <= 2 * kMostN, "a count of chosen chapters takes 1..32768 chapters");
  return select_load(reinterpret_cast<const long long*>(idx), weights, n, num_chapters, load, static_cast<cudaStream_t>(stream));
}

extern "C" int moc_select_bwd(const moc_select_shape* s, const void* logits, const int64_t* idx, const float* weights,
                              const float* comb_w, const float* row_stats, const float* g_weights, const float* g_comb,
                              void* d_logits, void* stream_) {
  const int rc = check(s);
  if (rc != MOC_OK) return rc;
  MOC_REQUIRE(logits && idx && weights && comb_w && row_stats && d_logits, "NULL selection-gradient buffer");
  MOC_REQUIRE((reinterpret_cast<uintptr_t>(row_stats) & 15) == 0, "row_stats must be 16-byte aligned");
  SelectGrads p{};
  p.logits = logits; p.idx = reinterpret_cast<const long long*>(idx); p.weights = weights; p.comb_w = comb_w;
  p.row_stats = row_stats; p.g_weights = g_weights; p.g_comb = g_comb; p.d_logits = d_logits; p.ld = s->ld;
  p.rows = s->rows; p.C = s->num_chapters; p.S = s->num_shared; p.k = s->top_k;
  p.sigmoid = s->score == MOC_SCORE_SIGMOID; p.renorm = s->renormalize != 0; p.rho = s->routed_scale;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  return s->dtype == MOC_F32 ? select_bwd<float>(p, stream) : select_bwd<__nv_bfloat16>(p, stream);
}

extern "C" int moc_balance_bias_step(float* bias, const int32_t* load, int32_t num_chapters, int32_t num_shared, float rate,
                                     void* stream) {
  MOC_REQUIRE(bias && load, "NULL balance-bias buffer");
  MOC_REQUIRE(num_shared >= 0 && num_chapters > num_shared, "num_shared must leave a chapter");
  balance_bias_kernel<<<1, 1024, 0, static_cast<cudaStream_t>(stream)>>>(bias, load, num_chapters, num_shared, rate);
  MOC_CUDA_OK(cudaGetLastError());
  return MOC_OK;
}
