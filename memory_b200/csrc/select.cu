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
// quotient; neighbours in the order that are closer than those errors allow (one row in some hundreds) send the row through
// the same selection in 64 bits.  Bare logits need no arithmetic and are always sure.
//
// Bound by HBM for many rows (4 bytes a logit read), by latency for a few.  Up to 512 candidates and k <= 32 a warp has a
// row in registers and picks one after the other (two warp reductions each); beyond that a CTA has the row, and the k + 1
// largest lie among the values above a bound that one warp finds from the threads' own maxima.
#include "moc_common.cuh"

namespace moc {
namespace {

constexpr float kMaskedLogit = -3.3895313892515355e38f;      // lowest finite bfloat16
constexpr int kMostK = 128, kWarpMostK = 32, kWarpMostN = 512, kMostN = 16384, kMostGroups = 64;
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
  int sigmoid, top2, renorm;
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

__device__ __forceinline__ uint32_t warp_most(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
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

// How far fp32 keys can be off: the score's exponential (2 ulp), sums and quotient, against the largest score; the bias's addition.
// Two of them are told apart beyond twice that.
__device__ __forceinline__ float key_error(const SelectParams& p, float v, float total) {
  return (p.sigmoid ? 1e-6f : 4e-6f / total) + 2.5e-7f * fabsf(v);
}
__device__ __forceinline__ bool apart(const SelectParams& p, uint32_t above, uint32_t below, float total) {
  if (!chosen_from(below) || !chosen_from(above)) return true;
  const float a = of_key(above), b = of_key(below);
  return a - b > key_error(p, a, total) + key_error(p, b, total);      // (NaN and infinities: not apart)
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

// One row's lists, by one warp; pick(j): candidate of the j-th place and whether it may be chosen at all.
template <typename LT, typename Pick>
__device__ __forceinline__ void write_row(const SelectParams& p, long long row, const LT* z, float m, float total, Pick pick) {
  const int lane = threadIdx.x & 31;
  constexpr int kEach = kMostK / 32;
  int id[kEach];
  float w[kEach], mass = 0.f;
#pragma unroll
  for (int q = 0; q < kEach; ++q) {
    const int j = lane + 32 * q;
    id[q] = 0;
    w[q] = 0.f;
    if (j < p.k) {
      bool ok;
      id[q] = pick(j, ok);
      if (ok) w[q] = score_of<float>(p, logit_of(z, id[q]), m, total);
      mass += w[q];
    }
  }
  mass = warp_total(mass);
  const float over = max_nan(mass, 1e-12f);
  float sum = 0.f;
#pragma unroll
  for (int q = 0; q < kEach; ++q) {
    const int j = lane + 32 * q;
    if (j >= p.k) break;
    if (p.renorm) w[q] = w[q] / over;
    sum += p.rho * w[q];
    p.idx[row * p.k + j] = id[q] + p.S;
    p.weights[row * p.k + j] = w[q];
    if (p.load != nullptr) atomicAdd(p.load + p.S + id[q], 1);
  }
  sum = static_cast<float>(p.S) + warp_total(sum);
  const float joint = max_nan(sum, 1e-12f);
  int* ci = p.comb_idx + row * (p.S + p.k);
  float* cw = p.comb_w + row * (p.S + p.k);
  for (int j = lane; j < p.S; j += 32) { ci[j] = j; cw[j] = 1.f / joint; }
#pragma unroll
  for (int q = 0; q < kEach; ++q) {
    const int j = lane + 32 * q;
    if (j >= p.k) break;
    ci[p.S + j] = id[q] + p.S;
    cw[p.S + j] = p.S > 0 ? p.rho * w[q] / joint : w[q];
  }
  if (lane == 0) reinterpret_cast<float4*>(p.row_stats)[row] = make_float4(m, total, mass, sum);
}

// ---- a warp a row ----------------------------------------------------------------------------
// Lane j keeps the j-th pick.  Returns false where fp32 cannot tell neighbours apart.
template <typename K, int NV>
__device__ __forceinline__ bool choose_warp(const SelectParams& p, const float (&z)[NV], float m, K total, uint64_t* shared_keys,
                                            int& pick, bool& ok) {
  using U = typename KeyOf<K>::type;
  constexpr bool kRough = sizeof(K) == 4;
  const int lane = threadIdx.x & 31;
  U key[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = lane + 32 * i;
    key[i] = c < p.N ? candidate_key<K>(p, z[i], c, m, total, false) : U(0);
  }
  if (p.keep < p.groups) {
    U* sk = reinterpret_cast<U*>(shared_keys);           // candidate c at c + c / 32: groups of 32 columns start in different banks
    __syncwarp();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane + 32 * i;
      if (c < p.N) sk[c + (c >> 5)] = p.bias == nullptr && p.top2 ? candidate_key<K>(p, z[i], c, m, total, true) : key[i];
    }
    __syncwarp();
    // groups in rounds of 32; a group has as many lanes as fit
    unsigned long long kept = 0;
    U value[2];
    int rank[2] = {0, 0};
    const int lanes = p.groups > 16 ? 1 : p.groups > 8 ? 2 : p.groups > 4 ? 4 : p.groups > 2 ? 8 : 16;
    const int sub = lane & (lanes - 1), rounds = (p.groups * lanes + 31) / 32;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int g = (lane + 32 * r) / lanes;
      Best2<U> t{U(0), U(0)};
      if (r < rounds) {
        if (g < p.groups)
          for (int c = g * p.per + sub; c < (g + 1) * p.per; c += lanes) take(t, sk[c + (c >> 5)]);
        for (int o = lanes >> 1; o > 0; o >>= 1) {
          const U a = __shfl_xor_sync(0xffffffffu, t.a, o), b = __shfl_xor_sync(0xffffffffu, t.b, o);
          take(t, a);
          take(t, b);
        }
      }
      value[r] = r < rounds && g < p.groups ? group_value(p, t) : U(0);
    }
    for (int g = 0; g < p.groups; ++g) {
      const U other = __shfl_sync(0xffffffffu, value[(g * lanes) >> 5 & 1], (g * lanes) & 31);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int mine = (lane + 32 * r) / lanes;
        rank[r] += other > value[r] || (other == value[r] && g < mine);
      }
    }
    U least = ~U(0), most = 0;           // of those that stay and of those that go
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int g = (lane + 32 * r) / lanes;
      if (r >= rounds || g >= p.groups) continue;
      if (rank[r] < p.keep) { kept |= 1ull << g; least = min(least, value[r]); }
      else most = max(most, value[r]);
    }
    kept = static_cast<unsigned long long>(__reduce_or_sync(0xffffffffu, static_cast<uint32_t>(kept >> 32))) << 32 |
           __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(kept));
    if constexpr (kRough) {
      least = __reduce_min_sync(0xffffffffu, least);
      most = __reduce_max_sync(0xffffffffu, most);
      if ((p.bias != nullptr || p.top2) && !apart(p, least, most, total)) return false;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = lane + 32 * i;
      if (c < p.N && !(kept >> (c / p.per) & 1)) key[i] = static_cast<U>(kFiller - c);
    }
  }
  U best = 0;
  int at = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (key[i] > best) { best = key[i]; at = lane + 32 * i; }
  const bool check = kRough && p.bias != nullptr;
  const int steps = check && p.k < p.N ? p.k + 1 : p.k;
  U before = 0;
  bool sure = true;
  for (int t = 0; t < steps; ++t) {
    const U top = warp_most(best);
    const int id = static_cast<int>(__reduce_min_sync(0xffffffffu, best == top ? static_cast<uint32_t>(at) : 0xFFFFFFFFu));
    if (lane == t) { pick = id; ok = chosen_from(top); }
    if constexpr (kRough) {
      if (check && t > 0 && !apart(p, before, top, total)) { sure = false; break; }
    }
    before = top;
    if (best == top && at == id) {
      best = 0;
      at = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (lane + 32 * i == id) key[i] = 0;
        if (key[i] > best) { best = key[i]; at = lane + 32 * i; }
      }
    }
  }
  return sure;
}

template <typename LT, int NV>
__global__ void __launch_bounds__(32 * kWarpRows)
select_warp_kernel(const SelectParams p) {
  __shared__ uint64_t keys[kWarpRows][NV * 33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * kWarpRows + warp;
  if (row >= p.rows) return;
  const LT* zr = static_cast<const LT*>(p.logits) + row * p.ld + p.S;
  float z[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) z[i] = lane + 32 * i < p.N ? logit_of(zr, lane + 32 * i) : -INFINITY;
  float m = 0.f, total = 1.f;
  if (!p.sigmoid) {
    m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i) m = fmaxf(m, z[i]);
    m = warp_max(m);
    total = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) total += masked(z[i]) ? 0.f : expf(z[i] - m);
    total = warp_total(total);
    if (total == 0.f) total = 1.f;                  // (every logit masked)
  }
  int pick = 0;
  bool ok = false;
  if (!choose_warp<float, NV>(p, z, m, total, keys[warp], pick, ok)) {
    double t64 = 1.0;
    if (!p.sigmoid) {
      t64 = 0.0;
#pragma unroll 1
      for (int c = lane; c < p.N; c += 32) {
        const float v = logit_of(zr, c);
        if (!masked(v)) t64 += exp(static_cast<double>(v) - static_cast<double>(m));
      }
      t64 = warp_total(t64);
    }
    choose_warp<double, NV>(p, z, m, t64, keys[warp], pick, ok);
  }
  const unsigned live = __ballot_sync(0xffffffffu, ok);
  write_row(p, row, zr, m, total, [&](int j, bool& good) {      // (k <= 32: place j is this lane's)
    good = live >> (j & 31) & 1;
    return pick;
  });
}

// ---- a CTA a row -----------------------------------------------------------------------------
template <typename K, int TH> __device__ __forceinline__ K cta_total(K v, K* red) {
  v = warp_total(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  K t = K(0);
  for (int w = 0; w < TH / 32; ++w) t += red[w];
  return t;
}
struct CtaShared {
  unsigned long long cand[kSelCand];       // key, then the id's complement: larger is earlier
  int place[kMostK];                       // the picks in order; negative: filled up
  uint64_t group[kMostGroups];
  unsigned long long kept;
  double red[32];
  uint64_t most[32];
  int count, unsure;
  uint32_t edge;
};

// Which groups stay; keys of all candidates in shared memory.  false: fp32 cannot tell.
template <typename K, int TH>
__device__ __forceinline__ bool choose_groups(const SelectParams& p, CtaShared& s, const typename KeyOf<K>::type* keys, float total) {
  using U = typename KeyOf<K>::type;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int g = warp; g < p.groups; g += TH / 32) {
    Best2<U> t{U(0), U(0)};
    for (int c = g * p.per + lane; c < (g + 1) * p.per; c += 32) take(t, keys[c]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const U a = __shfl_xor_sync(0xffffffffu, t.a, o), b = __shfl_xor_sync(0xffffffffu, t.b, o);
      take(t, a);
      take(t, b);
    }
    if (lane == 0) s.group[g] = group_value(p, t);
  }
  __syncthreads();
  if (warp == 0) {
    unsigned long long kept = 0;
    U least = ~U(0), most = 0;
    for (int g = lane; g < p.groups; g += 32) {
      const U mine = static_cast<U>(s.group[g]);
      int rank = 0;
      for (int o = 0; o < p.groups; ++o) {
        const U other = static_cast<U>(s.group[o]);
        rank += other > mine || (other == mine && o < g);
      }
      if (rank < p.keep) { kept |= 1ull << g; least = min(least, mine); }
      else most = max(most, mine);
    }
    kept = static_cast<unsigned long long>(__reduce_or_sync(0xffffffffu, static_cast<uint32_t>(kept >> 32))) << 32 |
           __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(kept));
    bool sure = true;
    if constexpr (sizeof(K) == 4) {
      least = __reduce_min_sync(0xffffffffu, least);
      most = __reduce_max_sync(0xffffffffu, most);
      sure = !(p.bias != nullptr || p.top2) || apart(p, least, most, total);
    }
    if (lane == 0) { s.kept = kept; s.unsure = !sure; }
  }
  __syncthreads();
  return !s.unsure;
}

// The picks one after the other from 64-bit keys in shared memory: any row, at the cost of two barriers a pick.
template <int TH>
__device__ __forceinline__ void choose_slowly(const SelectParams& p, CtaShared& s, uint64_t* keys) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
__global__ void __launch_bounds__(TH)
select_cta_kernel(const SelectParams p) {
  extern __shared__ uint64_t keys[];       // [N]: 64-bit keys of an unsure row, or 32-bit keys for the groups
  __shared__ CtaShared s;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = blockIdx.x;
  const LT* zr = static_cast<const LT*>(p.logits) + row * p.ld + p.S;
  float z[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) z[i] = threadIdx.x + TH * i < p.N ? logit_of(zr, threadIdx.x + TH * i) : -INFINITY;
  float m = 0.f, total = 1.f;
  if (!p.sigmoid) {
    m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i) m = fmaxf(m, z[i]);
    m = warp_max(m);
    float* red = reinterpret_cast<float*>(s.most);
    if (lane == 0) red[warp] = m;
    __syncthreads();
    m = warp_max(red[lane < TH / 32 ? lane : 0]);
    total = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) total += masked(z[i]) ? 0.f : expf(z[i] - m);
    total = cta_total<float, TH>(total, reinterpret_cast<float*>(s.red));
    if (total == 0.f) total = 1.f;
  }
  const bool exact = p.bias == nullptr;
  bool sure = true;
  uint32_t key[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = threadIdx.x + TH * i;
    key[i] = c < p.N ? candidate_key<float>(p, z[i], c, m, total, false) : 0u;
  }
  if (p.keep < p.groups) {
    uint32_t* k32 = reinterpret_cast<uint32_t*>(keys);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = threadIdx.x + TH * i;
      if (c < p.N) k32[c] = exact && p.top2 ? candidate_key<float>(p, z[i], c, m, total, true) : key[i];
    }
    __syncthreads();
    sure = choose_groups<float, TH>(p, s, k32, total);
    const unsigned long long kept = s.kept;
    if (sure) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = threadIdx.x + TH * i;
        if (c < p.N && !(kept >> (c / p.per) & 1)) key[i] = kFiller - c;
      }
    }
  }
  if (sure) {
    // A bound that at least k + 1 of the threads' own maxima reach (all of them where there are no more candidates), and few more.
    uint32_t* tops = reinterpret_cast<uint32_t*>(s.cand);          // [TH] <= kSelCand * 2
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) top = max(top, key[i]);
    tops[threadIdx.x] = top;
    if (threadIdx.x == 0) { s.count = 0; s.unsure = 0; }
    __syncthreads();
    const int need = min(p.k + 1, min(p.N, TH));
    if (warp == 0) {
      uint32_t v[TH / 32];
      uint32_t lo = 0xFFFFFFFFu, hi = 0;
#pragma unroll
      for (int i = 0; i < TH / 32; ++i) {
        v[i] = tops[lane + 32 * i];
        hi = max(hi, v[i]);
        lo = min(lo, v[i]);
      }
      hi = __reduce_max_sync(0xffffffffu, hi);
      lo = __reduce_min_sync(0xffffffffu, lo);
      // count(>= lo) >= need, count(> hi) == 0
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo + 1) / 2;
        int n = 0;
#pragma unroll
        for (int i = 0; i < TH / 32; ++i) n += v[i] >= mid;
        n = __reduce_add_sync(0xffffffffu, n);
        if (n >= need) {
          lo = mid;
          if (n <= need + need / 2 + 8) break;
        } else {
          hi = mid - 1;
        }
      }
      if (lo == 0) lo = 1;                                    // (threads without a candidate)
      if (!exact && chosen_from(lo)) {                        // what may yet turn out to reach the bound
        const float e = of_key(lo);
        lo = min(lo, to_key(e - 2.f * key_error(p, e, total)));
      }
      if (lane == 0) s.edge = lo;
    }
    __syncthreads();
    const uint32_t edge = s.edge;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (key[i] >= edge) {
        const int pos = atomicAdd(&s.count, 1);
        if (pos < kSelCand) s.cand[pos] = static_cast<unsigned long long>(key[i]) << 32 | ~static_cast<uint32_t>(threadIdx.x + TH * i);
      }
    }
    __syncthreads();
    const int n = s.count;
    sure = n <= kSelCand;
    if (sure) {
      for (int t = threadIdx.x; t < n; t += TH) {
        const unsigned long long mine = s.cand[t];
        unsigned long long next = 0;                // the largest below it
        int rank = 0;
        for (int j = 0; j < n; ++j) {
          const unsigned long long o = s.cand[j];
          rank += o > mine;
          if (o < mine && o > next) next = o;
        }
        if (rank < p.k) {
          const uint32_t k32 = static_cast<uint32_t>(mine >> 32);
          const int id = static_cast<int>(~static_cast<uint32_t>(mine));
          s.place[rank] = chosen_from(k32) ? id : ~id;
          if (!exact && next != 0 && !apart(p, k32, static_cast<uint32_t>(next >> 32), total)) s.unsure = 1;
        }
      }
      __syncthreads();
      sure = !s.unsure;
    }
  }
  if (!sure) {                       // (the same for every thread)
    double t64 = 1.0;
    if (!p.sigmoid) {
      t64 = 0.0;
#pragma unroll 1
      for (int c = threadIdx.x; c < p.N; c += TH) {
        const float v = logit_of(zr, c);
        if (!masked(v)) t64 += exp(static_cast<double>(v) - static_cast<double>(m));
      }
      t64 = cta_total<double, TH>(t64, s.red);
    }
    __syncthreads();
#pragma unroll 1
    for (int pass = p.keep < p.groups ? 0 : 1; pass < 2; ++pass) {
#pragma unroll 1
      for (int c = threadIdx.x; c < p.N; c += TH) {
        const bool out = pass == 1 && p.keep < p.groups && !(s.kept >> (c / p.per) & 1);
        keys[c] = out ? kFiller - c : candidate_key<double>(p, logit_of(zr, c), c, m, t64, pass == 0);
      }
      __syncthreads();
      if (pass == 0) choose_groups<double, TH>(p, s, keys, total);
    }
    choose_slowly<TH>(p, s, keys);
  }
  if (warp == 0) {
    write_row(p, row, zr, m, total, [&](int j, bool& good) {
      const int v = s.place[j];
      good = v >= 0;
      return v >= 0 ? v : ~v;
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
    id[q] = static_cast<int>(p.idx[row * p.k + j]);
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
    const bool live = p.weights[row * p.k + j] != 0.f;
    const float v = logit_of(z, id[q]);
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
  MOC_REQUIRE(n <= kMostN, "at most 16384 chapters to choose from");
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

template <typename LT> int select_fwd(const SelectParams& p, cudaStream_t stream) {
  if (p.N <= kWarpMostN && p.k <= kWarpMostK) {
    auto kern = p.N <= 64 ? select_warp_kernel<LT, 2> : p.N <= 128 ? select_warp_kernel<LT, 4>
                : p.N <= 256 ? select_warp_kernel<LT, 8> : select_warp_kernel<LT, 16>;
    kern<<<ceil_div(p.rows, kWarpRows), 32 * kWarpRows, 0, stream>>>(p);
  } else {
    const bool big = p.N > 4096;
    auto kern = p.N <= 1024 ? select_cta_kernel<LT, 4, 256> : p.N <= 2048 ? select_cta_kernel<LT, 8, 256>
                : !big ? select_cta_kernel<LT, 16, 256> : p.N <= 8192 ? select_cta_kernel<LT, 8, 1024> : select_cta_kernel<LT, 16, 1024>;
    MOC_CUDA_OK(allow_shared(kern, static_cast<size_t>(p.N) * 8, kMostN * 8));
    kern<<<p.rows, big ? 1024 : 256, static_cast<size_t>(p.N) * 8, stream>>>(p);
  }
  MOC_CUDA_OK(cudaGetLastError());
  return MOC_OK;
}
template <typename LT> int select_bwd(const SelectGrads& p, cudaStream_t stream) {
  // a warp a row up to 512 chapters, a CTA beyond
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
  MOC_REQUIRE(logits && idx && weights && comb_idx && comb_w && row_stats, "NULL selection buffer");
  MOC_REQUIRE((reinterpret_cast<uintptr_t>(row_stats) & 15) == 0, "row_stats must be 16-byte aligned");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  SelectParams p{};
  p.logits = logits; p.bias = balance_bias; p.idx = reinterpret_cast<long long*>(idx); p.weights = weights;
  p.comb_idx = comb_idx; p.comb_w = comb_w; p.row_stats = row_stats; p.load = load; p.ld = s->ld;
  p.rows = s->rows; p.N = s->num_chapters - s->num_shared; p.S = s->num_shared; p.k = s->top_k;
  p.groups = s->num_groups; p.keep = s->top_groups; p.per = p.N / p.groups;
  p.sigmoid = s->score == MOC_SCORE_SIGMOID; p.top2 = s->group_top2 != 0; p.renorm = s->renormalize != 0; p.rho = s->routed_scale;
  if (load != nullptr) MOC_CUDA_OK(cudaMemsetAsync(load, 0, static_cast<size_t>(s->num_chapters) * sizeof(int32_t), stream));
  return s->dtype == MOC_F32 ? select_fwd<float>(p, stream) : select_fwd<__nv_bfloat16>(p, stream);
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
