// The output of a block merged into the residual stream, with the norm behind the block, its gate, and the norm in front of the
// next block in one pass:
//
//   z = norm(f) = (f - mean) inv w + b          (RMSNorm: mean 0, no b),   inv = 1 / sqrt(mean((f - mean)^2) + eps)
//   y = s x + gate * z                          (gate: none, [dim], or [batch, dim], one row a sequence)
//   n = norm2(y)                                (optional; of y before it is rounded to its own type)
//
// Backward, with t = d_y + norm2'(d_n) the gradient that reaches y:
//   d_x = s t,  d_f = norm'(gate * t * w),  d_gate = sum t * z,  d_w = sum gate * t * fhat,  d_b = sum gate * t,
//   d_w2 = sum d_n * yhat,  d_b2 = sum d_n.
// y is formed again from x and f (it was rounded on its way out, and the sums over rows would carry that rounding): the same
// bytes as reading y.
//
// Bound by HBM (f, x -> y, n; backward d_y, d_n, x, f -> d_x, d_f).  A row belongs to one warp (up to 384 columns forward, 768
// backward, 512 of a LayerNorm; 2 to 8 warps beyond), which holds it in registers between the passes, so every tensor is read once and a row's sums are shuffles.  The
// warps stay for many rows; while one is worked on, the next ones are on their way into shared memory (asynchronous copies,
// each thread its own columns, so nobody waits for anybody else).  The backward pass runs one CTA an SM; its warps keep the
// column sums of their rows in registers.
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "moc_common.cuh"

namespace moc {
namespace {

constexpr int kResThreads = 256;
constexpr int kResCtas = 148;             // CTAs of the backward pass

struct ResParams {
  const void *x, *f;
  const float *w, *b, *gate, *w2, *b2;
  void *y, *n;
  float* stats;                 // [rows, 4] = mean, inv of f, then of y; NULL: not wanted
  long long rows;
  int d, seq;                   // rows of a sequence (gate_rows) 
  int ln, gate_rows, next;      // gate_rows: the gate has a row for every sequence
  int group;                    // warps of a row
  float scale, eps, eps2;
};
struct ResGrads {
  const void *dy, *dn;
  void *dx, *df;
  float* partial;               // [CTAs][sums][d]
  float* gate_part;             // [sequences * chunks][d]
  int chunks, chunk_rows;       // of a sequence
  long long items;              // sequences * chunks
};

// the pieces of V columns of a row that a thread has: lane-wise, so a warp's loads are contiguous
template <typename T, int V> struct Piece;
template <> struct Piece<float, 4> {
  using Raw = float4;
  static __device__ __forceinline__ void unpack(const float4& a, float (&v)[4]) { v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; }
  static __device__ __forceinline__ void load(const float* p, float (&v)[4]) { unpack(*reinterpret_cast<const float4*>(p), v); }
  static __device__ __forceinline__ void store(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};
template <> struct Piece<__nv_bfloat16, 4> {
  using Raw = uint2;
  static __device__ __forceinline__ void unpack(const uint2& a, float (&v)[4]) {
    v[0] = __uint_as_float(a.x << 16); v[1] = __uint_as_float(a.x & 0xFFFF0000u);
    v[2] = __uint_as_float(a.y << 16); v[3] = __uint_as_float(a.y & 0xFFFF0000u);
  }
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&v)[4]) { unpack(*reinterpret_cast<const uint2*>(p), v); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&v)[4]) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  }
};
template <> struct Piece<float, 1> {
  static __device__ __forceinline__ void load(const float* p, float (&v)[1]) { v[0] = *p; }
  static __device__ __forceinline__ void store(float* p, const float (&v)[1]) { *p = v[0]; }
};
template <> struct Piece<__nv_bfloat16, 1> {
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&v)[1]) { v[0] = __bfloat162float(*p); }
  static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&v)[1]) { *p = __float2bfloat16(v[0]); }
};

// This thread's place: `t` of the `n` threads of its row (n: 32 times 1, 2, 4 or 8 warps), and the row's sums, the same in
// each of them (one barrier of those warps; the next call uses the other half of `red`).
struct RowGroup {
  int t, n, id;       // id: of the group in the CTA
  float2* red;        // [2][warps of the CTA]
  int half;
  __device__ __forceinline__ RowGroup(int warps, float2* r) : t(threadIdx.x % (32 * warps)), n(32 * warps), id(threadIdx.x / (32 * warps)), red(r), half(0) {}
  __device__ __forceinline__ float2 sum(float a, float b) {
    a = warp_sum(a);
    b = warp_sum(b);
    return across(a, b);
  }
  __device__ __forceinline__ float sum(float a) { return across(warp_sum(a), 0.f).x; }
  __device__ __forceinline__ float2 across(float a, float b) {
    if (n == 32) return make_float2(a, b);
    float2* r = red + half * (kResThreads / 32) + id * (n >> 5);
    half ^= 1;
    if ((threadIdx.x & 31) == 0) r[t >> 5] = make_float2(a, b);
    asm volatile("bar.sync %0, %1;" ::"r"(id + 1), "r"(n) : "memory");
    float2 s = r[0];
    for (int i = 1; i < (n >> 5); ++i) { s.x += r[i].x; s.y += r[i].y; }
    return s;
  }
};

// mean and 1 / sqrt(variance + eps) of the row in `v`.  Columns past the end hold zeros, which an RMSNorm may sum with the others and
// a LayerNorm leaves out; it sums twice, as the difference of the mean of squares and the squared mean loses what is small against
// the mean.
template <bool LN, int NV, int V>
__device__ __forceinline__ float2 row_stats(const float (&v)[NV][V], float eps, int d, RowGroup& g) {
  float mean = 0.f, ss[2] = {0.f, 0.f};
  if constexpr (LN) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) s += (g.t + i * g.n) * V < d ? v[i][j] : 0.f;       // (the affine step leaves its bias there)
    mean = g.sum(s) / static_cast<float>(d);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float u = !LN ? v[i][j] : (g.t + i * g.n) * V + j < d ? v[i][j] - mean : 0.f;
      ss[i & 1] = fmaf(u, u, ss[i & 1]);
    }
  return make_float2(mean, 1.f / sqrtf(g.sum(ss[0] + ss[1]) / static_cast<float>(d) + eps));
}

template <typename T, int NV, int V>
__device__ __forceinline__ void load_row(const RowGroup& g, const T* p, int d, float (&v)[NV][V]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (g.t + i * g.n) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) v[i][j] = 0.f;
    if (c < d) Piece<T, V>::load(p + c, v[i]);
  }
}
// A row on its way through shared memory: thread-private slots of one piece, kResThreads of them behind each other.  Single columns
// (V = 1) are not staged: they are read from their place when they are needed.
template <typename T, int NV, int V> __host__ __device__ constexpr int row_bytes() { return V == 1 ? 0 : NV * V * static_cast<int>(sizeof(T)) * kResThreads; }
__device__ __forceinline__ void cp_async8(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
template <typename T, int NV, int V>
__device__ __forceinline__ void stage_row(const RowGroup& g, const T* p, int d, char* slots) {
  if constexpr (V > 1) {
    using Raw = typename Piece<T, V>::Raw;
    Raw* to = reinterpret_cast<Raw*>(slots) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (g.t + i * g.n) * V;
      if (c >= d) continue;
      if constexpr (sizeof(Raw) == 16) cp_async16(to + i * kResThreads, p + c);
      else cp_async8(to + i * kResThreads, p + c);
    }
  }
}
template <typename T, int NV, int V>
__device__ __forceinline__ void staged_row(const RowGroup& g, const T* p, int d, const char* slots, float (&v)[NV][V]) {
  if constexpr (V == 1) {
    load_row(g, p, d, v);
  } else {
    using Raw = typename Piece<T, V>::Raw;
    const Raw* from = reinterpret_cast<const Raw*>(slots) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < NV; ++i) Piece<T, V>::unpack(from[i * kResThreads], v[i]);       // (unused slots hold zeros)
  }
}
// zeros in the slots of columns that no row has (this thread's own)
template <int V> __device__ __forceinline__ void clear_slots(char* slots, int bytes) {
  if constexpr (V > 1)
    for (int i = threadIdx.x * 16; i < bytes; i += kResThreads * 16) *reinterpret_cast<uint4*>(slots + i) = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
}
// waits until at most `ahead` of this thread's committed rows are still on their way
__device__ __forceinline__ void wait_rows(int ahead) {
  if (ahead == 0) cp_async_wait<0>();
  else if (ahead == 1) cp_async_wait<1>();
  else if (ahead == 2) cp_async_wait<2>();
  else cp_async_wait<3>();
}
__device__ __forceinline__ void warm(const RowGroup& g, const float* p, int d) {       // a parameter row on its way into L1
  if (p == nullptr) return;
  for (int c = g.t * 32; c < d; c += g.n * 32) asm volatile("prefetch.global.L1 [%0];" ::"l"(p + c));
}
template <typename T, int NV, int V>
__device__ __forceinline__ void store_row(const RowGroup& g, T* p, int d, const float (&v)[NV][V]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (g.t + i * g.n) * V;
    if (c < d) Piece<T, V>::store(p + c, v[i]);
  }
}
// v = v * w (+ b); columns past the end meet zeros
template <int NV, int V>
__device__ __forceinline__ void affine(const RowGroup& g, float (&v)[NV][V], const float* w, const float* b, int d) {
  float a[NV][V];
  load_row(g, w, d, a);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) v[i][j] *= a[i][j];
  if (b == nullptr) return;
  load_row(g, b, d, a);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) v[i][j] += a[i][j];
}
template <bool LN, int NV, int V>
__device__ __forceinline__ void normalise(const RowGroup& g, float (&v)[NV][V], float2 st, int d) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) v[i][j] = !LN ? v[i][j] * st.y : (g.t + i * g.n) * V + j < d ? (v[i][j] - st.x) * st.y : 0.f;
}

// depth: rows of a warp group in shared memory at once
template <typename XT, typename FT, int NV, int V, bool LN>
__global__ void __launch_bounds__(kResThreads, NV * V <= 12 ? 4 : NV * V <= 24 ? 2 : 1)
residual_fwd_kernel(const ResParams p, const int depth) {
  __shared__ float2 red[2 * kResThreads / 32];
  extern __shared__ __align__(16) char slots[];
  constexpr int kF = row_bytes<FT, NV, V>(), kSlots = kF + row_bytes<XT, NV, V>();
  RowGroup g(p.group, red);
  const int groups = kResThreads / g.n;
  const long long stride = static_cast<long long>(gridDim.x) * groups;
  const FT* fp = static_cast<const FT*>(p.f);
  const XT* xp = static_cast<const XT*>(p.x);
  long long ahead = static_cast<long long>(blockIdx.x) * groups + g.id;
  int fill = 0;
  auto fetch = [&]() {
    if (ahead < p.rows) {
      stage_row<FT, NV, V>(g, fp + ahead * p.d, p.d, slots + fill * kSlots);
      stage_row<XT, NV, V>(g, xp + ahead * p.d, p.d, slots + fill * kSlots + kF);
    }
    cp_async_commit();
    ahead += stride;
    fill = fill + 1 == depth ? 0 : fill + 1;
  };
  int stage = 0;
  clear_slots<V>(slots, depth * kSlots);
  for (int i = 1; i < depth; ++i) fetch();
  warm(g, p.w, p.d); warm(g, p.b, p.d); warm(g, p.w2, p.d); warm(g, p.b2, p.d);
  if (!p.gate_rows) warm(g, p.gate, p.d);
  for (long long row = static_cast<long long>(blockIdx.x) * groups + g.id; row < p.rows; row += stride) {
    fetch();
    wait_rows(depth - 1);
    float f[NV][V], x[NV][V];
    staged_row(g, fp + row * p.d, p.d, slots + stage * kSlots, f);
    staged_row(g, xp + row * p.d, p.d, slots + stage * kSlots + kF, x);
    stage = stage + 1 == depth ? 0 : stage + 1;
    const float2 st = row_stats<LN>(f, p.eps, p.d, g);
    normalise<LN>(g, f, st, p.d);
    affine(g, f, p.w, p.b, p.d);
    if (p.gate != nullptr) affine(g, f, p.gate + (p.gate_rows ? row / p.seq * p.d : 0), nullptr, p.d);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) x[i][j] = fmaf(p.scale, x[i][j], f[i][j]);
    store_row(g, static_cast<XT*>(p.y) + row * p.d, p.d, x);
    float2 st2 = make_float2(0.f, 0.f);
    if (p.next) {
      st2 = row_stats<LN>(x, p.eps2, p.d, g);
      normalise<LN>(g, x, st2, p.d);
      affine(g, x, p.w2, p.b2, p.d);
      store_row(g, static_cast<FT*>(p.n) + row * p.d, p.d, x);
    }
    if (p.stats != nullptr && g.t == 0) reinterpret_cast<float4*>(p.stats)[row] = make_float4(st.x, st.y, st2.x, st2.y);
  }
}

// Column sums a thread keeps over its rows: [0] t fhat (times the gate where it has a row for every sequence),
// [1] the same without fhat, [2] d_n yhat, [3] d_n; LayerNorm has all four, RMSNorm [0] and [2].  A gate row's own sum
// leaves with each item (a run of rows of one sequence).
template <typename XT, typename FT, int NV, int V, bool LN>
__global__ void __launch_bounds__(kResThreads, 1)
residual_bwd_kernel(const ResParams p, const ResGrads q, const int depth) {
  __shared__ float2 red[2 * kResThreads / 32];
  extern __shared__ __align__(16) char slots[];         // rows on their way, at the end [groups of the CTA][d] column sums
  float* columns = reinterpret_cast<float*>(slots);
  constexpr int kF = row_bytes<FT, NV, V>(), kX = row_bytes<XT, NV, V>(), kSlots = 2 * (kF + kX);
  RowGroup g(p.group, red);
  constexpr int kSums = LN ? 4 : 2, kStep = LN ? 1 : 2;
  const int groups = kResThreads / g.n;
  float acc[kSums][NV][V];
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) acc[k][i][j] = 0.f;
  const float inv_d = 1.f / static_cast<float>(p.d);

  const long long first = static_cast<long long>(blockIdx.x) * groups + g.id, stride = static_cast<long long>(gridDim.x) * groups;
  auto rows_of = [&](long long item, long long& r0, long long& r1) {       // of a run; none behind the last
    const long long s = item / q.chunks;
    r0 = s * p.seq + (item - s * q.chunks) * q.chunk_rows;
    r1 = item < q.items ? min(r0 + q.chunk_rows, min((s + 1) * p.seq, p.rows)) : r0;
  };
  long long next_item = first, next_row, next_end;
  rows_of(next_item, next_row, next_end);
  int fill = 0, stage = 0;
  auto fetch = [&]() {
    if (next_row < next_end) {
      char* to = slots + fill * kSlots;
      const long long at = next_row * p.d;
      stage_row<FT, NV, V>(g, static_cast<const FT*>(p.f) + at, p.d, to);
      if (q.dy != nullptr) stage_row<XT, NV, V>(g, static_cast<const XT*>(q.dy) + at, p.d, to + kF);
      if (q.dn != nullptr) {
        stage_row<XT, NV, V>(g, static_cast<const XT*>(p.x) + at, p.d, to + kF + kX);
        stage_row<FT, NV, V>(g, static_cast<const FT*>(q.dn) + at, p.d, to + kF + 2 * kX);
      }
      if (++next_row == next_end) {
        next_item += stride;
        rows_of(next_item, next_row, next_end);
      }
    }
    cp_async_commit();
    fill = fill + 1 == depth ? 0 : fill + 1;
  };
  clear_slots<V>(slots, depth * kSlots);
  for (int i = 1; i < depth; ++i) fetch();
  for (long long item = first; item < q.items; item += stride) {
    const long long s = item / q.chunks;
    long long r0, r1;
    rows_of(item, r0, r1);
    const float* gate = p.gate == nullptr ? nullptr : p.gate + (p.gate_rows ? s * p.d : 0);
    // (a gate row's sum is rare: it is kept in its place in memory)
    for (long long row = r0; row < r1; ++row) {
      fetch();
      wait_rows(depth - 1);
      const char* from = slots + stage * kSlots;
      stage = stage + 1 == depth ? 0 : stage + 1;
      float f[NV][V], t[NV][V];
      staged_row(g, static_cast<const FT*>(p.f) + row * p.d, p.d, from, f);
      if (q.dy != nullptr) {
        staged_row(g, static_cast<const XT*>(q.dy) + row * p.d, p.d, from + kF, t);
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) t[i][j] = 0.f;
      }
      const float4 st = reinterpret_cast<const float4*>(p.stats)[row];
      if (q.dn != nullptr) {
        float y[NV][V], n[NV][V];
        staged_row(g, static_cast<const XT*>(p.x) + row * p.d, p.d, from + kF + kX, y);
        staged_row(g, static_cast<const FT*>(q.dn) + row * p.d, p.d, from + kF + 2 * kX, n);
        normalise<LN>(g, f, make_float2(st.x, st.y), p.d);
        {
          float z[NV][V];
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) z[i][j] = f[i][j];
          affine(g, z, p.w, p.b, p.d);
          if (gate != nullptr) affine(g, z, gate, nullptr, p.d);
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) y[i][j] = fmaf(p.scale, y[i][j], z[i][j]);
        }
        normalise<LN>(g, y, make_float2(st.z, st.w), p.d);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            acc[LN ? 2 : 1][i][j] = fmaf(n[i][j], y[i][j], acc[LN ? 2 : 1][i][j]);
            if (LN) acc[kSums - 1][i][j] += n[i][j];
          }
        affine(g, n, p.w2, nullptr, p.d);
        float c1 = 0.f, c2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) { c1 = fmaf(n[i][j], y[i][j], c1); if (LN) c2 += n[i][j]; }
        const float2 c = LN ? g.sum(c1, c2) : make_float2(g.sum(c1), 0.f);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (!LN || (g.t + i * g.n) * V + j < p.d) t[i][j] += st.w * (n[i][j] - (LN ? c.y * inv_d : 0.f) - y[i][j] * (c.x * inv_d));
      } else {
        normalise<LN>(g, f, make_float2(st.x, st.y), p.d);
      }
      // t: the gradient at y; f: the normalised branch
      if (q.dx != nullptr) {
        XT* dx = static_cast<XT*>(q.dx) + row * p.d;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          float u[V];
#pragma unroll
          for (int j = 0; j < V; ++j) u[j] = p.scale * t[i][j];
          const int c = (g.t + i * g.n) * V;
          if (c < p.d) Piece<XT, V>::store(dx + c, u);
        }
      }
      if (p.gate_rows) {
        float* sum = q.gate_part + item * p.d;
        float z[NV][V];
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) z[i][j] = f[i][j];
        affine(g, z, p.w, p.b, p.d);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) z[i][j] *= t[i][j];
        if (row > r0) {
          float old[NV][V];
          load_row(g, const_cast<const float*>(sum), p.d, old);
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) z[i][j] += old[i][j];
        }
        store_row(g, sum, p.d, z);
        affine(g, t, gate, nullptr, p.d);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          acc[0][i][j] = fmaf(t[i][j], f[i][j], acc[0][i][j]);
          if (LN) acc[1][i][j] += t[i][j];
        }
      if (!p.gate_rows && gate != nullptr) affine(g, t, gate, nullptr, p.d);
      affine(g, t, p.w, nullptr, p.d);
      float c1 = 0.f, c2 = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) { c1 = fmaf(t[i][j], f[i][j], c1); if (LN) c2 += t[i][j]; }
      const float2 c = LN ? g.sum(c1, c2) : make_float2(g.sum(c1), 0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) t[i][j] = st.y * (t[i][j] - (LN ? c.y * inv_d : 0.f) - f[i][j] * (c.x * inv_d));
      store_row(g, static_cast<FT*>(q.df) + row * p.d, p.d, t);
    }
  }
  // the groups' column sums -> the CTA's
#pragma unroll
  for (int k = 0; k < kSums; ++k) {
    float* out = q.partial + (static_cast<long long>(blockIdx.x) * 4 + k * kStep) * p.d;
    if (groups == 1) {
      store_row(g, out, p.d, acc[k]);
      continue;
    }
    __syncthreads();
    store_row(g, columns + g.id * p.d, p.d, acc[k]);
    __syncthreads();
    for (int c = threadIdx.x; c < p.d; c += kResThreads) {
      float t = 0.f;
      for (int i = 0; i < groups; ++i) t += columns[i * p.d + c];
      out[c] = t;
    }
  }
}

struct ResSums {
  const float *partial, *gate_part;
  const float *w, *b, *gate;
  float *dw, *db, *dgate, *dw2, *db2;
  int blocks, d, chunks, ln, gate_rows;
};
// 32 columns a CTA, 32 warps share the partial rows.  blockIdx.y == 0: the sums over all rows; blockIdx.y - 1: a sequence's gate row.
__global__ void __launch_bounds__(1024)
residual_sums_kernel(const ResSums s) {
  __shared__ float red[4][32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  if (blockIdx.y > 0) {
    const long long q = blockIdx.y - 1;
    if (c < s.d)
      for (int k = warp; k < s.chunks; k += 32) a[0] += s.gate_part[(q * s.chunks + k) * s.d + c];
  } else if (c < s.d) {
#pragma unroll 4
    for (int k = warp; k < s.blocks; k += 32) {
      const float* p = s.partial + static_cast<long long>(k) * 4 * s.d + c;
      a[0] += p[0];
      a[2] += p[2 * static_cast<long long>(s.d)];
      if (s.ln) { a[1] += p[s.d]; a[3] += p[3 * static_cast<long long>(s.d)]; }
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) red[k][lane][warp] = a[k];
  __syncthreads();
  // warp w adds column w up over the 32 warps
  const int col = blockIdx.x * 32 + warp;
#pragma unroll
  for (int k = 0; k < 4; ++k) a[k] = warp_sum(red[k][warp][lane]);
  if (lane > 0 || col >= s.d) return;
  if (blockIdx.y > 0) {
    s.dgate[static_cast<long long>(blockIdx.y - 1) * s.d + col] = a[0];
    return;
  }
  // with a gate of one row the sums are without it: d_w = gate * sum t fhat, d_gate = sum t (w fhat + b)
  const float gate = s.gate != nullptr && !s.gate_rows ? s.gate[col] : 1.f;
  if (s.dw != nullptr) s.dw[col] = gate * a[0];
  if (s.db != nullptr) s.db[col] = gate * a[1];
  if (s.dgate != nullptr && !s.gate_rows) s.dgate[col] = s.w[col] * a[0] + (s.b != nullptr ? s.b[col] * a[1] : 0.f);
  if (s.dw2 != nullptr) s.dw2[col] = a[2];
  if (s.db2 != nullptr) s.db2[col] = a[3];
}

struct Plan {
  int v, each, group;              // columns of an access, of a thread; warps of a row
};
// Pieces of four columns wherever rows and base addresses allow 16-byte (fp32) accesses, single columns otherwise.  Backward, 24 columns
// a lane fill a row of 768 with one warp; a LayerNorm keeps four sums a column and takes 16.  Forward, 12 make two warps a row.
// Backward plans of 32 columns (rows above 4,096) spill: 156 bytes a thread for RMS, 900 for LayerNorm; single columns from 24 bytes (16
// columns) to 1,880 (LayerNorm, 32).  Per element they cost up to twice (vector) and six times (single) what the others do.  fp32 stream, bf16
// branch, next norm, gate [d], us forward / backward: 8,192 x 768 RMS 20 / 39, LayerNorm 31 / 57, with a gate per sequence 21 / 47 and 31 / 65;
// 2,048 x 4,096 25 / 60 and 39 / 69; 1,024 x 8,192 29 / 70 and 47 / 104; single columns: 8,192 x 767 31 / 76 and 47 / 106, 1,024 x 8,191
// LayerNorm 115 / 288.
Plan plan_of(int d, bool wide, bool lean, bool fwd = false) {
  Plan p;
  p.v = wide ? 4 : 1;
  p.each = d <= 256 ? 8 : d <= 768 ? (fwd ? 12 : lean ? 16 : 24) : d <= 4096 ? 16 : 32;
  p.group = 1;
  while (p.group * 32 * p.each < d) p.group *= 2;
  return p;
}
// go(columns a thread / V, V, whether LayerNorm) for what plan_of gives: MIDDLE is its number of columns between 257 and 768
template <int V, int MIDDLE, bool LN, typename Go> int with_each(int each, Go go) {
  using std::integral_constant;
  using W = integral_constant<int, V>;
  using N = integral_constant<bool, LN>;
  if (each == 8) return go(integral_constant<int, 8 / V>{}, W{}, N{});
  if constexpr (MIDDLE != 16)
    if (each == MIDDLE) return go(integral_constant<int, MIDDLE / V>{}, W{}, N{});
  if (each == 16) return go(integral_constant<int, 16 / V>{}, W{}, N{});
  MOC_REQUIRE(each == 32, "no residual kernel for this number of columns a thread");
  return go(integral_constant<int, 32 / V>{}, W{}, N{});
}
template <int RMS, int LN, typename Go> int with_plan(const Plan& p, bool ln, Go go) {
  if (ln) return p.v == 4 ? with_each<4, LN, true>(p.each, go) : with_each<1, LN, true>(p.each, go);
  return p.v == 4 ? with_each<4, RMS, false>(p.each, go) : with_each<1, RMS, false>(p.each, go);
}
// Rows in flight a warp group: as many of `bytes` a CTA as fit, four at most
int depth_of(const Plan& p, int bytes, int room) {
  if (p.v == 1) return 1;
  return std::max(1, std::min(4, room / bytes));
}
template <typename Go> int with_types(const moc_residual_shape* s, Go go) {
  if (s->x_dtype == MOC_F32) return s->f_dtype == MOC_F32 ? go(float{}, float{}) : go(float{}, __nv_bfloat16{});
  return s->f_dtype == MOC_F32 ? go(__nv_bfloat16{}, float{}) : go(__nv_bfloat16{}, __nv_bfloat16{});
}

constexpr int kResMostDim = 8192;
int check(const moc_residual_shape* s) {
  MOC_REQUIRE(s != nullptr, "NULL residual shape");
  MOC_REQUIRE(s->rows > 0 && s->rows < (1ll << 31) && s->dim > 0 && s->dim <= kResMostDim, "rows must be positive and dim in 1..8192");
  MOC_REQUIRE(s->kind == MOC_NORM_RMS || s->kind == MOC_NORM_LAYERNORM, "normalisation kind must be RMS or LayerNorm");
  for (int dt : {s->x_dtype, s->f_dtype}) MOC_REQUIRE(dt == MOC_F32 || dt == MOC_BF16, "unknown dtype");
  MOC_REQUIRE(s->gate_seq >= 0 && (s->gate_seq == 0 || s->rows % s->gate_seq == 0), "rows must be whole sequences of the gate");
  return MOC_OK;
}
bool wide(int d, std::initializer_list<const void*> ptrs) {
  if (d % 4 != 0) return false;
  for (const void* q : ptrs)
    if ((reinterpret_cast<uintptr_t>(q) & 15) != 0) return false;
  return true;
}
ResParams params(const moc_residual_shape* s, const void* x, const void* f, const float* w, const float* b, const float* gate,
                 const float* w2, const float* b2, float* stats) {
  ResParams p{};
  p.x = x; p.f = f; p.w = w; p.b = b; p.gate = gate; p.w2 = w2; p.b2 = b2; p.stats = stats;
  p.rows = s->rows; p.d = s->dim; p.ln = s->kind == MOC_NORM_LAYERNORM;
  p.gate_rows = gate != nullptr && s->gate_seq > 0;
  p.seq = p.gate_rows ? s->gate_seq : static_cast<int>(s->rows);
  p.next = w2 != nullptr;
  p.scale = s->residual_scale; p.eps = s->eps; p.eps2 = s->next_eps;
  return p;
}
struct Split {
  int chunks, chunk_rows, blocks;
  long long items;
};
// Runs of rows of one sequence: about as many as there are groups of warps, whole sequences where those are shorter.
Split split_of(const ResParams& p) {
  Split s;
  const long long seqs = p.rows / p.seq;
  const int groups = kResThreads / (32 * p.group), most = kResCtas * groups;
  long long per = (most + seqs - 1) / seqs;                 // runs of a sequence
  if (per > p.seq) per = p.seq;
  s.chunk_rows = static_cast<int>((p.seq + per - 1) / per);
  s.chunks = (p.seq + s.chunk_rows - 1) / s.chunk_rows;
  s.items = seqs * s.chunks;
  s.blocks = static_cast<int>(std::min<long long>((s.items + groups - 1) / groups, kResCtas));
  return s;
}

}  // namespace
}  // namespace moc

using namespace moc;

extern "C" int moc_gated_residual_fwd(const moc_residual_shape* s, const void* x, const void* f, const float* weight, const float* bias,
                                      const float* gate, const float* next_weight, const float* next_bias, void* y, void* n,
                                      float* stats, void* stream) {
  int rc = check(s);
  if (rc != MOC_OK) return rc;
  MOC_REQUIRE(x && f && weight && y && (next_weight == nullptr || n), "NULL residual argument");
  MOC_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 15) == 0, "stats must be 16-byte aligned");
  ResParams p = params(s, x, f, weight, bias, gate, next_weight, next_bias, stats);
  p.y = y; p.n = n;
  const Plan plan = plan_of(s->dim, wide(s->dim, {x, f, weight, bias, gate, next_weight, next_bias, y, n}), false, true);
  p.group = plan.group;
  const int groups = kResThreads / (32 * p.group), ctas = plan.each <= 12 ? 4 : plan.each <= 24 ? 2 : 1;         // on an SM
  const int bytes = plan.each * kResThreads * ((s->x_dtype == MOC_F32 ? 4 : 2) + (s->f_dtype == MOC_F32 ? 4 : 2));
  const int depth = depth_of(plan, bytes, 160 * 1024 / ctas);          // (the rest is L1, for the parameters)
  const long long most = (p.rows + groups - 1) / groups;
  const unsigned grid = static_cast<unsigned>(std::min<long long>(most, static_cast<long long>(kResCtas) * ctas));
  return with_types(s, [&](auto xt, auto ft) {
    return with_plan<12, 12>(plan, p.ln, [&](auto nv, auto v, auto ln) {
      auto kern = residual_fwd_kernel<decltype(xt), decltype(ft), decltype(nv)::value, decltype(v)::value, decltype(ln)::value>;
      const size_t shared = plan.v == 1 ? 0 : static_cast<size_t>(depth) * bytes;
      MOC_CUDA_OK(allow_shared(kern, shared, 216 * 1024));
      kern<<<grid, kResThreads, shared, static_cast<cudaStream_t>(stream)>>>(p, depth);
      MOC_CUDA_OK(cudaGetLastError());
      return static_cast<int>(MOC_OK);
    });
  });
}

extern "C" int64_t moc_gated_residual_bwd_scratch_bytes(const moc_residual_shape* s, int32_t with_gate) {
  if (check(s) != MOC_OK) return -1;
  ResParams p{};
  p.rows = s->rows;
  p.seq = with_gate && s->gate_seq > 0 ? s->gate_seq : static_cast<int>(s->rows);
  p.group = plan_of(s->dim, true, s->kind == MOC_NORM_LAYERNORM).group;          // (the same for single columns)
  const Split sp = split_of(p);
  return (static_cast<int64_t>(sp.blocks) * 4 + (with_gate && s->gate_seq > 0 ? sp.items : 0)) * s->dim * 4 + 256;
}

extern "C" int moc_gated_residual_bwd(const moc_residual_shape* s, const void* x, const void* f, const float* weight,
                                      const float* bias, const float* gate, const float* next_weight, const float* stats,
                                      const void* d_y, const void* d_n, void* d_x, void* d_f, float* d_weight, float* d_bias,
                                      float* d_gate, float* d_next_weight, float* d_next_bias, void* scratch, void* stream) {
  int rc = check(s);
  if (rc != MOC_OK) return rc;
  MOC_REQUIRE(x && f && weight && stats && d_f && scratch && (d_y || d_n), "NULL residual-gradient argument");
  MOC_REQUIRE(d_n == nullptr || next_weight != nullptr, "a gradient of the next norm needs its weight");
  MOC_REQUIRE(d_gate == nullptr || gate != nullptr, "a gate gradient needs the gate");
  MOC_REQUIRE(((reinterpret_cast<uintptr_t>(stats) | reinterpret_cast<uintptr_t>(scratch)) & 15) == 0,
              "stats and scratch must be 16-byte aligned");
  ResParams p = params(s, x, f, weight, bias, gate, next_weight, nullptr, const_cast<float*>(stats));
  const Plan plan = plan_of(p.d, wide(p.d, {x, f, weight, bias, gate, next_weight, d_y, d_n, d_x, d_f}), p.ln);
  p.group = plan.group;
  const Split sp = split_of(p);
  MOC_REQUIRE(!p.gate_rows || sp.items / sp.chunks <= 65534, "too many sequences with a gate row of their own (65,534)");
  ResGrads g{};
  g.dy = d_y; g.dn = d_n; g.dx = d_x; g.df = d_f;
  g.partial = static_cast<float*>(scratch);
  g.gate_part = g.partial + static_cast<long long>(sp.blocks) * 4 * p.d;
  g.chunks = sp.chunks; g.chunk_rows = sp.chunk_rows; g.items = sp.items;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int bytes = 2 * plan.each * kResThreads * ((s->x_dtype == MOC_F32 ? 4 : 2) + (s->f_dtype == MOC_F32 ? 4 : 2));
  const int depth = depth_of(plan, bytes, 216 * 1024);
  rc = with_types(s, [&](auto xt, auto ft) {
    return with_plan<24, 16>(plan, p.ln, [&](auto nv, auto v, auto ln) {
      auto kern = residual_bwd_kernel<decltype(xt), decltype(ft), decltype(nv)::value, decltype(v)::value, decltype(ln)::value>;
      const int groups = kResThreads / (32 * p.group);
      const size_t shared = std::max(plan.v == 1 ? size_t{0} : static_cast<size_t>(depth) * bytes,
                                     groups > 1 ? static_cast<size_t>(groups) * p.d * sizeof(float) : size_t{0});
      MOC_CUDA_OK(allow_shared(kern, shared, 216 * 1024));
      kern<<<sp.blocks, kResThreads, shared, st>>>(p, g, depth);
      MOC_CUDA_OK(cudaGetLastError());
      return static_cast<int>(MOC_OK);
    });
  });
  if (rc != MOC_OK) return rc;
  if (d_weight || d_bias || d_gate || d_next_weight || d_next_bias) {
    ResSums q{g.partial, g.gate_part, weight, bias, gate, d_weight, d_bias, d_gate, d_next_weight, d_next_bias,
              sp.blocks, p.d, sp.chunks, p.ln, p.gate_rows};
    const unsigned seqs = p.gate_rows && d_gate ? static_cast<unsigned>(sp.items / sp.chunks) : 0u;
    residual_sums_kernel<<<dim3((p.d + 31) / 32, 1 + seqs), 1024, 0, st>>>(q);
    MOC_CUDA_OK(cudaGetLastError());
  }
  return MOC_OK;
}
