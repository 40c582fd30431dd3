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
// Bound by HBM (f, x -> y, n; backward d_y, d_n, x, f -> d_x, d_f).  A row belongs to one CTA of as many threads as the row has
// pieces of four columns (up to 256; past 1,024 columns up to 512 of 2 or 4 pieces each), which holds it in registers between the passes: every
// tensor is read once and a row's reductions are one barrier each.  Small CTAs beside each other hide the barriers.
#include <initializer_list>
#include <type_traits>

#include "moc_common.cuh"

namespace moc {
namespace {

constexpr int kResBlocks = 148 * 4;       // CTAs of the backward pass: each keeps its column sums over its rows

// threads of a CTA: 256 where a thread has one piece, 512 otherwise
constexpr int most_threads(int nv, int v) { return nv * v == 4 ? 256 : 512; }

struct ResParams {
  const void *x, *f;
  const float *w, *b, *gate, *w2, *b2;
  void *y, *n;
  float* stats;                 // [rows, 4] = mean, inv of f, then of y; NULL: not wanted
  long long rows;
  int d, seq;                   // rows of a sequence (gate_rows) 
  int ln, gate_rows, next;      // gate_rows: the gate has a row for every sequence
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

// the pieces of four columns of one row that a thread has: lane-wise, so a warp's loads are contiguous
template <typename T, int V> struct Piece;
template <> struct Piece<float, 4> {
  static __device__ __forceinline__ void load(const float* p, float (&v)[4]) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};
template <> struct Piece<__nv_bfloat16, 4> {
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&v)[4]) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(a.x << 16); v[1] = __uint_as_float(a.x & 0xFFFF0000u);
    v[2] = __uint_as_float(a.y << 16); v[3] = __uint_as_float(a.y & 0xFFFF0000u);
  }
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

// Sum over the CTA, the same in every thread.  One barrier: the next call uses the other half of `red`.
struct RowSum {
  float2* red;        // [2][16]
  int half;
  __device__ __forceinline__ float2 operator()(float a, float b) {
    a = warp_sum(a);
    b = warp_sum(b);
    if (blockDim.x == 32) return make_float2(a, b);
    float2* r = red + half * 16;
    half ^= 1;
    if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    float2 t = make_float2(0.f, 0.f);
    const int nw = blockDim.x >> 5;
    for (int i = 0; i < nw; ++i) { t.x += r[i].x; t.y += r[i].y; }
    return t;
  }
};

// mean and 1 / sqrt(variance + eps) of the row in `v` (zero past its end); LayerNorm sums twice, as the difference of the mean of
// squares and the squared mean loses what is small against the mean
template <int NV, int V>
__device__ __forceinline__ float2 row_stats(const float (&v)[NV][V], int ln, float eps, int d, RowSum& sum) {
  float mean = 0.f, ss = 0.f;
  if (ln) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) s += v[i][j];
    mean = sum(s, 0.f).x / static_cast<float>(d);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int c = (threadIdx.x + i * blockDim.x) * V + j;
      const float u = c < d ? v[i][j] - mean : 0.f;
      ss = fmaf(u, u, ss);
    }
  return make_float2(mean, 1.f / sqrtf(sum(ss, 0.f).x / static_cast<float>(d) + eps));
}

template <typename T, int NV, int V>
__device__ __forceinline__ void load_row(const T* p, int d, float (&v)[NV][V]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (threadIdx.x + i * blockDim.x) * V;
    if (c < d) {
      Piece<T, V>::load(p + c, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] = 0.f;
    }
  }
}
template <typename T, int NV, int V>
__device__ __forceinline__ void store_row(T* p, int d, const float (&v)[NV][V]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (threadIdx.x + i * blockDim.x) * V;
    if (c < d) Piece<T, V>::store(p + c, v[i]);
  }
}
// v = v * w (+ b), columns past the end stay zero; w / b may be NULL
template <int NV, int V>
__device__ __forceinline__ void affine(float (&v)[NV][V], const float* w, const float* b, int d) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (threadIdx.x + i * blockDim.x) * V;
    if (c >= d) continue;
    float a[V];
    if (w != nullptr) {
      Piece<float, V>::load(w + c, a);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] *= a[j];
    }
    if (b != nullptr) {
      Piece<float, V>::load(b + c, a);
#pragma unroll
      for (int j = 0; j < V; ++j) v[i][j] += a[j];
    }
  }
}
template <int NV, int V>
__device__ __forceinline__ void normalise(float (&v)[NV][V], float2 st, int d) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) v[i][j] = (threadIdx.x + i * blockDim.x) * V + j < d ? (v[i][j] - st.x) * st.y : 0.f;
}

template <typename XT, typename FT, int NV, int V>
__global__ void __launch_bounds__(most_threads(NV, V))
residual_fwd_kernel(const ResParams p) {
  __shared__ float2 red[32];
  RowSum sum{red, 0};
  const long long row = blockIdx.x;
  float f[NV][V], x[NV][V];
  load_row(static_cast<const FT*>(p.f) + row * p.d, p.d, f);
  load_row(static_cast<const XT*>(p.x) + row * p.d, p.d, x);
  const float2 st = row_stats(f, p.ln, p.eps, p.d, sum);
  normalise(f, st, p.d);
  affine(f, p.w, p.b, p.d);
  if (p.gate != nullptr) affine(f, p.gate + (p.gate_rows ? row / p.seq * p.d : 0), nullptr, p.d);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) x[i][j] = fmaf(p.scale, x[i][j], f[i][j]);
  store_row(static_cast<XT*>(p.y) + row * p.d, p.d, x);
  float2 st2 = make_float2(0.f, 0.f);
  if (p.next) {
    st2 = row_stats(x, p.ln, p.eps2, p.d, sum);
    normalise(x, st2, p.d);
    affine(x, p.w2, p.b2, p.d);
    store_row(static_cast<FT*>(p.n) + row * p.d, p.d, x);
  }
  if (p.stats != nullptr && threadIdx.x == 0) reinterpret_cast<float4*>(p.stats)[row] = make_float4(st.x, st.y, st2.x, st2.y);
}

// Column sums a thread keeps over the rows of its CTA: [0] t fhat (times the gate where it has a row for every sequence),
// [1] the same without fhat, [2] d_n yhat, [3] d_n; LayerNorm has all four, RMSNorm [0] and [2].  A gate row's own sum
// leaves with each item (a run of rows of one sequence).
template <typename XT, typename FT, int NV, int V, bool LN>
__global__ void __launch_bounds__(most_threads(NV, V))
residual_bwd_kernel(const ResParams p, const ResGrads g) {
  __shared__ float2 red[32];
  RowSum sum{red, 0};
  constexpr int kSums = LN ? 4 : 2, kStep = LN ? 1 : 2;
  float acc[kSums][NV][V];
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) acc[k][i][j] = 0.f;
  const float inv_d = 1.f / static_cast<float>(p.d);

  for (long long item = blockIdx.x; item < g.items; item += gridDim.x) {
    const long long s = item / g.chunks;
    const long long r0 = s * p.seq + (item - s * g.chunks) * g.chunk_rows;
    const long long r1 = min(r0 + g.chunk_rows, min((s + 1) * p.seq, p.rows));
    const float* gate = p.gate == nullptr ? nullptr : p.gate + (p.gate_rows ? s * p.d : 0);
    float gsum[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) gsum[i][j] = 0.f;
    for (long long row = r0; row < r1; ++row) {
      float f[NV][V], t[NV][V];
      load_row(static_cast<const FT*>(p.f) + row * p.d, p.d, f);
      if (g.dy != nullptr) {
        load_row(static_cast<const XT*>(g.dy) + row * p.d, p.d, t);
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) t[i][j] = 0.f;
      }
      const float4 st = reinterpret_cast<const float4*>(p.stats)[row];
      if (g.dn != nullptr) {
        float y[NV][V], n[NV][V];
        load_row(static_cast<const XT*>(p.x) + row * p.d, p.d, y);
        load_row(static_cast<const FT*>(g.dn) + row * p.d, p.d, n);
        normalise(f, make_float2(st.x, st.y), p.d);
        float z[NV][V];
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) z[i][j] = f[i][j];
        affine(z, p.w, p.b, p.d);
        if (gate != nullptr) affine(z, gate, nullptr, p.d);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) y[i][j] = fmaf(p.scale, y[i][j], z[i][j]);
        normalise(y, make_float2(st.z, st.w), p.d);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            acc[LN ? 2 : 1][i][j] = fmaf(n[i][j], y[i][j], acc[LN ? 2 : 1][i][j]);
            if (LN) acc[kSums - 1][i][j] += n[i][j];
          }
        affine(n, p.w2, nullptr, p.d);
        float c1 = 0.f, c2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) { c1 = fmaf(n[i][j], y[i][j], c1); c2 += n[i][j]; }
        const float2 c = sum(c1, c2);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j)
            if ((threadIdx.x + i * blockDim.x) * V + j < p.d)
              t[i][j] += st.w * (n[i][j] - (LN ? c.y * inv_d : 0.f) - y[i][j] * (c.x * inv_d));
      } else {
        normalise(f, make_float2(st.x, st.y), p.d);
      }
      // t: the gradient at y; f: the normalised branch
      if (g.dx != nullptr) {
        float dx[NV][V];
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) dx[i][j] = p.scale * t[i][j];
        store_row(static_cast<XT*>(g.dx) + row * p.d, p.d, dx);
      }
      if (p.gate_rows) {
        float z[NV][V];
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) z[i][j] = f[i][j];
        affine(z, p.w, p.b, p.d);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) gsum[i][j] = fmaf(t[i][j], z[i][j], gsum[i][j]);
        affine(t, gate, nullptr, p.d);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          acc[0][i][j] = fmaf(t[i][j], f[i][j], acc[0][i][j]);
          if (LN) acc[1][i][j] += t[i][j];
        }
      if (!p.gate_rows && gate != nullptr) affine(t, gate, nullptr, p.d);
      affine(t, p.w, nullptr, p.d);
      float c1 = 0.f, c2 = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) { c1 = fmaf(t[i][j], f[i][j], c1); c2 += t[i][j]; }
      const float2 c = sum(c1, c2);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) t[i][j] = st.y * (t[i][j] - (LN ? c.y * inv_d : 0.f) - f[i][j] * (c.x * inv_d));
      store_row(static_cast<FT*>(g.df) + row * p.d, p.d, t);
    }
    if (p.gate_rows) store_row(g.gate_part + item * p.d, p.d, gsum);
  }
#pragma unroll
  for (int k = 0; k < kSums; ++k) store_row(g.partial + (static_cast<long long>(blockIdx.x) * 4 + k * kStep) * p.d, p.d, acc[k]);
}

struct ResSums {
  const float *partial, *gate_part;
  const float *w, *b, *gate;
  float *dw, *db, *dgate, *dw2, *db2;
  int blocks, d, chunks, ln, gate_rows;
};
// 32 columns a CTA, 8 warps share the partial rows.  blockIdx.y == 0: the sums over all rows; blockIdx.y - 1: a sequence's gate row.
__global__ void __launch_bounds__(256)
residual_sums_kernel(const ResSums s) {
  __shared__ float red[4][8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float a[4] = {0.f, 0.f, 0.f, 0.f};
  if (blockIdx.y > 0) {
    const long long q = blockIdx.y - 1;
    if (c < s.d)
      for (int k = warp; k < s.chunks; k += 8) a[0] += s.gate_part[(q * s.chunks + k) * s.d + c];
    red[0][warp][lane] = a[0];
    __syncthreads();
    if (warp == 0 && c < s.d) {
      float t = 0.f;
      for (int k = 0; k < 8; ++k) t += red[0][k][lane];
      s.dgate[q * s.d + c] = t;
    }
    return;
  }
  if (c < s.d) {
#pragma unroll 4
    for (int k = warp; k < s.blocks; k += 8) {
      const float* p = s.partial + static_cast<long long>(k) * 4 * s.d + c;
      a[0] += p[0];
      a[2] += p[2 * static_cast<long long>(s.d)];
      if (s.ln) { a[1] += p[s.d]; a[3] += p[3 * static_cast<long long>(s.d)]; }
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) red[k][warp][lane] = a[k];
  __syncthreads();
  if (warp > 0 || c >= s.d) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    a[k] = 0.f;
    for (int i = 0; i < 8; ++i) a[k] += red[k][i][lane];
  }
  // with a gate of one row the sums are without it: d_w = gate * sum t fhat, d_gate = sum t (w fhat + b)
  const float gate = s.gate != nullptr && !s.gate_rows ? s.gate[c] : 1.f;
  if (s.dw != nullptr) s.dw[c] = gate * a[0];
  if (s.db != nullptr) s.db[c] = gate * a[1];
  if (s.dgate != nullptr && !s.gate_rows) s.dgate[c] = s.w[c] * a[0] + (s.b != nullptr ? s.b[c] * a[1] : 0.f);
  if (s.dw2 != nullptr) s.dw2[c] = a[2];
  if (s.db2 != nullptr) s.db2[c] = a[3];
}

struct Plan {
  int v, nv, threads;
};
// pieces of four columns wherever rows and base addresses allow 16-byte (fp32) accesses, single columns otherwise
Plan plan_of(int d, bool wide) {
  const int each = d <= 1024 ? 4 : d <= 4096 ? 8 : 16;       // columns of a thread
  Plan p;
  p.v = wide ? 4 : 1;
  p.nv = each / p.v;
  p.threads = ((d + each - 1) / each + 31) / 32 * 32;
  return p;
}
template <typename Go> int with_plan(const Plan& p, Go go) {
  using std::integral_constant;
  if (p.v == 4) {
    if (p.nv == 1) return go(integral_constant<int, 1>{}, integral_constant<int, 4>{});
    if (p.nv == 2) return go(integral_constant<int, 2>{}, integral_constant<int, 4>{});
    return go(integral_constant<int, 4>{}, integral_constant<int, 4>{});
  }
  if (p.nv == 4) return go(integral_constant<int, 4>{}, integral_constant<int, 1>{});
  if (p.nv == 8) return go(integral_constant<int, 8>{}, integral_constant<int, 1>{});
  return go(integral_constant<int, 16>{}, integral_constant<int, 1>{});
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
// Runs of rows of one sequence: about as many as there are CTAs, whole sequences where those are shorter.
Split split_of(const ResParams& p) {
  Split s;
  const long long seqs = p.rows / p.seq;
  long long per = (kResBlocks + seqs - 1) / seqs;           // runs of a sequence
  if (per > p.seq) per = p.seq;
  s.chunk_rows = static_cast<int>((p.seq + per - 1) / per);
  s.chunks = (p.seq + s.chunk_rows - 1) / s.chunk_rows;
  s.items = seqs * s.chunks;
  s.blocks = static_cast<int>(s.items < kResBlocks ? s.items : kResBlocks);
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
  const Plan plan = plan_of(s->dim, wide(s->dim, {x, f, weight, bias, gate, next_weight, next_bias, y, n}));
  return with_types(s, [&](auto xt, auto ft) {
    return with_plan(plan, [&](auto nv, auto v) {
      residual_fwd_kernel<decltype(xt), decltype(ft), decltype(nv)::value, decltype(v)::value>
          <<<static_cast<unsigned>(p.rows), plan.threads, 0, static_cast<cudaStream_t>(stream)>>>(p);
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
  const Split sp = split_of(p);
  MOC_REQUIRE(!p.gate_rows || sp.items / sp.chunks <= 65534, "too many sequences with a gate row of their own (65,534)");
  ResGrads g{};
  g.dy = d_y; g.dn = d_n; g.dx = d_x; g.df = d_f;
  g.partial = static_cast<float*>(scratch);
  g.gate_part = g.partial + static_cast<long long>(sp.blocks) * 4 * p.d;
  g.chunks = sp.chunks; g.chunk_rows = sp.chunk_rows; g.items = sp.items;
  const Plan plan = plan_of(p.d, wide(p.d, {x, f, weight, bias, gate, next_weight, d_y, d_n, d_x, d_f}));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  rc = with_types(s, [&](auto xt, auto ft) {
    return with_plan(plan, [&](auto nv, auto v) {
      auto kern = p.ln ? residual_bwd_kernel<decltype(xt), decltype(ft), decltype(nv)::value, decltype(v)::value, true>
                       : residual_bwd_kernel<decltype(xt), decltype(ft), decltype(nv)::value, decltype(v)::value, false>;
      kern<<<sp.blocks, plan.threads, 0, st>>>(p, g);
      MOC_CUDA_OK(cudaGetLastError());
      return static_cast<int>(MOC_OK);
    });
  });
  if (rc != MOC_OK) return rc;
  if (d_weight || d_bias || d_gate || d_next_weight || d_next_bias) {
    ResSums q{g.partial, g.gate_part, weight, bias, gate, d_weight, d_bias, d_gate, d_next_weight, d_next_bias,
              sp.blocks, p.d, sp.chunks, p.ln, p.gate_rows};
    const unsigned seqs = p.gate_rows && d_gate ? static_cast<unsigned>(sp.items / sp.chunks) : 0u;
    residual_sums_kernel<<<dim3((p.d + 31) / 32, 1 + seqs), 256, 0, st>>>(q);
    MOC_CUDA_OK(cudaGetLastError());
  }
  return MOC_OK;
}
