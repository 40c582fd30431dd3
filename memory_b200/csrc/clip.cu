// Global gradient norm over many tensors, and the clipped tensors.
//
//   norm = sqrt(sum over tensors i of w_i^2 sum g_i^2),  coefficient = min(1, max_norm / (norm + eps)),  out_i = coefficient g_i
//
// Two launches whatever the number of tensors (up to kMostEntries a launch: the table of tensors travels as a kernel
// parameter, so nothing is copied to the device beforehand and a captured call replays without host memory).  The first
// leaves one partial sum per CTA; in the second every CTA adds the partials up in one order, so no CTA waits for another,
// no counter has to be reset and the result is the same on every run.  Squares are summed in 64 bits: fp32 squares leave
// the range above 1.8e19 and below 1e-19, and the conversion and the product hide behind HBM, which bounds both passes.
#include <cuda_fp16.h>

#include <algorithm>

#include "moc_common.cuh"

namespace moc {
namespace {

constexpr int kClipThreads = 256;
constexpr int kClipChunk = 8192;              // elements of one tensor that a CTA takes at a time: 4 steps of 8 a thread
constexpr int kClipSteps = kClipChunk / (kClipThreads * 8);
constexpr int kClipBlocks = 148 * 4;          // (the registers leave room for at least four CTAs on an SM)
constexpr int kFewEntries = 64, kMostEntries = 680;

struct ClipEntry {
  const void* src;
  void* dst;
  long long n;               // elements
  const int* count;          // compact rows: the first *count units exist; NULL: all
  int unit;                  // elements of a unit
  int chunk0;                // chunks of the entries before
  float weight;
  int dtypes;                // of src, and of dst << 8
};
template <int N> struct ClipTable {
  ClipEntry e[N];
  int entries, chunks;
};

// the last entry whose first chunk is at or before `chunk` (an entry without elements has no chunk: the next starts where it does)
template <int N> __device__ __forceinline__ int entry_of(const ClipTable<N>& t, int chunk) {
  int lo = 0, hi = t.entries - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].chunk0 <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}
__device__ __forceinline__ int size_of(int dtype) { return dtype == MOC_F32 ? 4 : 2; }
__device__ __forceinline__ float load_one(const void* p, long long i, int dtype) {
  if (dtype == MOC_F32) return static_cast<const float*>(p)[i];
  if (dtype == MOC_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_one(void* p, long long i, int dtype, float v) {
  if (dtype == MOC_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == MOC_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16(v);
  else static_cast<__half*>(p)[i] = __float2half(v);
}
// 8 values a step of this thread from element `first` on; what lies outside [0, n) is 0.  (The type is known to the code, so that
// all of a chunk's loads are requested before the first is converted.)
template <int DT> __device__ __forceinline__ void load_chunk(const void* p, long long first, long long n, float (&v)[kClipSteps][8]) {
  constexpr int kPieces = DT == MOC_F32 ? 2 : 1;
  uint4 raw[kClipSteps][kPieces];
#pragma unroll
  for (int s = 0; s < kClipSteps; ++s) {
    const long long i = first + s * (kClipThreads * 8);
    if (i >= 0 && i + 8 <= n) {
      const uint4* q = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + i * (DT == MOC_F32 ? 4 : 2));
#pragma unroll
      for (int k = 0; k < kPieces; ++k) raw[s][k] = __ldcs(q + k);
    } else {
#pragma unroll
      for (int k = 0; k < kPieces; ++k) raw[s][k] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
#pragma unroll
  for (int s = 0; s < kClipSteps; ++s) {
    const long long i = first + s * (kClipThreads * 8);
    if constexpr (DT == MOC_F32) {
      const uint32_t w[8] = {raw[s][0].x, raw[s][0].y, raw[s][0].z, raw[s][0].w, raw[s][1].x, raw[s][1].y, raw[s][1].z, raw[s][1].w};
#pragma unroll
      for (int j = 0; j < 8; ++j) v[s][j] = __uint_as_float(w[j]);
    } else {
      const uint32_t w[4] = {raw[s][0].x, raw[s][0].y, raw[s][0].z, raw[s][0].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (DT == MOC_BF16) {
          v[s][2 * j] = __uint_as_float(w[j] << 16);
          v[s][2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
          v[s][2 * j] = f.x;
          v[s][2 * j + 1] = f.y;
        }
      }
    }
    if ((i < 0 || i + 8 > n) && i + 8 > 0 && i < n) {       // the ends of a tensor
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i + j >= 0 && i + j < n) v[s][j] = load_one(p, i + j, DT);
    }
  }
}
__device__ __forceinline__ void load_chunk(const void* p, long long first, long long n, int dtype, float (&v)[kClipSteps][8]) {
  if (dtype == MOC_F32) load_chunk<MOC_F32>(p, first, n, v);
  else if (dtype == MOC_BF16) load_chunk<MOC_BF16>(p, first, n, v);
  else load_chunk<MOC_F16>(p, first, n, v);
}
__device__ __forceinline__ void store8(void* p, long long i, int dtype, const float (&v)[8]) {
  if (dtype == MOC_F32) {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
    __stcs(q, make_float4(v[0], v[1], v[2], v[3]));
    __stcs(q + 1, make_float4(v[4], v[5], v[6], v[7]));
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (dtype == MOC_BF16) w[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
    else { const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]); w[j] = *reinterpret_cast<const uint32_t*>(&h); }
  }
  __stcs(reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i), make_uint4(w[0], w[1], w[2], w[3]));
}
// elements by which a tensor starts behind a 16-byte boundary: its chunks start that much earlier, on the boundary
__device__ __forceinline__ int behind(const void* p, int dtype) {
  return static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) / size_of(dtype));
}
__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int w = 0; w < kClipThreads / 32; ++w) t += red[w];
  return t;
}

template <int N>
__global__ void __launch_bounds__(kClipThreads, 4)
grad_sqnorm_kernel(const __grid_constant__ ClipTable<N> t, double* __restrict__ partial) {
  __shared__ double red[kClipThreads / 32];
  double acc = 0.0;
  for (int chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
    const ClipEntry& e = t.e[entry_of(t, chunk)];
    const int dtype = e.dtypes & 0xFF;
    const long long n = e.count != nullptr ? min(e.n, static_cast<long long>(max(0, *e.count)) * e.unit) : e.n;
    const long long first = static_cast<long long>(chunk - e.chunk0) * kClipChunk - behind(e.src, dtype) + threadIdx.x * 8;
    if (first - static_cast<long long>(threadIdx.x) * 8 >= n) continue;
    float v[kClipSteps][8];
    load_chunk(e.src, first, n, dtype, v);
    double sum = 0.0;
#pragma unroll
    for (int s = 0; s < kClipSteps; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fma(static_cast<double>(v[s][j]), static_cast<double>(v[s][j]), sum);
    acc = fma(static_cast<double>(e.weight) * e.weight, sum, acc);
  }
  acc = block_sum(acc, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// result = {norm, coefficient}
template <int N>
__global__ void __launch_bounds__(kClipThreads, 4)
grad_clip_kernel(const __grid_constant__ ClipTable<N> t, const double* __restrict__ partial, int partials, double max_norm,
                 double eps, float* __restrict__ result) {
  __shared__ double red[kClipThreads / 32];
  double sum = 0.0;
  for (int i = threadIdx.x; i < partials; i += kClipThreads) sum += partial[i];
  const double norm = sqrt(block_sum(sum, red));
  const double ratio = max_norm / (norm + eps);
  const float coef = static_cast<float>(ratio > 1.0 ? 1.0 : ratio);       // (NaN stays)
  if (blockIdx.x == 0 && threadIdx.x == 0 && result != nullptr) {
    result[0] = static_cast<float>(norm);
    result[1] = coef;
  }
  for (int chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
    const ClipEntry& e = t.e[entry_of(t, chunk)];
    if (e.dst == e.src && coef == 1.f) continue;         // in place and nothing to clip
    const int from = e.dtypes & 0xFF, to = e.dtypes >> 8, shift = behind(e.src, from);
    const bool whole = ((reinterpret_cast<uintptr_t>(e.dst) - static_cast<uintptr_t>(shift) * size_of(to)) & 15) == 0;
    const long long first = static_cast<long long>(chunk - e.chunk0) * kClipChunk - shift + threadIdx.x * 8;
    float v[kClipSteps][8];
    load_chunk(e.src, first, e.n, from, v);
#pragma unroll
    for (int s = 0; s < kClipSteps; ++s) {
      const long long i = first + s * (kClipThreads * 8);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[s][j] *= coef;
      if (whole && i >= 0 && i + 8 <= e.n) {
        store8(e.dst, i, to, v[s]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (i + j >= 0 && i + j < e.n) store_one(e.dst, i + j, to, v[s][j]);
      }
    }
  }
}

// The tensors of a call.
struct GradList {
  int32_t count, dense;
  const void* const* grads;
  const int64_t* elems;
  const uint8_t* dtypes;
  void* const* out;
  const uint8_t* out_dtypes;
  const int32_t* const* counts;
  const int32_t* units;
  const float* weights;
};
int bytes_of(int dtype) { return dtype == MOC_F32 ? 4 : 2; }

// go(table, CTAs, CTAs of the launches before) for the tensors in runs of as many as a table holds, once at least
template <int N, typename Go>
int each_table(const GradList& g, bool write, Go go) {
  static thread_local ClipTable<N> t;              // (32 KB: not on the stack of a caller's thread)
  int32_t i = 0;
  int before = 0;
  const int32_t end = write ? g.dense : g.count;
  do {
    t.entries = 0;
    long long chunks = 0;
    for (; i < end && t.entries < N; ++i) {
      const bool dense = i < g.dense;
      if (g.elems[i] == 0 || (write && g.out[i] == nullptr)) continue;
      ClipEntry& e = t.e[t.entries++];
      e.src = g.grads[i]; e.n = g.elems[i];
      e.dst = dense ? g.out[i] : nullptr;
      e.dtypes = g.dtypes[i] | (dense ? g.out_dtypes[i] << 8 : 0);
      e.count = dense ? nullptr : g.counts[i - g.dense];
      e.unit = dense ? 0 : g.units[i - g.dense];
      e.weight = dense ? 1.f : g.weights[i - g.dense];
      e.chunk0 = static_cast<int>(chunks);
      const long long shift = static_cast<long long>((reinterpret_cast<uintptr_t>(g.grads[i]) & 15) / bytes_of(g.dtypes[i]));
      chunks += (e.n + shift + kClipChunk - 1) / kClipChunk;
      MOC_REQUIRE(chunks < (1ll << 30), "too many gradient elements in one call");
    }
    t.chunks = static_cast<int>(chunks);
    const int blocks = t.chunks < 1 ? 1 : t.chunks < kClipBlocks ? t.chunks : kClipBlocks;
    const int rc = go(t, blocks, before);
    if (rc != MOC_OK) return rc;
    before += blocks;
  } while (i < end);
  return MOC_OK;
}

template <int N>
int grad_clip(const GradList& g, double max_norm, double eps, float* result, double* partial, cudaStream_t stream) {
  int partials = 0;
  int rc = each_table<N>(g, false, [&](const ClipTable<N>& t, int blocks, int before) {
    grad_sqnorm_kernel<N><<<blocks, kClipThreads, 0, stream>>>(t, partial + before);
    MOC_CUDA_OK(cudaGetLastError());
    partials = before + blocks;
    return MOC_OK;
  });
  if (rc != MOC_OK) return rc;
  return each_table<N>(g, true, [&](const ClipTable<N>& t, int blocks, int before) {
    grad_clip_kernel<N><<<blocks, kClipThreads, 0, stream>>>(t, partial, partials, max_norm, eps, before == 0 ? result : nullptr);
    MOC_CUDA_OK(cudaGetLastError());
    return MOC_OK;
  });
}

// Memory that is written may be read as the same gradient (clipped in place) and by nothing else.
struct Span {
  uintptr_t first, end;
  bool written;
};
int check_overlaps(const GradList& g) {
  static thread_local Span spans[2 * 4096];
  int n = 0;
  const int most = static_cast<int>(sizeof(spans) / sizeof(spans[0]));
  for (int32_t i = 0; i < g.count; ++i) {
    if (g.elems[i] == 0) continue;
    MOC_REQUIRE(n + 2 <= most, "at most 4096 tensors in one call");
    const uintptr_t p = reinterpret_cast<uintptr_t>(g.grads[i]);
    void* o = i < g.dense ? g.out[i] : nullptr;
    spans[n++] = Span{p, p + static_cast<uintptr_t>(g.elems[i]) * bytes_of(g.dtypes[i]), o == g.grads[i]};
    if (o != nullptr && o != g.grads[i]) {
      const uintptr_t q = reinterpret_cast<uintptr_t>(o);
      spans[n++] = Span{q, q + static_cast<uintptr_t>(g.elems[i]) * bytes_of(g.out_dtypes[i]), true};
    }
  }
  std::sort(spans, spans + n, [](const Span& a, const Span& b) { return a.first < b.first; });
  // (the furthest end so far, of everything and of what is written)
  uintptr_t end = 0, end_written = 0;
  for (int i = 0; i < n; ++i) {
    MOC_REQUIRE(spans[i].first >= (spans[i].written ? end : end_written), "gradients (and out) must not overlap");
    end = std::max(end, spans[i].end);
    if (spans[i].written) end_written = std::max(end_written, spans[i].end);
  }
  return MOC_OK;
}

}  // namespace
}  // namespace moc

using namespace moc;

extern "C" int64_t moc_grad_clip_workspace_bytes(int32_t count) {
  if (count < 0) return -1;
  const int64_t per = count <= kFewEntries ? kFewEntries : kMostEntries;
  return (count / per + 1) * kClipBlocks * static_cast<int64_t>(sizeof(double));
}

extern "C" int moc_grad_clip(int32_t count, int32_t dense, const void* const* grads, const int64_t* elems, const uint8_t* dtypes,
                             void* const* out, const uint8_t* out_dtypes, const int32_t* const* counts, const int32_t* units,
                             const float* weights, double max_norm, double eps, float* result, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  MOC_REQUIRE(count >= 0 && dense >= 0 && dense <= count && result && workspace, "NULL gradient-clipping argument");
  MOC_REQUIRE((grads && elems && dtypes) || count == 0, "NULL gradient list");
  MOC_REQUIRE((out && out_dtypes) || dense == 0, "NULL list of outputs");
  MOC_REQUIRE((counts && units && weights) || dense == count, "NULL list of counts");
  MOC_REQUIRE(max_norm >= 0.0 && eps >= 0.0, "max_norm and eps must not be negative");
  MOC_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 7) == 0 && workspace_bytes >= moc_grad_clip_workspace_bytes(count),
              "gradient-clipping workspace too small");
  for (int32_t i = 0; i < count; ++i) {
    MOC_REQUIRE(elems[i] >= 0 && (elems[i] == 0 || grads[i]), "NULL gradient");
    MOC_REQUIRE(dtypes[i] <= MOC_F16 && (i >= dense || out_dtypes[i] <= MOC_F16), "unknown gradient dtype");
    MOC_REQUIRE(reinterpret_cast<uintptr_t>(grads[i]) % bytes_of(dtypes[i]) == 0 &&
                (i >= dense || reinterpret_cast<uintptr_t>(out[i]) % bytes_of(out_dtypes[i]) == 0), "gradients must be aligned to their type");
    MOC_REQUIRE(i >= dense || out[i] != grads[i] || out_dtypes[i] == dtypes[i], "a gradient clipped in place keeps its type");
    MOC_REQUIRE(i < dense || (units[i - dense] > 0 && counts[i - dense]), "compact rows need a unit and a count");
  }
  const GradList g{count, dense, grads, elems, dtypes, out, out_dtypes, counts, units, weights};
  const int rc = check_overlaps(g);
  if (rc != MOC_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  double* partial = static_cast<double*>(workspace);
  return count <= kFewEntries ? grad_clip<kFewEntries>(g, max_norm, eps, result, partial, st)
                              : grad_clip<kMostEntries>(g, max_norm, eps, result, partial, st);
}
