// Decode-time memory attention over a cache of projected bank rows held in 8 bits, and the cache's making.
//
// The cache is e4m3 values v8 with an fp32 scale for each block of `scale_rows` rows, KV head, and K or V.  A row's scale leaves the
// products, so the values go into them as they are stored (u_c: the weight of chapter c):
//   s_r = scale * u_c * ks_r * <q, K8[r]>,   out = sum_r softmax(s)_r * u_c * vs_r * V8[r]   (one joint softmax).
//
// Bound by HBM for a full batch (one byte an element), by latency for a few sequences.  On CUDA cores, and with fp16 matrix
// instructions, 64 sequences of 4,160 rows and 12 heads took 95 to 97 us, bound by issuing 500 to 550 instructions for every 32 rows of
// a head.  So the values go into e4m3 matrix instructions as they lie in memory, and the other operand is split into e4m3 terms:
//   q = q0 + q1 / 16 + q2 / 256 (scaled so that its largest element is 128 to 256: 12 bits each, 2^-25 of the largest at the least),
//   p = (p0 + p1 / 16 + p2 / 256) / 256 (12 bits, 2^-26 at the least), each four significant bits of what the terms before leave.
// The terms are columns of the same instruction, which has eight and one query would use one of them: four columns a query.  e4m3
// products sum up in fp32 as fp16's do (2^-22 of the magnitudes, measured).
//   - scores: A = 16 keys x 32 dims.  The order of the dims is free, so a lane's 16 bytes of its row are the A fragments of both
//     steps as they come; keys are taken in the order that leaves the probabilities' bytes in theirs.
//   - values: A = 16 dims x 32 rows, transposed on the way out of shared memory (8-bit matrix loads); B = the probabilities, brought
//     from the scores' layout by a 16-bit matrix transposition of byte pairs.  Row scales that differ within a unit go in
//     relative to the unit's largest.
// Each warp has a ring of units (32 rows, K and V of one KV head) that bulk tensor copies fill two units ahead.  Maxima, sums and
// accumulators are fp32.  All queries on a KV head (its heads, the tokens of the step) share a row's fetch, up to eight a CTA.  A cluster
// of CTAs takes the units of one (sequence, KV head) in turns, warp by warp; parts merge through shared memory, then distributed
// shared memory.
#define MOC_KERNEL_TAG 7
#include <cuda_fp16.h>

#include "host_pass.cuh"

namespace moc {
namespace {

constexpr int kDD = 64, kThreads = 256, kWarps = kThreads / 32, kRows = 32;      // rows of a unit
constexpr float kLog2e = 1.4426950408889634f;

struct Attn8Params {
  const __nv_bfloat16* q;
  const float* scales;                 // [bank_rows / scale_rows, 2 * HK]
  long long bank_rows;
  const int* comb_idx;
  const float* comb_w;
  const int* counts;                   // chapters of each list that count (NULL: all)
  __nv_bfloat16* out;
  float* lse;
  int n_q, H, HK, n_ch, T, split, tiles;        // tiles of queries of a KV head
  float scale;
  FastDiv scale_rows, runs;
  int* status;
};

// D = A B, A 16 x 32 and B 32 x 8 of e4m3
__device__ __forceinline__ void mma_e4m3_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two 16 x 16 byte matrices, transposed: lane l gives row l (of the first for l < 16); A fragment of columns 0..15 x rows 0..31
__device__ __forceinline__ void ldsm_bytes_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared::cta.b8 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {           // of a warp's 8 x 8 matrix of 16-bit values
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {    // in the low 16 bits
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 of_e4m3x2(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(two)));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// x, y (at most 448) as three e4m3 terms each, the second times 16 and the third times 256
__device__ __forceinline__ void split_e4m3(float x, float y, uint32_t (&term)[3]) {
  term[0] = to_e4m3x2(x, y);
  float2 t = of_e4m3x2(term[0]);
  x = (x - t.x) * 16.f; y = (y - t.y) * 16.f;
  term[1] = to_e4m3x2(x, y);
  t = of_e4m3x2(term[1]);
  term[2] = to_e4m3x2((x - t.x) * 16.f, (y - t.y) * 16.f);
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

constexpr int kStages = 3, kUnitBytes = 2 * kRows * kDD;
constexpr int kShared = kWarps * kStages * kUnitBytes + 1024;          // (tiles start on 1,024 bytes)

// NT: tiles of 8 columns, two queries each.  Lane (g, t) = (lane / 4, lane % 4).
template <int NT>
__global__ void __launch_bounds__(kThreads, NT <= 2 ? 2 : 1)
decode_attn8_kernel(const __grid_constant__ CUtensorMap map, const Attn8Params p) {
  constexpr int kCols = 2 * NT;        // queries
  extern __shared__ char raw_ring[];
  __shared__ __align__(8) uint64_t full[kWarps][kStages];
  __shared__ int abort_flag;
  __shared__ __align__(16) float cta_part[kCols][kDD + 4];        // accumulator, maximum, sum of this CTA
  char* ring = raw_ring + (1024 - (smem_u32(raw_ring) & 1023)) % 1024;
  float (*red)[kWarps][kDD + 4] = reinterpret_cast<float (*)[kWarps][kDD + 4]>(ring);       // once the rings are done with
  const int split = p.split, HK = p.HK, T = p.T;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int rank = static_cast<int>(blockIdx.x) % split, tile = static_cast<int>(blockIdx.x) / split % p.tiles;
  const int kh = static_cast<int>(blockIdx.x) / split / p.tiles, b = blockIdx.y;
  const int per_kv = p.H / HK, columns = min(kCols, p.n_q * per_kv - tile * kCols);      // query j: token j / per_kv, head kh per_kv + j % per_kv
  auto q_row = [&](int col) {
    const int j = tile * kCols + col, iq = j / per_kv;
    return (static_cast<long long>(b) * p.n_q + iq) * p.H + kh * per_kv + (j - iq * per_kv);
  };
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int i = 0; i < kWarps * kStages; ++i) mbar_init(&full[0][0] + i, 1);
    fence_mbar_init();
    prefetch_tmap(&map);
  }
  __syncthreads();
  int n_ch = p.n_ch;
  if (p.counts != nullptr) n_ch = max(0, min(n_ch, p.counts[b]));
  const int* list = p.comb_idx + static_cast<long long>(b) * p.n_ch;
  const float* weights = p.comb_w + static_cast<long long>(b) * p.n_ch;
  const int total = n_ch * p.runs.d, stride = split * kWarps, first = rank * kWarps + warp;
  auto known = [&](int ch) { return ch >= 0 && (static_cast<long long>(ch) + 1) * T <= p.bank_rows; };
  char* stages = ring + warp * kStages * kUnitBytes;

  auto fetch = [&](int unit, int stage) {          // by one lane
    if (unit >= total) return;
    const int c = div_of(unit, p.runs), ch = list[c];
    if (!known(ch)) {
      atomicMax(p.status, MOC_DEV_BAD_INDEX);
      mbar_arrive(&full[warp][stage]);
      return;
    }
    const int row = ch * T + (unit - c * p.runs.d) * kRows;
    mbar_arrive_expect_tx(&full[warp][stage], kUnitBytes);
    tma_load_2d(stages + stage * kUnitBytes, &map, &full[warp][stage], kh * kDD, row);
    tma_load_2d(stages + stage * kUnitBytes + kRows * kDD, &map, &full[warp][stage], (HK + kh) * kDD, row);
  };
  if (lane == 0)
    for (int i = 0; i < kStages - 1; ++i) fetch(first + i * stride, i);

  // a unit's factors, fetched one unit ahead: of this lane's rows 16 mt + 2 g + h, i = 2 mt + h (one block of scales: the first)
  const bool one_block = p.scale_rows.d % kRows == 0;
  struct Factors {
    float u, k[4], v[4];
    int r0;                            // first row within the chapter; -1: unknown chapter
  };
  auto factors_of = [&](int unit, Factors& f) {
    if (unit >= total) return;
    const int c = div_of(unit, p.runs), ch = list[c];
    f.u = weights[c];
    f.r0 = known(ch) ? (unit - c * p.runs.d) * kRows : -1;
    if (f.r0 < 0) return;
    const float* sc = p.scales + static_cast<long long>(ch) * (T / p.scale_rows.d) * 2 * HK + kh;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (one_block && i > 0) { f.k[i] = f.k[0]; f.v[i] = f.v[0]; continue; }
      const int r = one_block ? f.r0 : f.r0 + 16 * (i >> 1) + 2 * g + (i & 1);
      const float* at = sc + static_cast<long long>(div_of(r < T ? r : 0, p.scale_rows)) * 2 * HK;
      f.k[i] = at[0];
      f.v[i] = at[HK];
    }
  };
  Factors now{}, next{};
  factors_of(first, now);

  // queries: B fragments (column g = term g % 4 of query g / 4; dims 16 t + 8 s + {0..3} and {4..7} in step s), and what this
  // lane's two score columns count: the even one of a query's pair of lanes has the first two terms, the odd one the third
  uint32_t qb[NT][2][2];
  float fa[NT], fb[NT], acc[NT][4][4], m[NT], l[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float f[16], top = 0.f;
    const int col = 2 * nt + (g >> 2);
    const uint4* src = reinterpret_cast<const uint4*>(p.q + q_row(col < columns ? col : 0) * kDD + 16 * t);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 raw = src[h];
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[8 * h + 2 * i] = __uint_as_float(w[i] << 16);
        f[8 * h + 2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max_nan(top, fabsf(f[i]));
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = static_cast<int>(__float_as_uint(top) >> 23);          // of 2^(e - 127); queries below 2^-99 count as zero
    const float up = e > 27 && e < 255 ? __uint_as_float(static_cast<uint32_t>(261 - e) << 23) : 0.f;       // 2^(134 - e)
    float down = e > 27 ? __uint_as_float(static_cast<uint32_t>(e - 7) << 23) : 0.f;
    if (e == 255) down = NAN;                                            // (infinite or NaN queries: every score NaN)
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t lo[3], hi[3];
        const float* x = f + 8 * s + 4 * h;
        split_e4m3(up > 0.f ? x[0] * up : 0.f, up > 0.f ? x[1] * up : 0.f, lo);
        split_e4m3(up > 0.f ? x[2] * up : 0.f, up > 0.f ? x[3] * up : 0.f, hi);
        const int term = g & 3;
        const uint32_t a = term == 0 ? lo[0] : term == 1 ? lo[1] : lo[2], c = term == 0 ? hi[0] : term == 1 ? hi[1] : hi[2];
        qb[nt][s][h] = term == 3 || col >= columns ? 0u : a | c << 16;
      }
    const float factor = __shfl_sync(0xffffffffu, down, (t >> 1) * 16) * p.scale * kLog2e;
    fa[nt] = t & 1 ? factor * (1.f / 256.f) : factor;
    fb[nt] = t & 1 ? 0.f : factor * (1.f / 16.f);
    m[nt] = -INFINITY;
    l[nt] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[nt][i][j] = 0.f;
  }

  int stage = 0;
  uint32_t phase = 0;
  const uint32_t k_at = 2 * g * kDD + ((t ^ (g & 3)) << 4);            // rows 2 g (and 2 g + 1, 64 bytes on), piece t, swizzled
  for (int unit = first; unit < total; unit += stride) {
    if (lane == 0) fetch(unit + (kStages - 1) * stride, stage == 0 ? kStages - 1 : stage - 1);
    factors_of(unit + stride, next);
    const bool alive = mbar_wait_w(&full[warp][stage], phase, &abort_flag, p.status);
    if (!alive) {                          // the copies still on their way land before the bytes change owner, or as long again passes
      for (int i = 0, at = stage; i < kStages && unit + i * stride < total; ++i) {
        for (uint32_t it = 0; it < kWaitPollLimit && !mbar_try_wait(&full[warp][at], phase); ++it) {}
        if (++at == kStages) { at = 0; phase ^= 1; }
      }
      break;
    }
    char* kt = stages + stage * kUnitBytes;
    char* vt = kt + kRows * kDD;
    if (++stage == kStages) { stage = 0; phase ^= 1; }
    if (now.r0 >= 0) {
      if (now.r0 + kRows > T) {            // rows of the next chapter: their values may be NaN, and meet probabilities of 0
        if (now.r0 + lane >= T) {
#pragma unroll
          for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(vt + lane * kDD + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async();               // (before the next copy into these bytes)
        __syncwarp();
      }
      float kf[4], vf[4], w_top;
      if (one_block) {
        w_top = now.v[0];
#pragma unroll
        for (int i = 0; i < 4; ++i) { kf[i] = now.k[0] * now.u; vf[i] = 256.f; }
      } else {
        w_top = max_nan(max_nan(now.v[0], now.v[1]), max_nan(now.v[2], now.v[3]));
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) w_top = max_nan(w_top, __shfl_xor_sync(0xffffffffu, w_top, o));
        const float inv = w_top > 0.f ? 256.f / w_top : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) { kf[i] = now.k[i] * now.u; vf[i] = now.v[i] * inv; }
      }
      w_top *= now.u * (1.f / 256.f);
      uint32_t kr[2][2][4];                // [mt][h]: rows 16 mt + 2 g + h, bytes 16 t ..
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 v = *reinterpret_cast<const uint4*>(kt + 16 * mt * kDD + k_at + h * kDD);
          kr[mt][h][0] = v.x; kr[mt][h][1] = v.y; kr[mt][h][2] = v.z; kr[mt][h][3] = v.w;
        }
      uint32_t pb[NT][2];                  // probabilities as B fragments: rows 4 t .. 4 t + 3 and 16 on, column g
      float corr[NT];
      bool moved = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float s[4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          float d[4];
          mma_e4m3_new(d, kr[mt][0][0], kr[mt][1][0], kr[mt][0][1], kr[mt][1][1], qb[nt][0][0], qb[nt][0][1]);
          mma_e4m3(d, kr[mt][0][2], kr[mt][1][2], kr[mt][0][3], kr[mt][1][3], qb[nt][1][0], qb[nt][1][1]);
#pragma unroll
          for (int h = 0; h < 2; ++h) s[2 * mt + h] = fmaf(d[2 * h + 1], fb[nt], d[2 * h] * fa[nt]);
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[i] = (s[i] + __shfl_xor_sync(0xffffffffu, s[i], 1)) * kf[i];
          if (now.r0 + 16 * (i >> 1) + 2 * g + (i & 1) >= T) s[i] = -INFINITY;
          top = fmaxf(top, s[i]);
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float m_new = fmaxf(m[nt], top), ref = m_new == -INFINITY ? 0.f : m_new;
        corr[nt] = exp2_fast(m[nt] - ref);               // 0 on the first rows (m = -inf)
        moved |= m_new != m[nt];
        m[nt] = m_new;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[i] = exp2_fast(s[i] - ref);
          sum += s[i];
        }
        l[nt] = fmaf(l[nt], corr[nt], sum);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          uint32_t term[3];
          split_e4m3(s[2 * mt] * vf[2 * mt], s[2 * mt + 1] * vf[2 * mt + 1], term);
          pb[nt][mt] = transpose8(t & 1 ? term[2] : term[0] | term[1] << 16);
        }
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          // (lane (g, t) has the column pair t in its accumulators: the maximum is that of the same query)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[nt][i][j] *= corr[nt];
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {        // dims 16 i + g and + 8
        uint32_t a[4];
        ldsm_bytes_t(a, smem_u32(vt) + lane * kDD + ((i ^ ((lane >> 1) & 3)) << 4));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float d[4];
          mma_e4m3_new(d, a[0], a[1], a[2], a[3], pb[nt][0], pb[nt][1]);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[nt][i][j] = fmaf(w_top, d[j], acc[nt][i][j]);
        }
      }
    }
    now = next;
    __syncwarp();                          // the ring's place is free from here on
  }
  __syncthreads();
  if (abort_flag) {                        // (reported in the status word; the same for the whole CTA)
    if (split > 1) { cluster_sync(); cluster_sync(); }
    return;
  }
  // a warp's part, the terms summed: query 2 nt + t / 2
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float sum = l[nt];
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    float* to = red[2 * nt + (t >> 1)][warp];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v = t & 1 ? acc[nt][i][2 * h] * (1.f / 256.f) : fmaf(acc[nt][i][2 * h + 1], 1.f / 16.f, acc[nt][i][2 * h]);
        v += __shfl_xor_sync(0xffffffffu, v, 1);
        if (!(t & 1)) to[16 * i + 8 * h + g] = v;
      }
    if (g == 0 && !(t & 1)) {
      to[kDD] = m[nt];
      to[kDD + 1] = sum;
    }
  }
  __syncthreads();
  // warps -> CTA: thread i finishes output element i % 64 of column i / 64
  for (int i = threadIdx.x; i < columns * kDD; i += kThreads) {
    const int col = i / kDD, e = i % kDD;
    float mt = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, red[col][w][kDD]);
    float lt = 0.f, a = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = (red[col][w][kDD] == -INFINITY) ? 0.f : exp2f(red[col][w][kDD] - mt);
      // (a warp whose scores are all NaN has no maximum, but a sum that is NaN)
      lt += red[col][w][kDD] == -INFINITY && red[col][w][kDD + 1] == 0.f ? 0.f : red[col][w][kDD + 1] * f;
      a += red[col][w][e] * f;
    }
    cta_part[col][e] = a;
    if (e == 0) { cta_part[col][kDD] = mt; cta_part[col][kDD + 1] = lt; }
  }
  // CTAs -> output: the cluster's first CTA reads the others' parts (one of its own needs no barrier beyond the CTA's)
  if (split > 1) cluster_sync(); else __syncthreads();
  if (rank == 0) {
    for (int i = threadIdx.x; i < columns * kDD; i += kThreads) {
      const int col = i / kDD, e = i % kDD;
      const uint32_t stat = smem_u32(&cta_part[col][kDD]), elem = smem_u32(&cta_part[col][e & ~1]);
      float mt = -INFINITY, lt = 0.f, a = 0.f;
      for (int r = 0; r < split; ++r) {
        const float2 st = split > 1 ? cluster_ld2(cluster_map(stat, r)) : make_float2(cta_part[col][kDD], cta_part[col][kDD + 1]);
        const float2 ab = split > 1 ? cluster_ld2(cluster_map(elem, r)) : make_float2(cta_part[col][e & ~1], cta_part[col][e | 1]);
        const float m_new = fmaxf(mt, st.x);
        const float f0 = mt == -INFINITY ? 0.f : exp2f(mt - m_new), f1 = st.x == -INFINITY ? 0.f : exp2f(st.x - m_new);
        lt = lt * f0 + st.y * f1;
        a = a * f0 + ((e & 1) ? ab.y : ab.x) * f1;
        mt = m_new;
      }
      const bool any = lt != 0.f;                // (a list without rows has no sum; a NaN in the cache or the query stays one)
      p.out[q_row(col) * kDD + e] = __float2bfloat16(any ? a / lt : 0.f);
      if (e == 0 && p.lse != nullptr) p.lse[q_row(col)] = any ? (mt + log2f(lt)) / kLog2e : -INFINITY;
    }
  }
  if (split > 1) cluster_sync();       // nobody leaves while its part is read
}

__device__ __forceinline__ void unpack8(const uint4& v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

// values = e4m3(x / scale), scale = (largest |x|) / 448 of each block of `block` rows and one head of 64 columns; a warp takes a
// block, eight lanes a row (16 bytes of its 128 each), four rows a load.  Blocks of up to 4 R rows stay in registers; longer ones
// are read a second time.  A block of zeros has scale 0 and values 0; one with a NaN or an infinity gets a scale that is
// NaN or infinite and stands for NaN as a whole.  Bound by HBM (2 bytes read and 1 written an element) once the quotient is a product
// corrected by its remainder (Markstein), equal to the division where its last bit can matter: 262,208 x 1,536: 371 us with
// divisions, 245 with products.
template <int R>
__global__ void __launch_bounds__(kThreads)
quantize_rows_kernel(const __nv_bfloat16* __restrict__ x, long long tiles, int heads, int block, uint8_t* __restrict__ values,
                     float* __restrict__ scales) {
  const long long tile = static_cast<long long>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (tile >= tiles) return;
  const int lane = threadIdx.x & 31, rg = lane >> 3, part = lane & 7;
  const long long blk = tile / heads;
  const int head = static_cast<int>(tile - blk * heads);
  const long long width = static_cast<long long>(heads) * kDD, first = blk * block * width + head * kDD + part * 8;
  uint4 raw[R];
  uint32_t top2 = 0;                 // magnitudes order like their bits, NaN above infinity; two columns at a time
  auto most = [&](uint32_t v) { asm("max.u16x2 %0, %0, %1;" : "+r"(top2) : "r"(v & 0x7FFF7FFFu)); };
  for (int r0 = 0; r0 < block; r0 += 4 * R) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = r0 + 4 * i + rg;
      raw[i] = r < block ? __ldcs(reinterpret_cast<const uint4*>(x + first + r * width)) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) { most(raw[i].x); most(raw[i].y); most(raw[i].z); most(raw[i].w); }
  }
  const uint32_t bits = __reduce_max_sync(0xffffffffu, max(top2 & 0xFFFFu, top2 >> 16));
  const float scale = __uint_as_float(bits << 16) * (1.f / 448.f);       // (a product, as torch divides by a constant: the last bit follows it)
  if (lane == 0) scales[tile] = scale;
  // A quotient of the correction below its range (x < 2^-100) rounds to 0 all the same while the scale is above 2^-80.
  const bool plain = scale > 0x1p-80f && scale < 0x1p80f;
  const float inv = plain ? 1.f / scale : 0.f;
  for (int r0 = 0; r0 < block; r0 += 4 * R) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = r0 + 4 * i + rg;
      if (r >= block) continue;
      if (block > 4 * R) raw[i] = *reinterpret_cast<const uint4*>(x + first + r * width);
      float f[8];
      unpack8(raw[i], f);
      if (plain) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float q = f[j] * inv;
          f[j] = fmaf(fmaf(-q, scale, f[j]), inv, q);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = scale > 0.f ? f[j] / scale : 0.f;
      }
      uint32_t w[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        asm("{\n\t.reg .b16 a, b;\n\tcvt.rn.satfinite.e4m3x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 b, %4, %3;\n\t"
            "mov.b32 %0, {a, b};\n\t}"
            : "=r"(w[j]) : "f"(f[4 * j]), "f"(f[4 * j + 1]), "f"(f[4 * j + 2]), "f"(f[4 * j + 3]));
      __stcs(reinterpret_cast<uint2*>(values + first + r * width), make_uint2(w[0], w[1]));
    }
  }
}

}  // namespace

int decode_attn_e4m3(const moc_decode_shape* s, const void* q, const void* values, const float* scales, int scale_rows, int64_t bank_rows,
                     const int32_t* comb_idx, const float* comb_w, const int32_t* counts, void* out, float* lse, int32_t* status,
                     void* stream) {
  MOC_REQUIRE(s && q && values && scales && comb_idx && comb_w && out && status, "NULL decode-attention argument");
  MOC_REQUIRE(s->head_dim == kDD, "decode attention needs head_dim 64");
  MOC_REQUIRE(s->batch > 0 && s->n_q > 0 && s->n_chapters > 0 && s->tokens_per_chapter > 0 && bank_rows > 0, "empty decode-attention problem");
  MOC_REQUIRE(s->num_heads > 0 && s->num_kv_heads > 0 && s->num_heads % s->num_kv_heads == 0,
              "num_heads must be a positive multiple of num_kv_heads");
  MOC_REQUIRE(scale_rows > 0 && s->tokens_per_chapter % scale_rows == 0, "a chapter must be whole blocks of scale_rows");
  MOC_REQUIRE(s->n_q <= 65535 && s->batch <= 65535, "too many query tokens or sequences for one launch");
  MOC_REQUIRE(bank_rows < (1ll << 31), "the 8-bit cache takes fewer than 2^31 rows");
  MOC_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(values)) & 15) == 0, "q and the K/V cache must be 16-byte aligned");
  const long long columns = static_cast<long long>(s->n_q) * (s->num_heads / s->num_kv_heads);
  const int nt = columns <= 2 ? 1 : columns <= 4 ? 2 : 4, runs = ceil_div(s->tokens_per_chapter, kRows);
  const long long tiles = (columns + 2 * nt - 1) / (2 * nt), units = static_cast<long long>(s->n_chapters) * runs;
  MOC_REQUIRE(tiles * s->num_kv_heads < (1ll << 27) && units < (1ll << 30), "decode-attention problem too large for one launch");
  CUtensorMap map;
  const int rc = make_tmap_u8_2d(&map, values, static_cast<uint64_t>(bank_rows), 2ull * s->num_kv_heads * kDD, kRows);
  if (rc != MOC_OK) return rc;
  auto kern = nt == 1 ? decode_attn8_kernel<1> : nt == 2 ? decode_attn8_kernel<2> : decode_attn8_kernel<4>;
  static_assert(kShared - 1024 >= 8 * kWarps * (kDD + 4) * 4, "the warps' parts fit the rings");
  MOC_CUDA_OK(allow_shared(kern, kShared, kShared));
  // Clusters of 1 to 8 CTAs for each (sequence, KV head, tile of queries): the fewest units in a row, counting three for a CTA's start
  // and end, over the rounds in which all of them run.
  const long long groups = tiles * s->num_kv_heads * s->batch;
  int split = 1;
  long long best = 0;
  for (int n = 1; n <= 8; n *= 2) {
    const long long resident = n == 1 ? (nt <= 2 ? 2 : 1) * 148 : resident_clusters(kern, kThreads, kShared, n);
    if (resident == 0) continue;
    const long long cost = (groups + resident - 1) / resident * ((units + n * kWarps - 1) / (n * kWarps) + 3);
    if (best == 0 || cost < best) { best = cost; split = n; }
  }
  Attn8Params p{};
  p.q = static_cast<const __nv_bfloat16*>(q); p.scales = scales; p.bank_rows = bank_rows;
  p.comb_idx = comb_idx; p.comb_w = comb_w; p.counts = counts; p.out = static_cast<__nv_bfloat16*>(out); p.lse = lse;
  p.n_q = s->n_q; p.H = s->num_heads; p.HK = s->num_kv_heads; p.n_ch = s->n_chapters; p.T = s->tokens_per_chapter;
  p.split = split; p.tiles = static_cast<int>(tiles); p.scale = s->scale; p.scale_rows = fast_div(scale_rows); p.runs = fast_div(runs);
  p.status = status;
  MOC_CUDA_OK(launch_clustered(kern, dim3(static_cast<unsigned>(tiles) * s->num_kv_heads * split, s->batch), kThreads, kShared, split,
                               static_cast<cudaStream_t>(stream), map, p));
  MOC_CUDA_OK(cudaGetLastError());
  return MOC_OK;
}

}  // namespace moc

using namespace moc;

extern "C" int moc_quantize_rows(const void* rows_bf16, int64_t rows, int32_t heads, int32_t head_dim, int32_t scale_rows,
                                 void* values, float* scales, void* stream) {
  MOC_REQUIRE(rows_bf16 && values && scales, "NULL quantisation buffer");
  MOC_REQUIRE(head_dim == kDD, "the 8-bit cache needs head_dim 64");
  MOC_REQUIRE(rows > 0 && heads > 0 && scale_rows > 0 && rows % scale_rows == 0, "rows must be whole blocks of scale_rows");
  MOC_REQUIRE(((reinterpret_cast<uintptr_t>(rows_bf16) | reinterpret_cast<uintptr_t>(values)) & 15) == 0,
              "rows and values must be 16-byte aligned");
  const long long tiles = rows / scale_rows * heads;
  MOC_REQUIRE(tiles < (1ll << 33), "too many blocks in one call");
  const unsigned grid = static_cast<unsigned>((tiles + kWarps - 1) / kWarps);
  auto kern = scale_rows <= 8 ? quantize_rows_kernel<2> : scale_rows <= 16 ? quantize_rows_kernel<4>
              : scale_rows <= 32 ? quantize_rows_kernel<8> : quantize_rows_kernel<16>;
  kern<<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const __nv_bfloat16*>(rows_bf16), tiles, heads, scale_rows,
                                                                static_cast<uint8_t*>(values), scales);
  MOC_CUDA_OK(cudaGetLastError());
  return MOC_OK;
}
