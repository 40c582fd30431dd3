// Decode-time memory attention over a cache of projected bank rows held in 8 bits, and the cache's making.
//
// The cache is e4m3 values v8 with an fp32 scale for each block of `scale_rows` rows, KV head, and K or V.  A row's scale leaves the
// products, so the values go into them as they are stored (u_c: the weight of chapter c):
//   s_r = scale * u_c * ks_r * <q, K8[r]>,   out = sum_r softmax(s)_r * u_c * vs_r * V8[r]   (one joint softmax).
//
// A full batch should be bound by HBM (one byte an element) and is bound by latency and issuing; a few sequences by latency.  All
// queries on a KV head (its heads, the tokens of the step) are the columns of one matrix instruction, so a row is fetched and converted
// once for up to 16 of them; e4m3 -> fp16 is exact.  64 sequences of 4,160 rows, 12 heads: 71 us (3.8 TB/s of HBM, 6.3 from L2's side;
// 356 instructions a unit of 32 rows at 0.53 a cycle and scheduler, 24 warps on an SM); 13 sequences of 3 tokens, 12 heads on 4, 47
// chapters of 64 rows: 17 us from launch to launch; one sequence of 4,160 rows, 12 heads: 10 us.  Measured on the way, of these kernels'
// own stages, with one term of the probabilities: on CUDA cores 95 us against 97 and 19 against 16; units by bulk tensor copies into a ring 99 against 92; e4m3 matrix instructions of single
// warps (16 of them take 175 instructions, fp16 ones 66: they convert too), queries and probabilities in three terms, 102 against 97 and
// 33 against 16; the next unit's rows in registers too, with 16 warps on an SM, 79 against 70; 32 warps at 64 registers 90 against 70.
//   - scores: A = 16 keys x 16 dims, B = dims x 8 queries.  The order of the dims is free, so a lane's 16 bytes of its row are
//     the A fragments of four steps as they come.  Queries are scaled by a power of two into fp16's range (their largest to
//     128..256; what falls below fp16's smallest number is 2^-31 of the largest).
//   - values: A = 16 dims x 16 rows, transposed from rows by byte permutations within a lane; B = the probabilities, which a matrix
//     transposition brings from the scores' layout.  They go in as two fp16 terms (the second in the odd columns where those are idle,
//     else by instructions of its own): 2^-21 of their own, not below 2^-32 of the largest.  With one term results that cancel lose
//     their last bits and one in ten elements rounds to the neighbouring bf16 number; it costs 70.7 us against 70.3 (64 sequences,
//     12 heads of their own), 25.1 against 23.7 (six queries a KV head), 16.8 against 16.5 (nine queries, scales of 16 rows).  Row scales that differ within a unit go in relative to the unit's largest.
// The softmax's reference of a column is a score already met; it moves to the largest only when a score passes it by 2^8, which saves
// most units the reduction across lanes and the rescaling (92 us with, 97 without, before the steps on addresses).  References, sums
// and accumulators are fp32.  A cluster of CTAs takes the units of one (sequence, KV head) in turns, warp by warp; parts merge through
// shared memory, then distributed shared memory.
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

#include "host_pass.cuh"

namespace moc {
namespace {

constexpr int kDD = 64, kThreads = 256, kWarps = kThreads / 32, kRows = 32;      // rows of a unit
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kHeadroom = 8.f;       // a score may pass its column's reference by 2^8 before that moves
constexpr float kLift = 128.f;         // on probabilities on their way into fp16: at most 2^8 of them, so 2^15 of 65,504; normal from 2^-21 on

struct Attn8Params {
  const __nv_bfloat16* q;
  const uint8_t* values;
  const float* scales;                 // [bank_rows / scale_rows, 2 * HK]
  int chapters;                        // of the cache
  const int* comb_idx;
  const float* comb_w;
  const int* counts;                   // chapters of each list that count (NULL: all)
  __nv_bfloat16* out;
  float* lse;
  int n_q, H, HK, n_ch, T, split, tiles, blocks;       // tiles of columns of a KV head; blocks of scales of a chapter
  float scale;
  FastDiv scale_rows, runs;
  int* status;
};

__device__ __forceinline__ uint32_t e4m3x2_to_f16(uint32_t two) {       // the low 16 bits
  uint32_t r;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16_high(uint32_t two) {
  uint32_t r;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, b;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
// D = A B + D of fp16, A 16 x 16, B 16 x 8 (_new: D = A B)
__device__ __forceinline__ void mma_f16_new(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {           // of a warp's 8 x 8 matrix of 16-bit values
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// x = first + rest to 2^-21 of x (2^-25 where x is below fp16's normal range): both go into the products
__device__ __forceinline__ float leading11(float x) { return __uint_as_float(__float_as_uint(x) & 0xFFFFE000u); }
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// NT: tiles of 8 columns.  Lane (g, t) = (lane / 4, lane % 4) has the scores of columns 2 t and 2 t + 1; NJ = 1: up to four queries take
// the even ones and the odd ones' work is left out (one query a KV head: 84 us against 92, likewise).
template <int NT, int NJ>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 3 : 2)
decode_attn8_kernel(const Attn8Params p) {
  constexpr int kCols = 4 * NJ * NT;
  __shared__ __align__(16) float red[kCols][kWarps][kDD + 4];
  __shared__ __align__(16) float cta_part[kCols][kDD + 4];        // accumulator, maximum, sum of this CTA
  const int split = p.split, HK = p.HK, T = p.T;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int rank = static_cast<int>(blockIdx.x) % split, tile = static_cast<int>(blockIdx.x) / split % p.tiles;
  const int kh = static_cast<int>(blockIdx.x) / split / p.tiles, b = blockIdx.y;
  const int per_kv = p.H / HK, columns = min(kCols, p.n_q * per_kv - tile * kCols);      // column j: token j / per_kv, head kh per_kv + j % per_kv
  const int row_bytes = 2 * HK * kDD;
  auto q_row = [&](int col) {
    const int j = tile * kCols + col, iq = j / per_kv;
    return (static_cast<long long>(b) * p.n_q + iq) * p.H + kh * per_kv + (j - iq * per_kv);
  };
  int n_ch = p.n_ch;
  if (p.counts != nullptr) n_ch = max(0, min(n_ch, p.counts[b]));
  const int* list = p.comb_idx + static_cast<long long>(b) * p.n_ch;
  const float* weights = p.comb_w + static_cast<long long>(b) * p.n_ch;

  // queries: B fragments (column g, dims 16 t + 4 s + {0, 1} and {2, 3} in step s), and the factors of this lane's score columns
  uint32_t qb[NT][4][2];
  float factor[NT][NJ], acc[NT][4][2][NJ], m[NT][NJ], l[NT][NJ];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float f[16], top = 0.f;
    const int col = NJ == 2 ? nt * 8 + g : g & 1 ? kCols : g >> 1;
    const uint4* src = reinterpret_cast<const uint4*>(p.q + q_row(col < columns ? col : 0) * kDD + 16 * t);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 raw = src[h];
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[8 * h + 2 * i] = col < columns ? __uint_as_float(w[i] << 16) : 0.f;
        f[8 * h + 2 * i + 1] = col < columns ? __uint_as_float(w[i] & 0xFFFF0000u) : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(f[i]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = static_cast<int>(__float_as_uint(top) >> 23);          // of 2^(e - 127); infinite queries and tiny ones stay as they are
    const bool shift = e > 27 && e < 255;
    const float up = shift ? __uint_as_float(static_cast<uint32_t>(261 - e) << 23) : 1.f;       // 2^(134 - e)
    const float down = shift ? __uint_as_float(static_cast<uint32_t>(max(e - 7, 1)) << 23) : 1.f;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      qb[nt][s][0] = pack_f16(f[4 * s] * up, f[4 * s + 1] * up);
      qb[nt][s][1] = pack_f16(f[4 * s + 2] * up, f[4 * s + 3] * up);
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      factor[nt][j] = __shfl_sync(0xffffffffu, down, (2 * t + j) * 4) * p.scale * kLog2e;
      m[nt][j] = -INFINITY;
      l[nt][j] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[nt][i][0][j] = acc[nt][i][1][j] = 0.f;
  }

  const bool one_block = p.scale_rows.d % kRows == 0;          // a unit lies in one block of scales
  const int units = n_ch * p.runs.d, stride = split * kWarps;
  int next_ch = 0, next_r0 = 0;                  // of the unit that follows, fetched while one is worked on
  float next_u = 0.f;
  auto look_up = [&](int unit) {
    if (unit < units) {
      const int c = div_of(unit, p.runs);
      next_r0 = (unit - c * p.runs.d) * kRows;
      next_ch = list[c];
      next_u = weights[c];
    }
  };
  look_up(rank * kWarps + warp);
  for (int unit = rank * kWarps + warp; unit < units; unit += stride) {
    const int ch = next_ch, r0 = next_r0;
    const float u = next_u;
    if (static_cast<unsigned>(ch) >= static_cast<unsigned>(p.chapters)) {
      if (lane == 0) atomicMax(p.status, MOC_DEV_BAD_INDEX);
      look_up(unit + stride);
      continue;
    }
    const bool whole = r0 + kRows <= T;
    const uint8_t* rows = p.values + (static_cast<long long>(ch) * T + r0) * row_bytes + kh * kDD;
    uint4 kr[2][2];                    // rows 16 mt + g and + 8, bytes 16 t ..
    uint2 vr[2][4];                    // rows 16 ks + {2 t, 2 t + 1, 2 t + 8, 2 t + 9}, bytes 8 g ..
    if (whole) {
      const uint8_t* k_at = rows + (g * row_bytes + 16 * t);
      const uint8_t* v_at = rows + (2 * t * row_bytes + HK * kDD + 8 * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) kr[i >> 1][i & 1] = *reinterpret_cast<const uint4*>(k_at + 8 * i * row_bytes);
#pragma unroll
      for (int i = 0; i < 8; ++i) vr[i >> 2][i & 3] = *reinterpret_cast<const uint2*>(v_at + ((i & 1) + 8 * (i >> 1)) * row_bytes);
    } else {                           // (what lies behind the chapter: its last row again, whose probability is 0)
      const int last = T - 1 - r0;
#pragma unroll
      for (int i = 0; i < 4; ++i) kr[i >> 1][i & 1] = *reinterpret_cast<const uint4*>(rows + min(8 * i + g, last) * row_bytes + 16 * t);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        vr[i >> 2][i & 3] = *reinterpret_cast<const uint2*>(rows + min((i & 1) + 8 * (i >> 1) + 2 * t, last) * row_bytes + HK * kDD + 8 * g);
    }
    look_up(unit + stride);
    // row factors of this lane's four rows (mt, h): scores, and values relative to `w_top`
    float kf[2][2], vf[2][2], w_top;
    const long long blk0 = static_cast<long long>(ch) * p.blocks;
    if (one_block) {
      const float* sc = p.scales + (blk0 + div_of(r0, p.scale_rows)) * 2 * HK + kh;
      const float ks = sc[0] * u;
      w_top = sc[HK] * (u * (1.f / kLift));
#pragma unroll
      for (int i = 0; i < 4; ++i) { kf[i >> 1][i & 1] = ks; vf[i >> 1][i & 1] = kLift; }
    } else {
      w_top = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = r0 + 16 * (i >> 1) + 8 * (i & 1) + g;
        const float* sc = p.scales + (blk0 + div_of(r < T ? r : 0, p.scale_rows)) * 2 * HK + kh;
        kf[i >> 1][i & 1] = sc[0] * u;
        vf[i >> 1][i & 1] = sc[HK];
        w_top = fmaxf(w_top, fabsf(sc[HK]));
      }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) w_top = fmaxf(w_top, __shfl_xor_sync(0xffffffffu, w_top, o));
      w_top = fmaxf(w_top, 0x1p-100f);           // (its reciprocal is finite; an infinite or NaN scale makes its row's factor NaN)
      const float inv = kLift / w_top;
#pragma unroll
      for (int i = 0; i < 4; ++i) vf[i >> 1][i & 1] *= inv;
      w_top *= u * (1.f / kLift);
    }
    uint32_t pb[NT][2][2];             // probabilities as B fragments: rows 16 ks + 2 t + {0, 1} and + 8, column g
    uint32_t rest[NJ == 2 ? NT : 1][2][2];       // ... and what fp16 leaves of them (NJ = 1: in the odd columns)
    float sc[2][NT][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const uint32_t lo[4] = {kr[mt][0].x, kr[mt][0].y, kr[mt][0].z, kr[mt][0].w}, hi[4] = {kr[mt][1].x, kr[mt][1].y, kr[mt][1].z, kr[mt][1].w};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const uint32_t a0 = e4m3x2_to_f16(lo[s]), a1 = e4m3x2_to_f16(hi[s]), a2 = e4m3x2_to_f16_high(lo[s]), a3 = e4m3x2_to_f16_high(hi[s]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (s == 0) mma_f16_new(sc[mt][nt], a0, a1, a2, a3, qb[nt][s][0], qb[nt][s][1]);
          else mma_f16(sc[mt][nt], a0, a1, a2, a3, qb[nt][s][0], qb[nt][s][1]);
        }
      }
    }
    bool above = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {           // rows (mt, h) = (i / 2, i % 2)
          float& s = sc[i >> 1][nt][2 * (i & 1) + j];
          s *= kf[i >> 1][i & 1] * factor[nt][j];
          if (!whole && r0 + 16 * (i >> 1) + 8 * (i & 1) + g >= T) s = -INFINITY;
          top = fmaxf(top, s);
        }
        above |= top > m[nt][j] + kHeadroom;
      }
    if (__any_sync(0xffffffffu, above)) {       // new references: the largest scores so far
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          float top = m[nt][j];
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[i >> 1][nt][2 * (i & 1) + j]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const float corr = top == -INFINITY ? 0.f : exp2_fast(m[nt][j] - top);       // 0 on the first rows (m = -inf)
          m[nt][j] = top;
          l[nt][j] *= corr;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            acc[nt][i][0][j] *= corr;
            acc[nt][i][1][j] *= corr;
          }
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const float ref = m[nt][j] == -INFINITY ? 0.f : m[nt][j];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float& s = sc[i >> 1][nt][2 * (i & 1) + j];
          s = exp2_fast(s - ref);
          l[nt][j] += s;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p0 = sc[i >> 1][nt][2 * (i & 1)] * vf[i >> 1][i & 1], h0 = leading11(p0);
        if constexpr (NJ == 2) {
          const float p1 = sc[i >> 1][nt][2 * (i & 1) + 1] * vf[i >> 1][i & 1], h1 = leading11(p1);
          pb[nt][i >> 1][i & 1] = transpose8(pack_f16(h0, h1));
          rest[nt][i >> 1][i & 1] = transpose8(pack_f16(p0 - h0, p1 - h1));
        } else {
          pb[nt][i >> 1][i & 1] = transpose8(pack_f16(h0, p0 - h0));
        }
      }
    }
    // values: tile i of 16 dims, dims 8 g + 2 i (fragment row g) and 8 g + 2 i + 1 (row g + 8)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float d[NT][4];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const uint32_t sel = i & 1 ? 0x7362u : 0x5140u;
        const uint32_t v01 = __byte_perm(i < 2 ? vr[ks][0].x : vr[ks][0].y, i < 2 ? vr[ks][1].x : vr[ks][1].y, sel);
        const uint32_t v89 = __byte_perm(i < 2 ? vr[ks][2].x : vr[ks][2].y, i < 2 ? vr[ks][3].x : vr[ks][3].y, sel);
        const uint32_t a0 = e4m3x2_to_f16(v01), a1 = e4m3x2_to_f16_high(v01), a2 = e4m3x2_to_f16(v89), a3 = e4m3x2_to_f16_high(v89);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (ks == 0) mma_f16_new(d[nt], a0, a1, a2, a3, pb[nt][ks][0], pb[nt][ks][1]);
          else mma_f16(d[nt], a0, a1, a2, a3, pb[nt][ks][0], pb[nt][ks][1]);
          if constexpr (NJ == 2) mma_f16(d[nt], a0, a1, a2, a3, rest[nt][ks][0], rest[nt][ks][1]);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          acc[nt][i][0][j] = fmaf(w_top, NJ == 2 ? d[nt][j] : d[nt][0] + d[nt][1], acc[nt][i][0][j]);
          acc[nt][i][1][j] = fmaf(w_top, NJ == 2 ? d[nt][2 + j] : d[nt][2] + d[nt][3], acc[nt][i][1][j]);
        }
    }
  }

  // a warp's part, of this lane's columns: dims 8 g ..
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      float sum = l[nt][j];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const int col = nt * 8 + NJ * t + j;
      float* to = red[col][warp];
      *reinterpret_cast<float4*>(to + 8 * g) = make_float4(acc[nt][0][0][j], acc[nt][0][1][j], acc[nt][1][0][j], acc[nt][1][1][j]);
      *reinterpret_cast<float4*>(to + 8 * g + 4) = make_float4(acc[nt][2][0][j], acc[nt][2][1][j], acc[nt][3][0][j], acc[nt][3][1][j]);
      if (g == 0) {
        to[kDD] = m[nt][j];
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
// divisions, 232 with products (185 at the copy rate).
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
  MOC_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(values)) & 15) == 0, "q and the K/V cache must be 16-byte aligned");
  const long long columns = static_cast<long long>(s->n_q) * (s->num_heads / s->num_kv_heads);
  const int wide = columns <= 4 ? 4 : columns <= 8 ? 8 : 16, runs = ceil_div(s->tokens_per_chapter, kRows);
  const long long tiles = (columns + wide - 1) / wide, units = static_cast<long long>(s->n_chapters) * runs;
  MOC_REQUIRE(s->num_kv_heads <= (1 << 18), "too many KV heads");          // (32 rows are below 2^31 bytes)
  MOC_REQUIRE(tiles * s->num_kv_heads < (1ll << 27) && units < (1ll << 30), "decode-attention problem too large for one launch");
  auto kern = wide == 4 ? decode_attn8_kernel<1, 1> : wide == 8 ? decode_attn8_kernel<1, 2> : decode_attn8_kernel<2, 2>;
  // a cluster per (sequence, KV head, tile of columns) while all of them are resident at once and every warp has a unit to take
  const long long groups = tiles * s->num_kv_heads * s->batch;
  int split = 8;
  while (split > 1 && (split / 2 * kWarps >= units || groups > resident_clusters(kern, kThreads, 0, split))) split /= 2;
  Attn8Params p{};
  p.q = static_cast<const __nv_bfloat16*>(q); p.values = static_cast<const uint8_t*>(values); p.scales = scales;
  p.chapters = static_cast<int>(std::min<int64_t>(bank_rows / s->tokens_per_chapter, INT_MAX)); p.blocks = s->tokens_per_chapter / scale_rows;
  p.comb_idx = comb_idx; p.comb_w = comb_w; p.counts = counts; p.out = static_cast<__nv_bfloat16*>(out); p.lse = lse;
  p.n_q = s->n_q; p.H = s->num_heads; p.HK = s->num_kv_heads; p.n_ch = s->n_chapters; p.T = s->tokens_per_chapter;
  p.split = split; p.tiles = static_cast<int>(tiles); p.scale = s->scale; p.scale_rows = fast_div(scale_rows); p.runs = fast_div(runs);
  p.status = status;
  MOC_CUDA_OK(launch_clustered(kern, dim3(static_cast<unsigned>(tiles) * s->num_kv_heads * split, s->batch), kThreads, 0, split,
                               static_cast<cudaStream_t>(stream), p));
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
