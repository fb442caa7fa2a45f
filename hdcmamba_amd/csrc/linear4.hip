// Rows of activations times a 4-bit weight with group scales, for the decode step's projections
// (in_proj, out_proj and the tied head; hdcmamba/model.py:313,325,340,383, train_fineweb.py:94, which
// hold them in the activation type):
//   out[m, n] = sum_g s[n, g] sum_{k in g} (c[n, k] - z[n, g]) x[m, k]  (+ bias[n]) (+ res[m, n])
// with codes c in 0..15, groups g of 32, 64 or 128 columns, scales bf16 or fp32, and zero points z
// (0..15, 8 where there are none).
//
// Packed weight: tiles of 16 rows x 128 columns, 1 KB each, tile (n / 16, k / 128) at index
// (n / 16) * ceil(K / 128) + k / 128.  Inside a tile lane l = 16 g + n % 16 of a wave owns 16
// bytes, four dwords j = 0..3, dword j holding the codes of columns 32 j + 8 g + 0..7: one 16-byte
// load per lane is a whole tile, dword j is the lane's B operand of the tile's j-th
// v_mfma_f32_16x16x32_bf16, and a wave reads 1 KB that is contiguous.  In a dword the codes of columns
// 2 p and 2 p + 1 lie at bits 3 and 19, rotated left by 4 p: rotated back, masked and or-ed with
// 0x41804180 they are the bf16 values 16 + c of both (the exponent of 16, the code in the top
// mantissa bits), 7 instructions for 8 codes.
// bf16 x: a group's sum is formed as sum x (16 + c) - (16 + z) sum x, the second term started with:
// all products are exact, so the roundings are those of the fp32 sums and the last one; the scale
// multiplies the group's sum, not the weights.  (An infinity in x meets its negative there: that
// row becomes NaN; 128 values of at most 2^115 times 31 stay finite.)  fp32 x, whose sums have no bits to spare
// for that: c - z is formed per weight.
#include "hdcm_common.h"

using namespace hdcm;

namespace {

constexpr int kTileN = 16, kTileK = 128;
constexpr int kTileBytes = kTileN * kTileK / 2;

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
// 16-byte loads at the type's own alignment (the row start of a matrix with an odd width)
__device__ __forceinline__ u32x4_t ldu16(const bf16_t* p) {
  typedef u32x4_t run_t __attribute__((aligned(2)));
  return *reinterpret_cast<const run_t*>(p);
}
__device__ __forceinline__ u32x4_t ldu16(const float* p) {
  typedef u32x4_t run_t __attribute__((aligned(4)));
  return *reinterpret_cast<const run_t*>(p);
}

// The 16 bytes of a row of K >= E columns from column k on, zero past its K columns (nothing there is
// read), in two steps, so that the loads of many need no branch between them: the load (from K - E
// on where k lies behind it) and, after all loads, the columns moved into place.
template <typename T> __device__ __forceinline__ u32x4_t load_run(const T* row, int k, int K) {
  constexpr int E = 16 / sizeof(T);
  return ldu16(row + min(k, K - E));
}
template <typename T> __device__ __forceinline__ u32x4_t place_run(u32x4_t v, int k, int K) {
  constexpr int E = 16 / sizeof(T);
  if (k >= K) return u32x4_t{0, 0, 0, 0};
  const int by = k > K - E ? (k - (K - E)) * (int)sizeof(T) : 0;
  if (by & 8) v = u32x4_t{v[2], v[3], 0, 0};
  if (by & 4) v = u32x4_t{v[1], v[2], v[3], 0};
  if (by & 2)
    v = u32x4_t{__builtin_amdgcn_alignbit(v[1], v[0], 16), __builtin_amdgcn_alignbit(v[2], v[1], 16),
                __builtin_amdgcn_alignbit(v[3], v[2], 16), v[3] >> 16};
  return v;
}

// 16 + c of a dword's codes as eight bf16.  The mask is kept in a scalar and the exponent in a vector
// register: with two literals the and and the or would not become one v_and_or_b32.
struct Decode {
  uint32_t mask, expo;
  __device__ __forceinline__ Decode() : mask(0x00780078u), expo(0x41804180u) {
    asm volatile("" : "+s"(mask));
    asm volatile("" : "+v"(expo));
  }
  __device__ __forceinline__ u32x4_t operator()(uint32_t d) const {
    return u32x4_t{(d & mask) | expo, ((d >> 4) & mask) | expo, ((d >> 8) & mask) | expo,
                   (__builtin_amdgcn_alignbit(d, d, 12) & mask) | expo};
  }
};
// The eight values of (16 + c) - z16 as fp32 (exact).
__device__ __forceinline__ void less_zero(u32x4_t v, float z16, float* c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    c[2 * i] = __uint_as_float(v[i] << 16) - z16;
    c[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u) - z16;
  }
}

// Eight columns of a row as A operands: bf16 as they are; an fp32 value as the sum of three bf16 (its
// leading, middle and last eight mantissa bits, cut off exactly), whose three products on the bf16
// MFMA take a fifth of the eight v_mfma_f32_16x16x4_f32 that fp32 operands would.
template <typename T> struct Rows {
  static constexpr int kParts = sizeof(T) == 2 ? 1 : 3;
  Frag<bf16_t> part[kParts];
};
template <typename T> __device__ __forceinline__ f32x4_t mma(const Rows<T>& a, const Frag<bf16_t>& b, f32x4_t c) {
#pragma unroll
  for (int i = Rows<T>::kParts - 1; i >= 0; --i) c = hdcm::mma(a.part[i], b, c);
  return c;
}
// The leading parts of four fp32 values as bf16, and what they leave in the values' place (of an infinity, which only
// the first part meets, nothing).
__device__ __forceinline__ uint2 take_part(u32x4_t& v, bool first) {
  const uint2 o = make_uint2(__builtin_amdgcn_perm(v[1], v[0], 0x07060302u), __builtin_amdgcn_perm(v[3], v[2], 0x07060302u));
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float f = __uint_as_float(v[e]), rest = f - __uint_as_float(v[e] & 0xffff0000u);
    v[e] = first && __builtin_amdgcn_classf(f, 0x204) ? 0u : __float_as_uint(rest);
  }
  return o;
}
__device__ __forceinline__ Frag<bf16_t> fill(uint32_t v) {
  Frag<bf16_t> f;
  f.v = __builtin_bit_cast(bf16x8_t, u32x4_t{v, v, v, v});
  return f;
}

struct Linear4Args {
  const void* x;
  const char *codes, *scales;
  const uint8_t* zeros;
  const void *bias, *res;
  void* out;
  int64_t x_rs, r_rs, o_rs;
  int M, N, K, tiles_n, tiles_k, np, segs;
  bool s_f32;
  const float* row_sums;  // of the weight, where x's rows are to be normalised
  float eps;
};

// A lane's scale of a row of a tile: the loads take a uniform address and a 32-bit lane offset, and of
// bf16 scales the dword that holds two, so that no branch on the type stands between them.
struct Scales {
  const char* p;
  int log;
  uint32_t off, shift, mask;
  __device__ __forceinline__ Scales(const char* s, bool f32, int n)
      : p(s), log(f32 ? 2 : 1), off(f32 ? 4 * n : 2 * n & ~3), shift(f32 || (n & 1) ? 0 : 16), mask(f32 ? ~0u : 0xffff0000u) {}
  // at: the index of the scale of row 0 of the lane's sixteen (even)
  __device__ __forceinline__ uint32_t raw(int64_t at) const { return *reinterpret_cast<const uint32_t*>(p + (at << log) + off); }
  __device__ __forceinline__ float value(uint32_t raw) const { return __uint_as_float((raw << shift) & mask); }
};
__device__ __forceinline__ uint4 load_tile(const Linear4Args& p, int t, int kt, int lane) {
  const char* at = p.codes + ((int64_t)t * p.tiles_k + kt) * kTileBytes;
  return *reinterpret_cast<const uint4*>(at + (uint32_t)(lane * 16));
}

__device__ __forceinline__ void lds_barrier() {  // orders LDS only: loads in flight stay in flight
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// What a wave does with one tile: acc += scale (sum x (16 + c) - (16 + z) sum x) per group.  q: the
// tile's dwords; xa: the rows' fragments; xsum: with one group per tile the rows' sums (or -24 times
// them without zero points), else unused.
template <typename T, int MT, int GS, bool ZERO>
__device__ __forceinline__ void tile_mma(uint4 q, const uint32_t (&sr)[4 / GS], const int (&zr)[4 / GS], const Scales& sc,
                                         const Decode& decode, const Rows<T> (&xa)[4][MT], const f32x4_t (&xsum)[MT],
                                         f32x4_t (&acc)[MT]) {
  constexpr bool BF = sizeof(T) == 2;
  f32x4_t sum[MT];
#pragma unroll
  for (int u = 0; u < 4 / GS; ++u) {
    const float z16 = ZERO ? (float)(zr[u] + 16) : 24.f;
    if constexpr (!BF) {
#pragma unroll
      for (int r = 0; r < MT; ++r) sum[r] = {0.f, 0.f, 0.f, 0.f};
    } else if constexpr (GS == 4) {
#pragma unroll
      for (int r = 0; r < MT; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[r][e] = ZERO ? -z16 * xsum[r][e] : xsum[r][e];
    } else {
      // smaller groups: -(16 + z) as a constant operand (bf16 0xc180 + 8 z), one MFMA a step instead of
      // four multiplications and the registers of the sums
      uint32_t c = 0xc1c0c1c0u;
      if constexpr (ZERO) {
        c = 0xc180u + 8u * (uint32_t)zr[u];
        c |= c << 16;
      }
      const Frag<bf16_t> k = fill(c);
#pragma unroll
      for (int r = 0; r < MT; ++r) {
        sum[r] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < GS; ++j) sum[r] = mma(xa[u * GS + j][r], k, sum[r]);
      }
    }
#pragma unroll
    for (int j = 0; j < GS; ++j) {
      const int i = u * GS + j;
      const u32x4_t v = decode(i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w);
      Frag<bf16_t> b;
      if constexpr (BF) {
        b.v = __builtin_bit_cast(bf16x8_t, v);
      } else {
        float c[8];
        less_zero(v, z16, c);
        frag_from_f32(b, c);
      }
#pragma unroll
      for (int r = 0; r < MT; ++r) sum[r] = mma(xa[i][r], b, sum[r]);
    }
    const float s = sc.value(sr[u]);
#pragma unroll
    for (int r = 0; r < MT; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[r][e] = fmaf(s, sum[r][e], acc[r][e]);
  }
}

// The sums of the rows over a tile's columns (times -24 without zero points), in the MFMA's D layout.
template <typename T, int MT, bool ZERO>
__device__ __forceinline__ void row_sums(const Rows<T> (&xa)[4][MT], f32x4_t (&xsum)[MT]) {
  const Frag<bf16_t> k = fill(ZERO ? 0x3f803f80u : 0xc1c0c1c0u);
#pragma unroll
  for (int r = 0; r < MT; ++r) {
    xsum[r] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) xsum[r] = mma(xa[j][r], k, xsum[r]);
  }
}

// The end of four rows (row0 + 0..3) of one column n: what is added is loaded ahead of the products (at
// clamped places, without a branch per lane, and converted only here), then one rounding and the store.
// NORM: stats holds the mean and the reciprocal deviation of the four rows.
template <typename T, bool NORM = false> struct Ending {
  T bias, res[4];
  float wsum;
  __device__ __forceinline__ void load(const Linear4Args& p, int row0, int rows_end, int n) {
    n = min(n, p.N - 1);
    if constexpr (NORM) wsum = p.row_sums[n];
    if (p.bias) bias = reinterpret_cast<const T*>(p.bias)[n];
    if (p.res) {
#pragma unroll
      for (int e = 0; e < 4; ++e) res[e] = reinterpret_cast<const T*>(p.res)[(int64_t)min(row0 + e, rows_end - 1) * p.r_rs + n];
    }
  }
  __device__ __forceinline__ void store(const Linear4Args& p, f32x4_t v, int row0, int rows_end, int n,
                                        const float2* stats = nullptr) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float y = v[e];
      if constexpr (NORM) y = (y - stats[e].x * wsum) * stats[e].y;
      if (p.bias) y += to_f<T>(bias);
      if (p.res) y += to_f<T>(res[e]);
      if (row0 + e < rows_end && n < p.N) reinterpret_cast<T*>(p.out)[(int64_t)(row0 + e) * p.o_rs + n] = from_f<T>(y);
    }
  }
};

// Rows held in registers.  The W waves of a workgroup split K, P (one or two) 128-column tiles each, and keep
// the fragments of up to 16 MT rows of x for their columns while the workgroup walks over column
// tiles of the output; the next tile's codes are in flight while one is multiplied.  Per output tile
// each wave leaves its partial sums in LDS (two buffers, so one barrier a tile) and the waves take
// turns in adding them up.  x is read once per workgroup, a quarter row per load instruction (whole
// lines; fragments read straight from the rows, 16 rows x 64 bytes an instruction, took 1.4 us
// longer at 16 rows of 2048 and 6.5 us at 64), and brought into fragments through LDS, fp32 part by part
// (split there a run of four is split once, and rows past M cost nothing: 3 x 3264 x 768 4.6 us, 5.6 with
// the fragments split).
// What a launch takes beyond its weight stream: about 2 us of launch, 1 of x, and the issue of ~40
// instructions per wave and tile.  Figures here and at the rules below are recorded calls with the weight in the caches;
// from HBM, as a step reads it: 16 x 8576 x 2048 6.3 us (5.5), 16 x 50304 x 2048 15.3 (13.5), 33 x 50277 x 768 18.9 (16.5),
// 128 x 8576 x 2048 14.0 (13.1), 16 x 2048 x 2176 4.4 (4.4).
// NORM (bf16): out = rstd (x w - mean sum w) takes the row LayerNorm without affine behind the product.  The rows' sums
// and sums of squares come from MFMAs on the fragments that are there (squares: the diagonal of x x'), so they cost no pass
// and no barrier: 0.6 us at 16 x 2048 x 2176 (5.1 us, 4.5 without).  Normalising the rows on their way in, with two
// sums over the waves before the first product, took 4.2 us, the LayerNorm as a launch of its own 2.6.
template <typename T, int MT, int P, int GS, bool ZERO, int MAXW, bool NORM, bool SEG>
__global__ __launch_bounds__(MAXW* kWave, P == 1 && MT > 1 ? 4 : 1) void linear4_kernel(Linear4Args p) {
  constexpr int GPT = 4 / GS;
  constexpr int E = 16 / sizeof(T), CPR = kTileK / E, NLD = 16 * CPR / kWave, PITCH = kTileK + 8;
  extern __shared__ __attribute__((aligned(16))) f32x4_t part[];  // [2][WP][MT][64]; at first the waves' slabs of x
  const int tid = threadIdx.x, lane = tid & (kWave - 1), w = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int W = blockDim.x / kWave, WP = (W + 3) & ~3;
  const int l16 = lane & 15, g = lane >> 4;
  const int m0 = blockIdx.y * 16 * MT;
  const int rows = min(16 * MT, p.M - m0);
  const Decode decode;
  const Scales scales(p.scales, p.s_f32, l16);

  // with more than one segment: the sums of the workgroup's tiles so far, behind the slabs and the partial sums
  f32x4_t* hold = part + max(2 * WP * MT * kWave, W * 16 * PITCH * 2 / 16) + lane;
  __shared__ float2 sums[NORM ? MAXW : 1][16 * MT], stats[NORM ? 16 * MT : 1];
  const int segs = SEG ? p.segs : 1;
  for (int seg = 0; seg < segs; ++seg) {
    int64_t x_rs = p.x_rs;
    int ln = lane;
    // with many rows their addresses are formed anew: kept over the products they would spill (64 x 8576 x 4096: 22.6 us, 25.1;
    // for 16 rows, which have the registers, 11.4 and 10.5)
    if constexpr (SEG && MT > 2) asm volatile("" : "+s"(x_rs), "+v"(ln));
    const int k0 = (seg * W + w) * P;  // the wave's first column tile

    // x: 16 rows x 128 columns in NLD loads
    const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)m0 * x_rs;
    u32x4_t raw[MT][P][NLD];
#pragma unroll
    for (int r = 0; r < MT; ++r)
#pragma unroll
      for (int i = 0; i < P; ++i)
#pragma unroll
        for (int n = 0; n < NLD; ++n) {
          // rows past M re-read the last; a whole load of them is left out (their fragments hold what LDS held:
          // every row of a product depends on its own row of x alone, and theirs are not stored)
          if (n * kWave / CPR + 16 * r >= rows) {
            if constexpr (SEG) raw[r][i][n] = u32x4_t{0, 0, 0, 0};  // (else the last segment's stay in registers)
            continue;
          }
          const int at = n * kWave + ln, row = min(16 * r + at / CPR, rows - 1);
          raw[r][i][n] = load_run<T>(x + (int64_t)row * x_rs, (k0 + i) * kTileK + at % CPR * E, p.K);
        }
    uint4 q[P];
    uint32_t sr[P][GPT];
    int zr[P][GPT];
    auto fetch = [&](int t) {  // tiles past the last re-read it
      t = min(t, p.tiles_n - 1);
#pragma unroll
      for (int i = 0; i < P; ++i) q[i] = load_tile(p, t, min(k0 + i, p.tiles_k - 1), lane);
#pragma unroll
      for (int i = 0; i < P; ++i)
#pragma unroll
        for (int u = 0; u < GPT; ++u) {
          const int64_t at = (int64_t)(min(k0 + i, p.tiles_k - 1) * GPT + u) * p.np + kTileN * t;
          sr[i][u] = scales.raw(at);
          if constexpr (ZERO) zr[i][u] = (p.zeros + at)[(uint32_t)l16];
        }
    };
    fetch(blockIdx.x);

    if constexpr (SEG) __syncthreads();  // the partial sums are read
    bf16_t* slab = reinterpret_cast<bf16_t*>(part) + w * 16 * PITCH;  // the wave's own: no barrier
    Rows<T> xa[P][4][MT];
#pragma unroll
    for (int r = 0; r < MT; ++r)
#pragma unroll
      for (int i = 0; i < P; ++i)
#pragma unroll
        for (int h = 0; h < Rows<T>::kParts; ++h) {
          asm volatile("" ::: "memory");  // a wave's LDS accesses complete in order; they stay in this one
#pragma unroll
          for (int n = 0; n < NLD; ++n) {
            if (n * kWave / CPR + 16 * r >= rows) continue;
            const int at = n * kWave + ln, k = (k0 + i) * kTileK + at % CPR * E;
            u32x4_t& v = raw[r][i][n];
            if (h == 0 && (k0 + i + 1) * kTileK > p.K) v = place_run<T>(v, k, p.K);  // (uniform)
            bf16_t* to = slab + at / CPR * PITCH + at % CPR * E;
            if constexpr (sizeof(T) == 2) *reinterpret_cast<u32x4_t*>(to) = v;
            else *reinterpret_cast<uint2*>(to) = take_part(v, h == 0);
          }
          asm volatile("" ::: "memory");
#pragma unroll
          for (int j = 0; j < 4; ++j)
            xa[i][j][r].part[h].v = *reinterpret_cast<const bf16x8_t*>(slab + (ln & 15) * PITCH + 32 * j + 8 * (ln >> 4));
          asm volatile("" ::: "memory");
        }
    f32x4_t xsum[P][MT];
    if constexpr (GS == 4 && sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < P; ++i) row_sums<T, MT, ZERO>(xa[i], xsum[i]);
    }
    if constexpr (NORM) {
#pragma unroll
      for (int r = 0; r < MT; ++r) {
        f32x4_t s1 = {0.f, 0.f, 0.f, 0.f}, s2 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s1 = mma(xa[i][j][r], fill(0x3f803f80u), s1);
            s2 = mma(xa[i][j][r], xa[i][j][r].part[0], s2);
          }
        const int e = l16 & 3;  // row 4 g + e, column l16
        if (l16 / 4 == g) {  // (of every segment the same lane)
          const float2 before = seg ? sums[w][16 * r + l16] : make_float2(0.f, 0.f);
          sums[w][16 * r + l16] = make_float2(before.x + (e == 0 ? s1[0] : e == 1 ? s1[1] : e == 2 ? s1[2] : s1[3]),
                                              before.y + (e == 0 ? s2[0] : e == 1 ? s2[1] : e == 2 ? s2[2] : s2[3]));
        }
      }
    }
    __syncthreads();  // the slabs become the partial sums' buffers
    if constexpr (NORM)
      if (seg == segs - 1 && tid < 16 * MT) {  // (seen by the others from the first barrier of the loop on)
        float s1 = 0.f, s2 = 0.f;
        for (int k = 0; k < W; ++k) s1 += sums[k][tid].x, s2 += sums[k][tid].y;
        const float mean = s1 / (float)p.K;
        stats[tid] = make_float2(mean, rsqrtf(fmaxf(s2 / (float)p.K - mean * mean, 0.f) + p.eps));
      }
    for (int k = W + w; k < WP; k += W)  // waves that are not there add nothing
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) part[(i / MT * WP + k) * MT * kWave + i % MT * kWave + lane] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    int buf = 0, turn = 0;
    f32x4_t* kept = hold;
    for (int t = blockIdx.x; t < p.tiles_n; t += gridDim.x, kept += MT * kWave) {
      Ending<T, NORM> end;
      const int own = w >= turn ? w - turn : w + W - turn;  // the row tile that this wave adds up (none past MT)
      if (own < MT) end.load(p, m0 + 16 * own + 4 * g, m0 + rows, kTileN * t + l16);
      f32x4_t acc[MT];
#pragma unroll
      for (int r = 0; r < MT; ++r) acc[r] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < P; ++i)
        if ((i == 0 && !SEG) || k0 + i < p.tiles_k)
          tile_mma<T, MT, GS, ZERO>(q[i], sr[i], zr[i], scales, decode, xa[i], xsum[i], acc);
      fetch(t + gridDim.x);
      if (P == 1 && MT <= 2 && W == 1) {  // nothing to add up
#pragma unroll
        for (int r = 0; r < MT; ++r) {
          if (r > 0) end.load(p, m0 + 16 * r + 4 * g, m0 + rows, kTileN * t + l16);
          end.store(p, acc[r], m0 + 16 * r + 4 * g, m0 + rows, kTileN * t + l16, NORM ? stats + 16 * r + 4 * g : nullptr);
        }
        continue;
      }
      f32x4_t* mine = part + (buf * WP + w) * MT * kWave + lane;
#pragma unroll
      for (int r = 0; r < MT; ++r) mine[r * kWave] = acc[r];
      lds_barrier();
      for (int r = own; r < MT; r += W) {  // (fewer waves than row tiles: the others follow)
        if (r != own) end.load(p, m0 + 16 * r + 4 * g, m0 + rows, kTileN * t + l16);
        const f32x4_t* from = part + buf * WP * MT * kWave + r * kWave + lane;
        f32x4_t v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = from[k * MT * kWave];
        f32x4_t sum = (v[0] + v[1]) + (v[2] + v[3]);
#pragma unroll
        for (int b = 4; b < MAXW; b += 4)
          if (W > b) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = from[(b + k) * MT * kWave];
            sum += (v[0] + v[1]) + (v[2] + v[3]);
          }
        if (seg > 0) sum += kept[r * kWave];  // the same wave's in every segment
        if (seg < segs - 1) {
          kept[r * kWave] = sum;
          continue;
        }
        end.store(p, sum, m0 + 16 * r + 4 * g, m0 + rows, kTileN * t + l16, NORM ? stats + 16 * r + 4 * g : nullptr);
      }
      turn += MT;
      while (turn >= W) turn -= W;
      buf ^= 1;
    }
  }
}

// The registers hold up to 64 bf16 rows of 16 column tiles (2048 columns) in 8 waves, or 32 rows of 24
// in 12; of fp32 rows, whose three parts take three times as many, 16.  More rows run as row blocks of
// equal height, which read the weight again (out of the caches); longer rows in segments of K, whose
// sums wait in LDS (a workgroup takes no more tiles than fit).  Figures below in us, rows x N x K.
//
// Height of a row block: 64 rows where that takes no more segments than 32 (with 64 and 32: 64 x 4096 x 4352, three
// segments or two, 22.9, 14.4; 384 rows 43.1, 36.7; 64 x 50304 x 4096, two both ways, 45.3, 53.5) and K has more than four
// tiles, below which the few waves of a workgroup with the registers of 64 rows leave the SIMDs empty (64 x 20000 x 384 10.4,
// 7.6; 106 x 46400 x 192 21.0, 16.6; but 33 x 50277 x 768 17.1, 22.7); lower where there are so few column tiles that
// more blocks still make no more than four workgroups for every CU: a block's rows take the longest part of such a run
// (64 x 1024 x 1152 in one block and four 7.1, 3.9; 64 x 2048 x 2176 in two and four 6.8, 5.7; 128 x 3264 x 768 in
// two and five 7.3, 6.3; with eight workgroups for every CU 128 x 8576 x 2048 13.6, 14.2).
//
// A row block has the CUs that the others leave (128 x 8576 x 2048 with all of them for each block 19.0, with half 14.1; 192
// rows 27.4, 17.9): x is read once per workgroup, 256 KB at 64 rows of 2048.
//
// Column tiles a wave: one, where that makes no more than 12 waves (16 of fp32, 8 with more than 32 rows: the registers),
// since the rows' way into the fragments then has twice the waves (with two and one: 16 x 1024 x 1152 3.9, 3.5; 32 x 3264 x
// 768 4.6, 4.0; 64 x 3264 x 768 6.7, 5.5; 64 x 50277 x 768 19.9, 18.4; fp32 3 x 3264 x 768 5.9, 5.6, 16 x 8576 x 2048
// 17.8, 11.5).  Two for one row tile of bf16 and more than two output tiles for every CU: there the sums over the
// waves count (16 x 8192 x 1152 5.1, 4.6, x 12800 6.3, 6.7, x 25600 7.8, 9.9).
constexpr int kCUs = 256, kHeldBytes = kWave * 16;
constexpr int kLds = 152 * 1024;  // for the slabs, partial and held sums; NORM's sums take up to 6 KB more

template <typename T, int MT, int P, int GS, bool ZERO, int MAXW, bool SEG>
void launch_linear4(const Linear4Args& a, int blocks_m, hipStream_t s) {
  const int W = ((a.tiles_k + a.segs - 1) / a.segs + P - 1) / P;
  // waves per CU: 8 where the registers hold more than one row tile of two column tiles, else 16: whole workgroups
  const int per_cu = (MT == 1 || P == 1 ? 16 : 8) / W;
  int most = kCUs * (per_cu > 1 ? per_cu : 1) / blocks_m;
  const int slabs = W * 16 * (kTileK + 8) * 2, parts = 2 * ((W + 3) & ~3) * MT * kHeldBytes;
  int shmem = slabs > parts ? slabs : parts;
  if (a.segs > 1) {
    const int room = (kLds - shmem) / kHeldBytes / MT, least = (a.tiles_n + room - 1) / room;  // column tiles of a workgroup
    most = most > least ? most : least;
  }
  if (most < 1) most = 1;
  if (most > a.tiles_n) most = a.tiles_n;
  if (a.segs > 1) shmem += (a.tiles_n + most - 1) / most * MT * kHeldBytes;
  const dim3 grid((unsigned)most, (unsigned)blocks_m);
  if constexpr (sizeof(T) == 2)
    if (a.row_sums) {
      HDCM_LAUNCH((linear4_kernel<T, MT, P, GS, ZERO, MAXW, true, SEG>), grid, dim3(W * kWave), shmem, s, a);
      return;
    }
  HDCM_LAUNCH((linear4_kernel<T, MT, P, GS, ZERO, MAXW, false, SEG>), grid, dim3(W * kWave), shmem, s, a);
}
template <typename T, int MT, int GS, bool ZERO, int MAXW> void pick_tiles(const Linear4Args& a, int blocks_m, hipStream_t s) {
  constexpr int most1 = MT > 2 ? 8 : sizeof(T) == 4 ? 16 : 12;
  const bool one = a.tiles_k <= most1 && (MT > 1 || sizeof(T) == 4 || a.tiles_n <= 2 * kCUs);
  if (a.segs > 1) launch_linear4<T, MT, 2, GS, ZERO, MAXW, true>(a, blocks_m, s);
  else if (one) launch_linear4<T, MT, 1, GS, ZERO, most1, false>(a, blocks_m, s);
  else launch_linear4<T, MT, 2, GS, ZERO, MAXW, false>(a, blocks_m, s);
}
template <typename T, int GS, bool ZERO> void pick_rows(Linear4Args a, hipStream_t s) {
  const int tiles_m = (a.M + 15) / 16;
  const auto segments = [&](int widest) { return (a.tiles_k + widest - 1) / widest; };
  const int most = sizeof(T) == 4 ? 1 : a.tiles_k <= 4 || segments(24) < segments(16) ? 2 : 4;
  const int least = (tiles_m + most - 1) / most, room = 4 * kCUs / a.tiles_n, fill = room < tiles_m ? room : tiles_m;
  const int wanted = least > fill ? least : fill, mt = (tiles_m + wanted - 1) / wanted;
  const int blocks = (tiles_m + mt - 1) / mt;  // none without rows
  a.segs = segments(mt > 2 ? 16 : 24);
  if (mt == 1) pick_tiles<T, 1, GS, ZERO, 12>(a, blocks, s);
  if constexpr (sizeof(T) == 2) {
    if (mt == 2) pick_tiles<T, 2, GS, ZERO, 12>(a, blocks, s);
    if (mt == 3) pick_tiles<T, 3, GS, ZERO, 8>(a, blocks, s);
    if (mt == 4) pick_tiles<T, 4, GS, ZERO, 8>(a, blocks, s);
  }
}
template <typename T, int GS> void pick_zero(const Linear4Args& a, hipStream_t s) {
  a.zeros ? pick_rows<T, GS, true>(a, s) : pick_rows<T, GS, false>(a, s);
}
template <typename T> void pick_group(const Linear4Args& a, int group, hipStream_t s) {
  if (group == 32) pick_zero<T, 1>(a, s);
  else if (group == 64) pick_zero<T, 2>(a, s);
  else pick_zero<T, 4>(a, s);
}

// ------------------------------------------------------------ packing and unpacking
// The bits of code c of column e of a dword's eight.
__device__ __forceinline__ uint32_t code_bits(uint32_t c, int e) {
  const uint32_t v = c << (e & 1 ? 19 : 3);
  return __builtin_amdgcn_alignbit(v, v, (32 - 4 * (e / 2)) & 31);  // rotated left by 4 (e / 2)
}
__device__ __forceinline__ int64_t dword_at(int n, int k8, int tiles_k) {  // columns 8 k8 .. +8 of row n
  const int kt = k8 / 16, j = (k8 % 16) / 4, g = k8 % 4;
  return (((int64_t)(n / kTileN) * tiles_k + kt) * kWave + 16 * g + n % kTileN) * 4 + j;
}

// One thread per dword of the packed weight; rows and columns past the weight hold code 8.
__global__ __launch_bounds__(256) void w4_pack_kernel(const uint8_t* __restrict__ codes, int64_t rs, int N, int K,
                                                      int tiles_k, int64_t total, uint32_t* __restrict__ packed) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const int k8 = (int)(i % (tiles_k * 16)), n = (int)(i / (tiles_k * 16));
  uint32_t d = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int k = 8 * k8 + e;
    const uint32_t c = n < N && k < K ? codes[(int64_t)n * rs + k] & 15u : 8u;
    d |= code_bits(c, e);
  }
  packed[dword_at(n, k8, tiles_k)] = d;
}

// One thread per (row, group) of the padded weight.  Without zero points the scale is the group's largest
// magnitude / 7 and c = round(w / s) + 8 in 1..15; with them the range from min(w, 0) to max(w, 0) in 15
// steps, z = round(-min / s).  The codes are taken with the scale as rounded to its type.  Once per weight: 8576 x
// 2048 167 us (hdcm_w4_pack 18), by loads that do not share lines.
template <typename T, typename S>
__global__ __launch_bounds__(256) void w4_quantize_kernel(const T* __restrict__ w, int64_t rs, int N, int K, int group,
                                                          int tiles_k, int np, uint32_t* __restrict__ packed,
                                                          S* __restrict__ scales, uint8_t* __restrict__ zeros) {
  const int groups = tiles_k * kTileK / group;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)np * groups) return;
  const int g = (int)(i % groups), n = (int)(i / groups);
  const int k0 = g * group, k1 = n < N ? min(k0 + group, K) : k0;
  const T* row = w + (int64_t)n * rs;
  float lo = 0.f, hi = 0.f;
  for (int k = k0; k < k1; ++k) {
    const float v = to_f<T>(row[k]);
    lo = fminf(lo, v);
    hi = fmaxf(hi, v);
  }
  // the range is divided before it is subtracted: hi - lo may be beyond the largest float
  const float s = rnd<S>(zeros ? hi / 15.f - lo / 15.f : fmaxf(hi, -lo) / 7.f);
  const float z = zeros ? (s > 0.f ? fminf(rintf(-lo / s), 15.f) : 8.f) : 8.f;
  scales[(int64_t)g * np + n] = from_f<S>(s);
  if (zeros) zeros[(int64_t)g * np + n] = (uint8_t)z;
  for (int k8 = k0 / 8; k8 < (k0 + group) / 8; ++k8) {
    uint32_t d = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = 8 * k8 + e;
      const float c = k >= k1 ? 8.f : s > 0.f ? fminf(fmaxf(rintf(to_f<T>(row[k]) / s) + z, 0.f), 15.f) : z;
      d |= code_bits((uint32_t)c, e);
    }
    packed[dword_at(n, k8, tiles_k)] = d;
  }
}

// s (c - z), rounded to T: a wave per tile, eight columns of a row per lane and step, so that four lanes
// write 64 (bf16) or 128 (fp32) bytes of a row: the write's rate, 8576 x 2048 to bf16 (9 MB read, 35 written) in 11.0 us.
template <typename T>
__global__ __launch_bounds__(256) void w4_dequant_kernel(const char* __restrict__ packed, const char* scales, bool s_f32,
                                                         const uint8_t* __restrict__ zeros, int N, int K, int group,
                                                         int tiles_k, int64_t tiles, int np, T* __restrict__ out, int64_t o_rs) {
  const int64_t tile = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
  if (tile >= tiles) return;
  const int lane = threadIdx.x % kWave, l16 = lane & 15, g = lane >> 4;
  const int t = (int)(tile / tiles_k), kt = (int)(tile % tiles_k), n = kTileN * t + l16;
  const uint4 q = *reinterpret_cast<const uint4*>(packed + tile * kTileBytes + lane * 16);
  const Scales sc(scales, s_f32, l16);
  const Decode decode;
  if (n >= N) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int k = kt * kTileK + 32 * j + 8 * g;
    const int64_t at = (int64_t)((kt * kTileK + 32 * j) / group) * np + kTileN * t;
    const float s = sc.value(sc.raw(at));
    float c[8];
    less_zero(decode(j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w), zeros ? (float)(zeros[at + l16] + 16) : 24.f, c);
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] *= s;
    T* o = out + (int64_t)n * o_rs + k;
    if (k + 8 <= K) {
      if constexpr (sizeof(T) == 2) {
        typedef u32x4_t run_t __attribute__((aligned(2)));
        *reinterpret_cast<run_t*>(o) = u32x4_t{pack_bf16x2(c[0], c[1]), pack_bf16x2(c[2], c[3]), pack_bf16x2(c[4], c[5]),
                                               pack_bf16x2(c[6], c[7])};
      } else {
        typedef float run_t __attribute__((ext_vector_type(4), aligned(4)));
        *reinterpret_cast<run_t*>(o) = run_t{c[0], c[1], c[2], c[3]};
        *reinterpret_cast<run_t*>(o + 4) = run_t{c[4], c[5], c[6], c[7]};
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k + e < K) o[e] = from_f<T>(c[e]);
    }
  }
}

bool sizes_ok(int64_t N, int64_t K, int64_t group) {
  return (group == 32 || group == 64 || group == 128) && N < ((int64_t)1 << 30) && K < ((int64_t)1 << 24);
}
int tiles_of(int64_t n, int tile) { return (int)((n + tile - 1) / tile); }
dim3 threads256(int64_t n) { return dim3((unsigned)((n + 255) / 256)); }

}  // namespace

extern "C" size_t hdcm_w4_packed_bytes(int64_t N, int64_t K) {
  return N > 0 && K > 0 ? (size_t)tiles_of(N, kTileN) * tiles_of(K, kTileK) * kTileBytes : 0;
}

extern "C" int hdcm_w4_pack(const uint8_t* codes, int64_t codes_row_stride, int64_t N, int64_t K, void* packed,
                            void* stream) {
  HDCM_CHECK_ARG(N >= 0 && K > 0, HDCM_EINVAL);
  HDCM_CHECK_ARG((codes && packed) || N == 0, HDCM_EINVAL);
  HDCM_CHECK_ARG(codes_row_stride >= K || N <= 1, HDCM_EINVAL);
  HDCM_CHECK_ARG(sizes_ok(N, K, 32), HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(hdcm_aligned16(packed), HDCM_EALIGN);
  if (N == 0) return HDCM_OK;
  const int tk = tiles_of(K, kTileK);
  const int64_t total = (int64_t)tiles_of(N, kTileN) * kTileN * tk * 16;
  HDCM_CHECK_ARG(total < ((int64_t)1 << 38), HDCM_EUNSUPPORTED);
  HDCM_LAUNCH(w4_pack_kernel, threads256(total), dim3(256), 0, (hipStream_t)stream, codes, codes_row_stride, (int)N, (int)K,
              tk, total, (uint32_t*)packed);
  return hdcm_launch_status();
}

extern "C" int hdcm_w4_quantize(const void* w, int64_t w_row_stride, int64_t N, int64_t K, int64_t group, void* packed,
                                void* scales, int scale_dtype, uint8_t* zeros, int dtype, void* stream) {
  HDCM_CHECK_ARG((dtype == HDCM_F32 || dtype == HDCM_BF16) && (scale_dtype == HDCM_F32 || scale_dtype == HDCM_BF16),
                 HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(N >= 0 && K > 0, HDCM_EINVAL);
  HDCM_CHECK_ARG((w && packed && scales) || N == 0, HDCM_EINVAL);
  HDCM_CHECK_ARG(w_row_stride >= K || N <= 1, HDCM_EINVAL);
  HDCM_CHECK_ARG(sizes_ok(N, K, group), HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(hdcm_aligned16(packed), HDCM_EALIGN);
  if (N == 0) return HDCM_OK;
  const int tk = tiles_of(K, kTileK), np = tiles_of(N, kTileN) * kTileN, g = (int)group, n = (int)N, k = (int)K;
  const int64_t total = (int64_t)np * (tk * kTileK / g);
  HDCM_CHECK_ARG(total < ((int64_t)1 << 38), HDCM_EUNSUPPORTED);
  const dim3 grid = threads256(total);
  hipStream_t s = (hipStream_t)stream;
  uint32_t* d = (uint32_t*)packed;
  if (dtype == HDCM_F32 && scale_dtype == HDCM_F32)
    HDCM_LAUNCH((w4_quantize_kernel<float, float>), grid, dim3(256), 0, s, (const float*)w, w_row_stride, n, k, g, tk, np, d,
                (float*)scales, zeros);
  else if (dtype == HDCM_F32)
    HDCM_LAUNCH((w4_quantize_kernel<float, bf16_t>), grid, dim3(256), 0, s, (const float*)w, w_row_stride, n, k, g, tk, np,
                d, (bf16_t*)scales, zeros);
  else if (scale_dtype == HDCM_F32)
    HDCM_LAUNCH((w4_quantize_kernel<bf16_t, float>), grid, dim3(256), 0, s, (const bf16_t*)w, w_row_stride, n, k, g, tk, np,
                d, (float*)scales, zeros);
  else
    HDCM_LAUNCH((w4_quantize_kernel<bf16_t, bf16_t>), grid, dim3(256), 0, s, (const bf16_t*)w, w_row_stride, n, k, g, tk,
                np, d, (bf16_t*)scales, zeros);
  return hdcm_launch_status();
}

extern "C" int hdcm_w4_dequant(const void* packed, const void* scales, int scale_dtype, const uint8_t* zeros, int64_t group,
                               void* out, int64_t out_row_stride, int64_t N, int64_t K, int dtype, void* stream) {
  HDCM_CHECK_ARG((dtype == HDCM_F32 || dtype == HDCM_BF16) && (scale_dtype == HDCM_F32 || scale_dtype == HDCM_BF16),
                 HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(N >= 0 && K > 0, HDCM_EINVAL);
  HDCM_CHECK_ARG((packed && scales && out) || N == 0, HDCM_EINVAL);
  HDCM_CHECK_ARG(out_row_stride >= K || N <= 1, HDCM_EINVAL);
  HDCM_CHECK_ARG(sizes_ok(N, K, group), HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(hdcm_aligned16(packed) && ((uintptr_t)scales & 3u) == 0, HDCM_EALIGN);
  if (N == 0) return HDCM_OK;
  const int tk = tiles_of(K, kTileK), np = tiles_of(N, kTileN) * kTileN, g = (int)group, n = (int)N, k = (int)K;
  const int64_t tiles = (int64_t)tiles_of(N, kTileN) * tk;
  HDCM_CHECK_ARG(tiles < ((int64_t)1 << 32), HDCM_EUNSUPPORTED);
  const dim3 grid((unsigned)((tiles + 3) / 4));
  hipStream_t s = (hipStream_t)stream;
  const char *d = (const char*)packed, *sc = (const char*)scales;
  const bool f = scale_dtype == HDCM_F32;
  if (dtype == HDCM_F32)
    HDCM_LAUNCH(w4_dequant_kernel<float>, grid, dim3(256), 0, s, d, sc, f, zeros, n, k, g, tk, tiles, np, (float*)out,
                out_row_stride);
  else
    HDCM_LAUNCH(w4_dequant_kernel<bf16_t>, grid, dim3(256), 0, s, d, sc, f, zeros, n, k, g, tk, tiles, np, (bf16_t*)out,
                out_row_stride);
  return hdcm_launch_status();
}

extern "C" int hdcm_w4_linear_fwd(const void* x, int64_t x_row_stride, const float* row_sums, float eps, const void* packed,
                                  const void* scales, int scale_dtype, const uint8_t* zeros, int64_t group, const void* bias,
                                  const void* res, int64_t res_row_stride, void* out, int64_t out_row_stride, int64_t M,
                                  int64_t N, int64_t K, int dtype, void* stream) {
  HDCM_CHECK_ARG((dtype == HDCM_F32 || dtype == HDCM_BF16) && (scale_dtype == HDCM_F32 || scale_dtype == HDCM_BF16),
                 HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(M >= 0 && N >= 0 && K > 0, HDCM_EINVAL);
  HDCM_CHECK_ARG(M == 0 || N == 0 || (x && packed && scales && out), HDCM_EINVAL);
  HDCM_CHECK_ARG(M <= 1 || (x_row_stride >= K && out_row_stride >= N && (!res || res_row_stride >= N)), HDCM_EINVAL);
  HDCM_CHECK_ARG(!row_sums || dtype == HDCM_BF16, HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(!row_sums || eps >= 0.f, HDCM_EINVAL);
  HDCM_CHECK_ARG(sizes_ok(N, K, group) && K >= (dtype == HDCM_F32 ? 4 : 8) && M <= 16 * 65535, HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(hdcm_aligned16(packed) && ((uintptr_t)scales & 3u) == 0, HDCM_EALIGN);
  if (M == 0 || N == 0) return HDCM_OK;
  Linear4Args a;
  a.x = x, a.codes = (const char*)packed, a.scales = (const char*)scales, a.zeros = zeros, a.bias = bias, a.res = res, a.out = out;
  a.x_rs = x_row_stride, a.r_rs = res_row_stride, a.o_rs = out_row_stride;
  a.M = (int)M, a.N = (int)N, a.K = (int)K;
  a.tiles_n = tiles_of(N, kTileN), a.tiles_k = tiles_of(K, kTileK), a.np = a.tiles_n * kTileN;
  a.s_f32 = scale_dtype == HDCM_F32, a.row_sums = row_sums, a.eps = eps;
  hipStream_t s = (hipStream_t)stream;
  dtype == HDCM_F32 ? pick_group<float>(a, (int)group, s) : pick_group<bf16_t>(a, (int)group, s);
  return hdcm_launch_status();
}
