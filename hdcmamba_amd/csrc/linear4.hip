// Rows of activations times a 4-bit weight with group scales, for the decode step's projections
// (in_proj, out_proj and the tied head; hdcmamba/model.py:313,325,340,383, train_fineweb.py:94, which
// hold them in the activation type):
//   out[m, n] = sum_g s[n, g] sum_{k in g} (c[n, k] - z[n, g]) x[m, k]  (+ bias[n]) (+ res[m, n])
// with codes c in 0..15, groups g of 32, 64 or 128 columns, scales bf16 or fp32, and zero points z
// (0..15, 8 where there are none).
//
// Packed weight: tiles of 16 rows x 128 columns, 1 KB each, tile (n / 16, k / 128) at index
// (n / 16) * ceil(K / 128) + k / 128.  Inside a tile lane l = 16 g + n % 16 of a wave owns 16
// bytes, four dwords j = 0..3, dword j holding the codes of columns 32 j + 8 g + 0..7 from its lowest
// nibble up: one 16-byte load per lane is a whole tile, dword j is the lane's B operand of the
// tile's j-th v_mfma_f32_16x16x32_bf16, and a wave reads 1 KB that is contiguous.  A code is stored
// as c ^ 8, the two's complement of c - 8, which v_cvt_off_f32_i4 turns into (c - 8) / 16; a zero
// point other than 8 is subtracted there.  (c - z) / 16 is exact in bf16, so a product's only
// roundings are those of the fp32 sums: the scale multiplies a group's sum, not the weights.
#include "hdcm_common.h"

using namespace hdcm;

namespace {

constexpr int kTileN = 16, kTileK = 128;
constexpr int kTileBytes = kTileN * kTileK / 2;

// 16-byte loads at the type's own alignment (the row start of a matrix with an odd width)
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x4_t ldu16(const bf16_t* p) {
  typedef u32x4_t run_t __attribute__((aligned(2)));
  return *reinterpret_cast<const run_t*>(p);
}
__device__ __forceinline__ u32x4_t ldu16(const float* p) {
  typedef u32x4_t run_t __attribute__((aligned(4)));
  return *reinterpret_cast<const run_t*>(p);
}

// Eight activations of a row from column k on; past the row's K columns zero, whatever lies there.
template <typename T> __device__ __forceinline__ void load_x(Frag<T>& f, const T* row, int k, int K);
template <> __device__ __forceinline__ void load_x<bf16_t>(Frag<bf16_t>& f, const bf16_t* row, int k, int K) {
  if (k + 8 <= K) {
    f.v = __builtin_bit_cast(bf16x8_t, ldu16(row + k));
  } else {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k + e < K) w[e / 2] |= (uint32_t)row[k + e] << (16 * (e & 1));
    f.v = __builtin_bit_cast(bf16x8_t, u32x4_t{w[0], w[1], w[2], w[3]});
  }
}
template <> __device__ __forceinline__ void load_x<float>(Frag<float>& f, const float* row, int k, int K) {
  if (k + 8 <= K) {
    const u32x4_t a = ldu16(row + k), b = ldu16(row + k + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) f.v[e] = __uint_as_float(a[e]), f.v[4 + e] = __uint_as_float(b[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = k + e < K ? row[k + e] : 0.f;
  }
}

// (c - z) / 16 of the eight codes of a dword; z16 = (z - 8) / 16.
template <bool ZERO> __device__ __forceinline__ void decode8(uint32_t d, float z16, float* w) {
  const uint32_t h = d >> 4;
  w[0] = __builtin_amdgcn_cvt_off_f32_i4(d);
  w[1] = __builtin_amdgcn_cvt_off_f32_i4(h);
  w[2] = __builtin_amdgcn_cvt_off_f32_i4((d >> 8) & 255);
  w[3] = __builtin_amdgcn_cvt_off_f32_i4((h >> 8) & 255);
  w[4] = __builtin_amdgcn_cvt_off_f32_i4((d >> 16) & 255);
  w[5] = __builtin_amdgcn_cvt_off_f32_i4((h >> 16) & 255);
  w[6] = __builtin_amdgcn_cvt_off_f32_i4(d >> 24);
  w[7] = __builtin_amdgcn_cvt_off_f32_i4(h >> 24);
  if constexpr (ZERO) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] -= z16;
  }
}

__device__ __forceinline__ float load_scale(const void* s, bool f32, int64_t i) {
  return f32 ? reinterpret_cast<const float*>(s)[i] : bf2f(reinterpret_cast<const bf16_t*>(s)[i]);
}

struct Linear4Args {
  const void* x;
  const uint4* codes;
  const void* scales;
  const uint8_t* zeros;
  const void *bias, *res;
  void* out;
  int64_t x_rs, r_rs, o_rs;
  int M, N, K, tiles_n, tiles_k, np;
  bool s_f32;
};

// A workgroup of W waves computes MT row tiles of 16 by NT column tiles of 16, the waves taking the
// 128-column tiles of K in turn; their partial sums are added in wave order through LDS.
template <typename T, int MT, int NT, int W, int GS, bool ZERO>
__global__ __launch_bounds__(W* kWave) void linear4_kernel(Linear4Args p) {
  constexpr int ROWS = 16 * MT, COLS = 16 * NT, PITCH = COLS + 1;
  constexpr int GPT = 4 / GS;  // groups per tile
  __shared__ float part[W][ROWS * PITCH];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), w = tid / kWave;
  const int l16 = lane & 15, g = lane >> 4;
  const int t0 = blockIdx.x * NT, m0 = blockIdx.y * ROWS;
  const T* x = reinterpret_cast<const T*>(p.x);
  const T* xr[MT];  // rows past M read row M-1 (their outputs are not stored)
#pragma unroll
  for (int r = 0; r < MT; ++r) xr[r] = x + (int64_t)min(m0 + 16 * r + l16, p.M - 1) * p.x_rs;
  f32x4_t acc[MT][NT];
#pragma unroll
  for (int r = 0; r < MT; ++r)
#pragma unroll
    for (int c = 0; c < NT; ++c) acc[r][c] = {0.f, 0.f, 0.f, 0.f};

  for (int kt = w; kt < p.tiles_k; kt += W) {
    uint4 q[NT];
    float s[NT][GPT], z[NT][GPT];
#pragma unroll
    for (int c = 0; c < NT; ++c) {  // column tiles past the last re-read it
      const int t = min(t0 + c, p.tiles_n - 1);
      q[c] = p.codes[((int64_t)t * p.tiles_k + kt) * kWave + lane];
#pragma unroll
      for (int i = 0; i < GPT; ++i) {
        const int64_t at = (int64_t)(kt * GPT + i) * p.np + 16 * t + l16;
        s[c][i] = 16.f * load_scale(p.scales, p.s_f32, at);
        z[c][i] = ZERO ? ((int)p.zeros[at] - 8) * 0.0625f : 0.f;
      }
    }
    f32x4_t sum[MT][NT];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      Frag<T> a[MT];
#pragma unroll
      for (int r = 0; r < MT; ++r) load_x<T>(a[r], xr[r], kt * kTileK + 32 * j + 8 * g, p.K);
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        const uint32_t d = j == 0 ? q[c].x : j == 1 ? q[c].y : j == 2 ? q[c].z : q[c].w;
        float v[8];
        decode8<ZERO>(d, z[c][j / GS], v);
        Frag<T> b;
        frag_from_f32(b, v);
#pragma unroll
        for (int r = 0; r < MT; ++r) {
          const f32x4_t none = {0.f, 0.f, 0.f, 0.f};
          sum[r][c] = mma(a[r], b, j % GS == 0 ? none : sum[r][c]);
          if ((j + 1) % GS == 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[r][c][e] = fmaf(s[c][j / GS], sum[r][c][e], acc[r][c][e]);
          }
        }
      }
    }
  }
  // D layout: lane holds D[4 g + e][l16]
#pragma unroll
  for (int r = 0; r < MT; ++r)
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[w][(16 * r + 4 * g + e) * PITCH + 16 * c + l16] = acc[r][c][e];
  __syncthreads();
  for (int i = tid; i < ROWS * COLS; i += W * kWave) {
    const int m = i / COLS, c = i % COLS, row = m0 + m, n = 16 * t0 + c;
    if (row >= p.M || n >= p.N) continue;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) v += part[k][m * PITCH + c];
    if (p.bias) v += to_f<T>(reinterpret_cast<const T*>(p.bias)[n]);
    if (p.res) v += to_f<T>(reinterpret_cast<const T*>(p.res)[(int64_t)row * p.r_rs + n]);
    reinterpret_cast<T*>(p.out)[(int64_t)row * p.o_rs + n] = from_f<T>(v);
  }
}

template <typename T, int MT, int NT, int GS, bool ZERO> void launch_linear4(const Linear4Args& a, hipStream_t s) {
  constexpr int W = 8;
  const dim3 grid((unsigned)((a.tiles_n + NT - 1) / NT), (unsigned)((a.M + 16 * MT - 1) / (16 * MT)));
  HDCM_LAUNCH((linear4_kernel<T, MT, NT, W, GS, ZERO>), grid, dim3(W * kWave), 0, s, a);
}
template <typename T, int GS, bool ZERO> void pick_rows(const Linear4Args& a, hipStream_t s) {
  if (a.M <= 16) launch_linear4<T, 1, 2, GS, ZERO>(a, s);
  else if (a.M <= 32) launch_linear4<T, 2, 2, GS, ZERO>(a, s);
  else launch_linear4<T, 4, 2, GS, ZERO>(a, s);
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
    d |= (c ^ 8u) << (4 * e);
  }
  packed[dword_at(n, k8, tiles_k)] = d;
}

// One thread per (row, group) of the padded weight.  Without zero points the scale is the group's largest
// magnitude / 7 and c = round(w / s) + 8 in 1..15; with them the range from min(w, 0) to max(w, 0) in 15
// steps, z = round(-min / s).  The codes are taken with the scale as rounded to its type.
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
      d |= ((uint32_t)c ^ 8u) << (4 * e);
    }
    packed[dword_at(n, k8, tiles_k)] = d;
  }
}

// One thread per eight columns of a row: s (c - z), rounded to T.
template <typename T>
__global__ __launch_bounds__(256) void w4_dequant_kernel(const uint32_t* __restrict__ packed, const void* scales, bool s_f32,
                                                         const uint8_t* __restrict__ zeros, int N, int K, int group,
                                                         int tiles_k, int np, T* __restrict__ out, int64_t o_rs) {
  const int k8s = (K + 7) / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)N * k8s) return;
  const int k8 = (int)(i % k8s), n = (int)(i / k8s);
  const int64_t at = (int64_t)(8 * k8 / group) * np + n;
  const float s = 16.f * load_scale(scales, s_f32, at);
  float v[8];
  decode8<true>(packed[dword_at(n, k8, tiles_k)], zeros ? ((int)zeros[at] - 8) * 0.0625f : 0.f, v);
  T* o = out + (int64_t)n * o_rs + 8 * k8;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (8 * k8 + e < K) o[e] = from_f<T>(s * v[e]);
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
  HDCM_CHECK_ARG(hdcm_aligned16(packed), HDCM_EALIGN);
  if (N == 0) return HDCM_OK;
  const int tk = tiles_of(K, kTileK), np = tiles_of(N, kTileN) * kTileN, g = (int)group, n = (int)N, k = (int)K;
  const int64_t total = N * ((K + 7) / 8);
  HDCM_CHECK_ARG(total < ((int64_t)1 << 38), HDCM_EUNSUPPORTED);
  const dim3 grid = threads256(total);
  hipStream_t s = (hipStream_t)stream;
  const uint32_t* d = (const uint32_t*)packed;
  const bool f = scale_dtype == HDCM_F32;
  if (dtype == HDCM_F32)
    HDCM_LAUNCH(w4_dequant_kernel<float>, grid, dim3(256), 0, s, d, scales, f, zeros, n, k, g, tk, np, (float*)out,
                out_row_stride);
  else
    HDCM_LAUNCH(w4_dequant_kernel<bf16_t>, grid, dim3(256), 0, s, d, scales, f, zeros, n, k, g, tk, np, (bf16_t*)out,
                out_row_stride);
  return hdcm_launch_status();
}

extern "C" int hdcm_w4_linear_fwd(const void* x, int64_t x_row_stride, const void* packed, const void* scales,
                                  int scale_dtype, const uint8_t* zeros, int64_t group, const void* bias, const void* res,
                                  int64_t res_row_stride, void* out, int64_t out_row_stride, int64_t M, int64_t N, int64_t K,
                                  int dtype, void* stream) {
  HDCM_CHECK_ARG((dtype == HDCM_F32 || dtype == HDCM_BF16) && (scale_dtype == HDCM_F32 || scale_dtype == HDCM_BF16),
                 HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(M >= 0 && N >= 0 && K > 0, HDCM_EINVAL);
  HDCM_CHECK_ARG(M == 0 || N == 0 || (x && packed && scales && out), HDCM_EINVAL);
  HDCM_CHECK_ARG(M <= 1 || (x_row_stride >= K && out_row_stride >= N && (!res || res_row_stride >= N)), HDCM_EINVAL);
  HDCM_CHECK_ARG(sizes_ok(N, K, group) && M <= 64 * 65535, HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(hdcm_aligned16(packed), HDCM_EALIGN);
  if (M == 0 || N == 0) return HDCM_OK;
  Linear4Args a;
  a.x = x, a.codes = (const uint4*)packed, a.scales = scales, a.zeros = zeros, a.bias = bias, a.res = res, a.out = out;
  a.x_rs = x_row_stride, a.r_rs = res_row_stride, a.o_rs = out_row_stride;
  a.M = (int)M, a.N = (int)N, a.K = (int)K;
  a.tiles_n = tiles_of(N, kTileN), a.tiles_k = tiles_of(K, kTileK), a.np = a.tiles_n * kTileN;
  a.s_f32 = scale_dtype == HDCM_F32;
  hipStream_t s = (hipStream_t)stream;
  dtype == HDCM_F32 ? pick_group<float>(a, (int)group, s) : pick_group<bf16_t>(a, (int)group, s);
  return hdcm_launch_status();
}
