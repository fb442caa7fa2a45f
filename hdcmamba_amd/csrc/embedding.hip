// Token rows of an embedding and the weight's gradient (the reference's nn.Embedding and its autograd,
// train_fineweb.py:49,87):
//   lookup:    y[t] = scale w[id_t], zeros where id_t is no row of the weight
//   gradient:  dw[v] = scale sum_{t: id_t = v} dy[t], fp32 sums in an order that the ids alone fix
// The gradient sorts the positions by token (stable radix passes), cuts the sorted list into units of equal
// length, so that a frequent token costs no more than many rare ones, sums each unit's runs of equal tokens
// in registers and joins the runs that units share in a second launch.  No floating-point atomics.
#include "hdcm_common.h"

using namespace hdcm;

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------ 16 bytes of a row
// E consecutive elements at the type's own alignment (rows of an odd width start anywhere).
template <typename T> constexpr int kE = 16 / sizeof(T);
template <typename T> struct Loose;
template <> struct Loose<bf16_t> {
  typedef u32x4_t type __attribute__((aligned(2)));
};
template <> struct Loose<float> {
  typedef u32x4_t type __attribute__((aligned(4)));
};
// The first n of them (all from E on), zero bits behind
template <typename T> __device__ __forceinline__ u32x4_t load_piece(const T* p, int n) {
  if (n >= kE<T>) return *reinterpret_cast<const typename Loose<T>::type*>(p);
  u32x4_t r = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < kE<T>; ++e)
    if (e < n) {
      if constexpr (sizeof(T) == 2) r[e / 2] |= (uint32_t)p[e] << (16 * (e & 1));
      else r[e] = __float_as_uint(p[e]);
    }
  return r;
}
template <typename T> __device__ __forceinline__ void store_piece(T* p, u32x4_t r, int n) {
  if (n >= kE<T>) {
    *reinterpret_cast<typename Loose<T>::type*>(p) = r;
    return;
  }
#pragma unroll
  for (int e = 0; e < kE<T>; ++e)
    if (e < n) {
      if constexpr (sizeof(T) == 2) p[e] = (T)(r[e / 2] >> (16 * (e & 1)));
      else p[e] = __uint_as_float(r[e]);
    }
}
template <typename T> __device__ __forceinline__ void values(u32x4_t r, float* v) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(r[i] << 16), v[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
  }
}
template <typename T> __device__ __forceinline__ u32x4_t packed(const float* v) {
  const uint4 r = pack16<T>(v);
  return u32x4_t{r.x, r.y, r.z, r.w};
}

// ------------------------------------------------------------------ lookup
// A thread copies U pieces of 16 bytes, 256 pieces apart in the order of the output, so that all lanes work at any
// width; every piece's id, then every piece's row, is in flight before the first is used.
constexpr int kLookThreads = 256;

template <typename T, typename I, int U, bool SCALED>
__global__ __launch_bounds__(kLookThreads) void embedding_kernel(const I* __restrict__ ids, const T* __restrict__ w, int64_t w_rs,
                                                                 T* __restrict__ out, int64_t out_rs, int64_t rows, int V, int D,
                                                                 float scale) {
  const uint32_t P = (D + kE<T> - 1) / kE<T>;
  const int64_t begin = (int64_t)blockIdx.x * (U * kLookThreads), row0 = begin / P;
  const uint32_t at0 = (uint32_t)(begin - row0 * P);
  int64_t row[U], id[U];
  int col[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t at = at0 + u * kLookThreads + threadIdx.x, r = at / P;
    row[u] = row0 + r;
    col[u] = kE<T> * (int)(at - r * P);
    id[u] = row[u] < rows ? (int64_t)ids[row[u]] : -1;
  }
  u32x4_t x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    x[u] = u32x4_t{0, 0, 0, 0};
    if ((uint64_t)id[u] < (uint64_t)V) x[u] = load_piece<T>(w + id[u] * w_rs + col[u], D - col[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (row[u] >= rows) continue;
    if constexpr (SCALED) {
      float v[kE<T>];
      values<T>(x[u], v);
#pragma unroll
      for (int e = 0; e < kE<T>; ++e) v[e] *= scale;
      x[u] = packed<T>(v);
      if ((uint64_t)id[u] >= (uint64_t)V) x[u] = u32x4_t{0, 0, 0, 0};  // of an infinite or negative scale too
    }
    store_piece<T>(out + row[u] * out_rs + col[u], x[u], D - col[u]);
  }
}

template <typename T, typename I>
void launch_lookup(const void* ids, const void* w, int64_t w_rs, void* out, int64_t out_rs, int64_t rows, int64_t V, int64_t D,
                   float scale, hipStream_t s) {
  const int64_t pieces = rows * ((D + kE<T> - 1) / kE<T>);
  const auto go = [&](auto kernel, int U) {
    HDCM_LAUNCH(kernel, dim3((unsigned)((pieces + U * kLookThreads - 1) / (U * kLookThreads))), dim3(kLookThreads), 0, s,
                (const I*)ids, (const T*)w, w_rs, (T*)out, out_rs, rows, (int)V, (int)D, scale);
  };
  if (scale == 1.f) go(embedding_kernel<T, I, 4, false>, 4);
  else go(embedding_kernel<T, I, 4, true>, 4);
}

// ------------------------------------------------------------------ positions in the order of their tokens
// Stable radix passes over digits of up to kDigitBits bits of the token, least significant first: a pass
// counts the digits of each workgroup's stretch of the list, and scatters every stretch behind what the
// counts put before it.  Ids outside the weight and the padding index become the key V, behind all tokens.
constexpr int kSortThreads = 512, kSortWaves = kSortThreads / kWave;
constexpr int kTile = 2048, kPer = kTile / kSortThreads;  // keys of a workgroup's round, and of a thread in it
constexpr int kDigitBits = 9, kBins = 1 << kDigitBits;
constexpr int kMaxGroups = 128;  // workgroups of a pass, so that each may add all counts up by itself

// A pass' input: the caller's ids (first pass) or the keys and positions of the pass before.
struct SortIn {
  const void* ids;  // null: keys, pos
  const int *keys, *pos;
  int id_bytes, V, padding;
  __device__ __forceinline__ int key(int64_t i) const {
    if (!ids) return keys[i];
    const int64_t id = id_bytes == 8 ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
    return (uint64_t)id < (uint64_t)V && id != padding ? (int)id : V;
  }
  __device__ __forceinline__ int position(int64_t i) const { return ids ? (int)i : pos[i]; }
};

__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(SortIn in, int n, int stretch, int shift, int bits, int* counts) {
  __shared__ int count[kBins];
  const int tid = threadIdx.x, bins = 1 << bits;
  if (tid < bins) count[tid] = 0;
  __syncthreads();
  const int64_t b = (int64_t)blockIdx.x * stretch, e = min(b + stretch, (int64_t)n);
  for (int64_t i = b + tid; i < e; i += kSortThreads) atomicAdd(&count[(in.key(i) >> shift) & (bins - 1)], 1);
  __syncthreads();
  if (tid < bins) counts[blockIdx.x * bins + tid] = count[tid];
}

__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(SortIn in, int n, int stretch, int shift, int bits,
                                                                    const int* counts, int* keys, int* pos) {
  __shared__ int next[kBins];              // where the next key of a digit goes
  __shared__ int sums[kSortWaves];
  __shared__ int mine[kSortWaves][kBins];  // a wave's keys of a digit, then where its first goes
  const int tid = threadIdx.x, w = tid / kWave, lane = tid % kWave, bins = 1 << bits;
  // all keys of lower digits, and this digit's in the stretches before
  int before = 0, total = 0;
  if (tid < bins)
    for (int g = 0; g < (int)gridDim.x; ++g) {
      const int c = counts[g * bins + tid];
      before += g < (int)blockIdx.x ? c : 0;
      total += c;
    }
  int scan = total;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int up = __shfl_up(scan, o, kWave);
    scan += lane >= o ? up : 0;
  }
  if (lane == kWave - 1) sums[w] = scan;
  __syncthreads();
  int lower = scan - total;
  for (int i = 0; i < w; ++i) lower += sums[i];
  next[tid] = lower + before;  // kBins == kSortThreads
  const int64_t b = (int64_t)blockIdx.x * stretch, e = min(b + stretch, (int64_t)n);
  for (int64_t t = b; t < e; t += kTile) {
#pragma unroll
    for (int i = 0; i < kSortWaves; ++i) mine[i][tid] = 0;
    __syncthreads();
    int key[kPer], at[kPer], digit[kPer], rank[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int64_t i = t + w * (kPer * kWave) + j * kWave + lane;
      key[j] = i < e ? in.key(i) : 0;
      at[j] = i < e ? in.position(i) : -1;
      digit[j] = (key[j] >> shift) & (bins - 1);
    }
    // the wave's lanes with the same digit, found a bit at a time, rank themselves behind the wave's earlier ones
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      uint64_t same = __ballot(at[j] >= 0);
      for (int k = 0; k < bits; ++k) {
        const bool set = (digit[j] >> k) & 1;
        const uint64_t with = __ballot(set);
        same &= set ? with : ~with;
      }
      const int below = __popcll(same & ((1ull << lane) - 1));
      const int had = mine[w][digit[j]];
      rank[j] = had + below;
      __builtin_amdgcn_wave_barrier();  // all lanes have read before one of them writes
      if (at[j] >= 0 && below == 0) mine[w][digit[j]] = had + __popcll(same);
      __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    int run = next[tid];
#pragma unroll
    for (int i = 0; i < kSortWaves; ++i) {
      const int c = mine[i][tid];
      mine[i][tid] = run;
      run += c;
    }
    next[tid] = run;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int to = mine[w][digit[j]] + rank[j];
      if (at[j] >= 0 && (unsigned)to < (unsigned)n) keys[to] = key[j], pos[to] = at[j];  // (inside, whatever the ids became since)
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ sums of the sorted rows
constexpr int kRowsAhead = 16;  // rows of dy in flight
constexpr int kUnit = 32;       // sorted positions of a wave, a multiple of kRowsAhead
constexpr int kSumThreads = 256, kSumWaves = kSumThreads / kWave;

// dy [.., L, D]: position p lies at (p / L) batch stride + (p % L) row stride.
struct GradRows {
  const void* p;
  int64_t batch, row;
  uint32_t L;
  __device__ __forceinline__ int64_t offset(uint32_t at) const { return (at / L) * batch + (at % L) * row; }
};
struct Sorted {
  const int *keys, *pos;
  int n, V;
};

// Writes (or adds) a finished sum: v[0..E) at columns inside the row.
template <typename TG, typename TO>
__device__ __forceinline__ void put_row(TO* p, const float* sum, float scale, int n, bool add) {
#pragma unroll
  for (int e0 = 0; e0 < kE<TG>; e0 += 4) {
    if (e0 >= n) break;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = sum[e0 + e] * scale;
    if (add) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e0 + e < n) v[e] += to_f<TO>(p[e0 + e]);
    }
    if (e0 + 4 <= n) {
      if constexpr (sizeof(TO) == 2) {
        typedef uint32_t pair_t __attribute__((ext_vector_type(2), aligned(2)));
        *reinterpret_cast<pair_t*>(p + e0) = pair_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
      } else {
        typedef float quad_t __attribute__((ext_vector_type(4), aligned(4)));
        *reinterpret_cast<quad_t*>(p + e0) = quad_t{v[0], v[1], v[2], v[3]};
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e0 + e < n) p[e0 + e] = from_f<TO>(v[e]);
    }
  }
}

__device__ __forceinline__ int64_t lane_value(int64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, lane), hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), lane);
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// A wave takes one unit and 64 pieces of its rows.  A run of equal tokens that lies inside the unit is written
// to dw at once; what the unit holds of a run that began before it goes to its partial row 0, of one that
// begins in it and goes on behind it to its partial row 1.
template <typename TG, typename TO>
__global__ __launch_bounds__(kSumThreads) void embedding_sum_kernel(Sorted s, GradRows g, TO* out, int64_t out_rs, float* part, int D,
                                                                    int slices, float scale, bool add) {
  constexpr int E = kE<TG>;
  const int lane = threadIdx.x % kWave;
  const int64_t wave = (int64_t)blockIdx.x * kSumWaves + threadIdx.x / kWave;
  const int64_t begin = wave / slices * kUnit;
  if (begin >= s.n) return;
  const int slice = (int)(wave % slices), col = (slice * kWave + lane) * E;
  const int end = (int)min(begin + kUnit, (int64_t)s.n);
  const TG* rows = static_cast<const TG*>(g.p) + col;
  float* mine = part + (begin / kUnit * 2 * slices * kWave + slice * kWave + lane) * E;
  const int64_t one = (int64_t)slices * kWave * E;
  float sum[E];
#pragma unroll
  for (int e = 0; e < E; ++e) sum[e] = 0.f;
  bool began = begin == 0 || s.keys[begin - 1] != s.keys[begin], open = false;
  for (int b = (int)begin; b < end; b += kRowsAhead) {
    const int at = min(b + lane, s.n - 1), count = min(kRowsAhead, end - b);
    const int keys = b + lane < s.n ? s.keys[at] : -1;  // no token behind the last
    const int64_t offs = g.offset((uint32_t)s.pos[at]);
    u32x4_t x[kRowsAhead];
#pragma unroll
    for (int j = 0; j < kRowsAhead; ++j) x[j] = load_piece<TG>(rows + lane_value(offs, min(j, count - 1)), D - col);
#pragma unroll
    for (int j = 0; j < kRowsAhead; ++j) {
      const int key = __builtin_amdgcn_readlane(keys, j);
      if (j < count && key < s.V) {
        float v[E];
        values<TG>(x[j], v);
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] += v[e];
        open = __builtin_amdgcn_readlane(keys, j + 1) == key;
        if (!open) {
          if (began) {
            if (col < D) put_row<TG, TO>(out + key * out_rs + col, sum, scale, D - col, add);
          } else {
#pragma unroll
            for (int e = 0; e < E; ++e) mine[e] = sum[e];
          }
#pragma unroll
          for (int e = 0; e < E; ++e) sum[e] = 0.f;
          began = true;
        }
      }
    }
  }
  if (open) {
#pragma unroll
    for (int e = 0; e < E; ++e) mine[(began ? one : 0) + e] = sum[e];
  }
}

// The runs that begin in a unit and end in a later one: the partial rows in the units' order.
template <typename TG, typename TO>
__global__ __launch_bounds__(kSumThreads) void embedding_join_kernel(Sorted s, TO* out, int64_t out_rs, const float* part, int D,
                                                                     int slices, float scale, bool add) {
  constexpr int E = kE<TG>;
  const int lane = threadIdx.x % kWave;
  const int64_t wave = (int64_t)blockIdx.x * kSumWaves + threadIdx.x / kWave;
  const int64_t unit = wave / slices, begin = unit * kUnit, end = begin + kUnit;
  if (end >= s.n) return;
  const int key = s.keys[end];
  if (key >= s.V || s.keys[end - 1] != key) return;
  if (begin > 0 && s.keys[begin - 1] == key) return;  // it began before
  const int slice = (int)(wave % slices), col = (slice * kWave + lane) * E;
  const int64_t one = (int64_t)slices * kWave * E;
  const float* p = part + unit * 2 * one + (slice * kWave + lane) * E;
  float sum[E];
#pragma unroll
  for (int e = 0; e < E; ++e) sum[e] = p[one + e];
  for (int64_t u = unit + 1;; ++u) {
    const float* q = p + (u - unit) * 2 * one;
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] += q[e];
    if ((u + 1) * kUnit >= s.n || s.keys[(u + 1) * kUnit] != key) break;
  }
  if (col < D) put_row<TG, TO>(out + key * out_rs + col, sum, scale, D - col, add);
}

// Zeros in all V rows of D columns.
template <typename T>
__global__ __launch_bounds__(256) void zero_rows_kernel(T* out, int64_t rs, int64_t rows, int D) {
  const uint32_t P = (D + kE<T> - 1) / kE<T>;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / P;
  const int col = kE<T> * (int)(i - row * P);
  if (row < rows) store_piece<T>(out + row * rs + col, u32x4_t{0, 0, 0, 0}, D - col);
}

// ------------------------------------------------------------------ host side
int bit_length(int64_t v) {
  int n = 0;
  for (; v; v >>= 1) ++n;
  return n;
}

// How a call's passes and workspace are cut.
struct Plan {
  int passes, bits, groups, stretch, slices;
  int64_t units;
  size_t list, counts, part;  // bytes of one list of n positions, of the counts, of the partial rows
  size_t bytes() const { return 4 * list + counts + part; }
};
Plan plan_of(int64_t n, int64_t V, int64_t D, int dtype) {
  Plan p;
  const int bits = bit_length(V);  // of the largest key, V
  p.passes = (bits + kDigitBits - 1) / kDigitBits;
  p.bits = (bits + p.passes - 1) / p.passes;
  const int64_t tiles = (n + kTile - 1) / kTile;
  p.stretch = (int)((tiles + kMaxGroups - 1) / kMaxGroups * kTile);
  p.groups = (int)((n + p.stretch - 1) / p.stretch);
  const int E = 16 / hdcm_elt_size(dtype);
  p.slices = (int)((D + kWave * E - 1) / (kWave * E));
  p.units = (n + kUnit - 1) / kUnit;
  const auto whole = [](size_t b) { return (b + 255) / 256 * 256; };
  p.list = whole((size_t)n * 4);
  p.counts = whole((size_t)p.groups * kBins * 4);
  p.part = whole((size_t)p.units * 2 * p.slices * kWave * E * 4);
  return p;
}

constexpr int64_t kMaxVocab = (int64_t)1 << 30, kMaxPositions = (int64_t)1 << 30, kMaxWidth = (int64_t)1 << 24;

template <typename TG, typename TO>
void launch_sums(const Plan& p, const Sorted& s, const GradRows& g, void* out, int64_t out_rs, float* part, int64_t D, float scale,
                 bool add, hipStream_t stream) {
  const dim3 grid((unsigned)((p.units * p.slices + kSumWaves - 1) / kSumWaves));
  HDCM_LAUNCH((embedding_sum_kernel<TG, TO>), grid, dim3(kSumThreads), 0, stream, s, g, (TO*)out, out_rs, part, (int)D, p.slices,
              scale, add);
  if (p.units > 1)
    HDCM_LAUNCH((embedding_join_kernel<TG, TO>), grid, dim3(kSumThreads), 0, stream, s, (TO*)out, out_rs, (const float*)part, (int)D,
                p.slices, scale, add);
}

}  // namespace

extern "C" int hdcm_embedding_fwd(const void* ids, int id_bytes, const void* w, int64_t w_row_stride, void* out,
                                  int64_t out_row_stride, int64_t rows, int64_t V, int64_t D, float scale, int dtype, void* stream) {
  HDCM_CHECK_ARG(dtype == HDCM_F32 || dtype == HDCM_BF16, HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(id_bytes == 4 || id_bytes == 8, HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(rows >= 0 && V >= 0 && D >= 0, HDCM_EINVAL);
  if (rows == 0 || D == 0) return HDCM_OK;
  HDCM_CHECK_ARG(ids && out && (w || V == 0), HDCM_EINVAL);
  HDCM_CHECK_ARG((w_row_stride >= D || V <= 1) && (out_row_stride >= D || rows <= 1), HDCM_EINVAL);
  HDCM_CHECK_ARG(V <= kMaxVocab && D <= kMaxWidth && rows <= kMaxPositions, HDCM_EUNSUPPORTED);
  hipStream_t s = (hipStream_t)stream;
  const auto go = [&](auto launch) { launch(ids, w, w_row_stride, out, out_row_stride, rows, V, D, scale, s); };
  if (dtype == HDCM_F32) id_bytes == 8 ? go(launch_lookup<float, int64_t>) : go(launch_lookup<float, int32_t>);
  else id_bytes == 8 ? go(launch_lookup<bf16_t, int64_t>) : go(launch_lookup<bf16_t, int32_t>);
  return hdcm_launch_status();
}

extern "C" size_t hdcm_embedding_grad_workspace_bytes(int64_t B, int64_t L, int64_t V, int64_t D, int dtype) {
  if (B <= 0 || L <= 0 || V <= 0 || D <= 0 || L > kMaxPositions / B || V > kMaxVocab || D > kMaxWidth) return 0;
  return plan_of(B * L, V, D, dtype).bytes();
}

extern "C" int hdcm_embedding_grad(const void* ids, int id_bytes, const void* dy, int64_t dy_batch_stride, int64_t dy_row_stride,
                                   void* dw, int64_t dw_row_stride, int dw_dtype, void* ws, size_t ws_bytes, int64_t B, int64_t L,
                                   int64_t V, int64_t D, float scale, int64_t padding_idx, int accumulate, int dtype,
                                   void* stream) {
  HDCM_CHECK_ARG(dtype == HDCM_F32 || dtype == HDCM_BF16, HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(dw_dtype == HDCM_F32 || dw_dtype == HDCM_BF16, HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(id_bytes == 4 || id_bytes == 8, HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(B >= 0 && L >= 0 && V >= 0 && D >= 0, HDCM_EINVAL);
  HDCM_CHECK_ARG(padding_idx >= -1 && (padding_idx < V || V == 0), HDCM_EINVAL);
  const bool none = B == 0 || L == 0;
  if (V == 0 || D == 0 || (none && accumulate)) return HDCM_OK;
  HDCM_CHECK_ARG(dw && (none || (ids && dy)), HDCM_EINVAL);
  HDCM_CHECK_ARG(dw_row_stride >= D || V == 1, HDCM_EINVAL);
  HDCM_CHECK_ARG(none || ((dy_row_stride >= D || dy_row_stride == 0 || L == 1) && (dy_batch_stride >= 0 || B == 1)), HDCM_EINVAL);
  HDCM_CHECK_ARG(V <= kMaxVocab && D <= kMaxWidth && (none || L <= kMaxPositions / B), HDCM_EUNSUPPORTED);
  hipStream_t s = (hipStream_t)stream;
  Plan p{};
  if (!none) {
    p = plan_of(B * L, V, D, dtype);
    HDCM_CHECK_ARG(ws && ws_bytes >= p.bytes(), HDCM_EWORKSPACE);
    HDCM_CHECK_ARG(hdcm_aligned16(ws), HDCM_EALIGN);
  }
  if (!accumulate) {
    const int64_t P = (D + 16 / hdcm_elt_size(dw_dtype) - 1) / (16 / hdcm_elt_size(dw_dtype));
    const dim3 grid((unsigned)((V * P + 255) / 256));
    if (dw_dtype == HDCM_F32) HDCM_LAUNCH(zero_rows_kernel<float>, grid, dim3(256), 0, s, (float*)dw, dw_row_stride, V, (int)D);
    else HDCM_LAUNCH(zero_rows_kernel<bf16_t>, grid, dim3(256), 0, s, (bf16_t*)dw, dw_row_stride, V, (int)D);
  }
  if (none) return hdcm_launch_status();
  const int n = (int)(B * L);
  char* at = (char*)ws;
  int* lists[4];
  for (int i = 0; i < 4; ++i, at += p.list) lists[i] = (int*)at;
  int* counts = (int*)at;
  float* part = (float*)(at + p.counts);
  SortIn in{ids, nullptr, nullptr, id_bytes, (int)V, (int)padding_idx};
  for (int k = 0; k < p.passes; ++k) {
    int *keys = lists[2 * (k & 1)], *pos = lists[2 * (k & 1) + 1];
    HDCM_LAUNCH(sort_count_kernel, dim3(p.groups), dim3(kSortThreads), 0, s, in, n, p.stretch, k * p.bits, p.bits, counts);
    HDCM_LAUNCH(sort_scatter_kernel, dim3(p.groups), dim3(kSortThreads), 0, s, in, n, p.stretch, k * p.bits, p.bits,
                (const int*)counts, keys, pos);
    in = SortIn{nullptr, keys, pos, 4, (int)V, -1};
  }
  const Sorted sorted{in.keys, in.pos, n, (int)V};
  const GradRows g{dy, dy_batch_stride, dy_row_stride, (uint32_t)L};
  const auto go = [&](auto launch) { launch(p, sorted, g, dw, dw_row_stride, part, D, scale, accumulate != 0, s); };
  if (dtype == HDCM_F32) dw_dtype == HDCM_F32 ? go(launch_sums<float, float>) : go(launch_sums<float, bf16_t>);
  else dw_dtype == HDCM_F32 ? go(launch_sums<bf16_t, float>) : go(launch_sums<bf16_t, bf16_t>);
  return hdcm_launch_status();
}
