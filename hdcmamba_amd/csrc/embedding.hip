// Token rows of an embedding and the weight's gradient (the reference's nn.Embedding and its autograd,
// train_fineweb.py:49,87):
//   lookup:    y[t] = scale w[id_t], zeros where id_t is no row of the weight
//   gradient:  dw[v] = scale sum_{t: id_t = v} dy[t], fp32 sums in an order that the ids, the sizes and the types fix
// The gradient of many positions sorts them by token (stable radix passes), cuts the sorted list into units of equal
// length, so that a frequent token costs no more than many rare ones, sums each unit's runs of equal tokens in
// registers, joins the runs that units share in LDS, and those that workgroups share in a last launch.  Few positions
// need no sorting: every workgroup looks for its own tokens among all ids.  No floating-point atomics.
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
template <typename T, bool STREAM = false> __device__ __forceinline__ u32x4_t load_piece(const T* p, int n) {
  if (STREAM && n >= kE<T>) return __builtin_nontemporal_load(reinterpret_cast<const typename Loose<T>::type*>(p));
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
template <typename T, bool STREAM = false> __device__ __forceinline__ void store_piece(T* p, u32x4_t r, int n) {
  if (n >= kE<T>) {
    if constexpr (STREAM) __builtin_nontemporal_store(r, reinterpret_cast<typename Loose<T>::type*>(p));
    else *reinterpret_cast<typename Loose<T>::type*>(p) = r;
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

// What is read or written once goes past the caches where it is more than they hold of it until it is used again.  us
// a call, three sets of inputs in turn, cached and past the caches.  Rows of dy (bf16, 50304 tokens, dy and dw together):
// 32768 x 768 (121 MiB) 44.9 and 47.1, 32768 x 1024 (162) 52.7 and 50.0, 131072 x 1024 (354) 115 and 100, 131072 x 2048
// (708) 205 and 160.  Rows looked up: 131072 x 2048 (512 MiB) 157 and 113; 32768 x 1024 (64) 16.7 and 16.2, but there the next
// kernel finds them in the caches.
constexpr int64_t kStreamBytes = (int64_t)128 << 20;

// ------------------------------------------------------------------ lookup
// A thread copies U pieces of 16 bytes, 256 pieces apart in the order of the output, so that all lanes work at any
// width; every piece's id, then every piece's row, is in flight before the first is used.
// us recorded with 1, 2 and 4: 16 x 2048 bf16 1.9, 2.0, 2.7; 1024 x 1024 2.1, 2.3, 3.0; 8192 x 1024 6.1, 5.7, 6.7; 32768 x 1024
// 16.8, 16.7, 17.0 (4 TB/s of writes, 5 in all).
constexpr int kLookThreads = 256;
constexpr int64_t kLookSmall = 1 << 18;

template <typename T, typename I, int U, bool SCALED, bool STREAM>
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
    store_piece<T, STREAM>(out + row[u] * out_rs + col[u], x[u], D - col[u]);
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
  const bool scaled = scale != 1.f;
  if (pieces <= kLookSmall) scaled ? go(embedding_kernel<T, I, 1, true, false>, 1) : go(embedding_kernel<T, I, 1, false, false>, 1);
  else if (pieces * 16 <= kStreamBytes) scaled ? go(embedding_kernel<T, I, 2, true, false>, 2) : go(embedding_kernel<T, I, 2, false, false>, 2);
  else scaled ? go(embedding_kernel<T, I, 2, true, true>, 2) : go(embedding_kernel<T, I, 2, false, true>, 2);
}

// ------------------------------------------------------------------ the gradient's rows
// dy [.., L, D]: position p lies at (p / L) batch stride + (p % L) row stride; L 0: one batch.
struct GradRows {
  const void* p;
  int64_t batch, row;
  uint32_t L;
  __device__ __forceinline__ int64_t offset(uint32_t at) const {
    if (!L) return at * row;
    const uint32_t b = at / L;
    return b * batch + (at - b * L) * row;
  }
};

// The caller's ids as keys: what is no token of the weight, and the padding index, becomes V.
struct Ids {
  const void* p;
  int bytes, V, padding;
  __device__ __forceinline__ int key(int64_t i) const {
    const int64_t id = bytes == 8 ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
    return (uint64_t)id < (uint64_t)V && id != padding ? (int)id : V;
  }
};

// Writes (or adds) a finished sum: E columns from p on, n of them inside the row.
template <int E, typename TO> __device__ __forceinline__ void put_row(TO* p, const float* sum, float scale, int n, bool add) {
#pragma unroll
  for (int e0 = 0; e0 < E; e0 += 4) {
    if (e0 >= n) break;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = sum[e0 + e] * scale;
    if (e0 + 4 <= n) {
      if constexpr (sizeof(TO) == 2) {
        typedef uint32_t pair_t __attribute__((ext_vector_type(2), aligned(2)));
        if (add) {
          const pair_t old = *reinterpret_cast<const pair_t*>(p + e0);
#pragma unroll
          for (int i = 0; i < 2; ++i) v[2 * i] += __uint_as_float(old[i] << 16), v[2 * i + 1] += __uint_as_float(old[i] & 0xffff0000u);
        }
        *reinterpret_cast<pair_t*>(p + e0) = pair_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
      } else {
        typedef float quad_t __attribute__((ext_vector_type(4), aligned(4)));
        quad_t q = {v[0], v[1], v[2], v[3]};
        if (add) q += *reinterpret_cast<const quad_t*>(p + e0);
        *reinterpret_cast<quad_t*>(p + e0) = q;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e0 + e < n) p[e0 + e] = from_f<TO>(v[e] + (add ? to_f<TO>(p[e0 + e]) : 0.f));
    }
  }
}

__device__ __forceinline__ int64_t lane_value(int64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, lane), hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), lane);
  return (int64_t)((uint64_t)hi << 32 | lo);
}

constexpr int kAhead = 8;                                       // rows of dy that a wave has in flight
constexpr int kSumThreads = 512, kSumWaves = kSumThreads / kWave;  // of the kernels that add rows up

// A wave's lanes hold the offsets of `count` (1..kAhead) rows: loads them all.
template <bool STREAM, typename T>
__device__ __forceinline__ void load_rows(u32x4_t (&x)[kAhead], const T* rows, int64_t offs, int count, int n) {
#pragma unroll
  for (int j = 0; j < kAhead; ++j) x[j] = load_piece<T, STREAM>(rows + lane_value(offs, min(j, count - 1)), n);
}
template <typename T> __device__ __forceinline__ void add_piece(float* sum, u32x4_t x) {
  float v[kE<T>];
  values<T>(x, v);
#pragma unroll
  for (int e = 0; e < kE<T>; ++e) sum[e] += v[e];
}

// Sums of the rows of a list that is sorted by token, by the kSumWaves waves of a workgroup, for 64 pieces of the
// rows.  A wave takes `unit` positions in a row (a multiple of kAhead), the first from `first` on.  A run of equal
// tokens inside a unit is written to dw at once.  What a unit holds of a run that began before it (its head) or goes on
// behind it meets in LDS: the wave in which a run begins adds the heads behind it.  A run that goes on behind the
// workgroup leaves the workgroup's part of it at partial + one where it began here, else at partial.
struct List {
  int64_t first;
  int n, V, unit;  // of n positions; keys from V on are no tokens
  uint32_t last;   // the largest position
  // Nor are negative ones, which a caller that writes its ids meanwhile could leave in the sorted list, and positions are
  // taken into the list: nothing outside the buffers is read or written then either.
  __device__ __forceinline__ bool token(int key) const { return (unsigned)key < (unsigned)V; }
};
template <typename TG, typename TO> struct Sums {
  const TG* rows;  // at the lane's columns
  GradRows g;
  TO* out;
  int64_t out_rs;
  int col, D;
  float scale;
  bool add;
  __device__ __forceinline__ void put(int64_t token, const float* sum) const {
    if (col < D) put_row<kE<TG>, TO>(out + token * out_rs + col, sum, scale, D - col, add);
  }
};
template <typename TG> struct Heads {
  __attribute__((aligned(16))) float sum[kSumWaves][kWave * kE<TG>];
  int passes[kSumWaves];  // whether a wave's unit is one run that began before it and goes on behind it
};

template <bool STREAM, typename TG, typename TO, typename Key, typename Pos>
__device__ __forceinline__ void add_up(const List& l, Key key_at, Pos pos_at, const Sums<TG, TO>& o, Heads<TG>& head, float* partial,
                                       int64_t one) {
  constexpr int E = kE<TG>;
  const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
  const int64_t begin = l.first + (int64_t)w * l.unit, end = min(begin + l.unit, (int64_t)l.n);
  float sum[E] = {};
  // before: the run at hand began before the unit; open: it goes on behind what was added
  bool before = false, open = false, has_head = false;
  int last = l.V;
  for (int64_t b = begin; b < end; b += kAhead) {
    // lanes up to kAhead: the batch and the key behind it; the last lane: the key before it
    const int64_t mine = lane < kWave - 1 ? b + lane : b - 1, at = max(min(mine, (int64_t)l.n - 1), (int64_t)0);
    const int count = (int)min((int64_t)kAhead, end - b);
    const int found = key_at(at), keys = mine >= 0 && mine < l.n ? found : -1;  // no token before the first or behind the last
    u32x4_t x[kAhead];
    load_rows<STREAM, TG>(x, o.rows, o.g.offset(min((uint32_t)pos_at(at), l.last)), count, o.D - o.col);
    if (b == begin) has_head = before = __builtin_amdgcn_readlane(keys, kWave - 1) == __builtin_amdgcn_readlane(keys, 0);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int key = __builtin_amdgcn_readlane(keys, j);
      if (j < count && l.token(key)) {
        add_piece<TG>(sum, x[j]);
        open = __builtin_amdgcn_readlane(keys, j + 1) == key;
        last = key;
        if (!open) {
          if (before) {
#pragma unroll
            for (int e = 0; e < E; ++e) head.sum[w][lane * E + e] = sum[e];
          } else {
            o.put(key, sum);
          }
#pragma unroll
          for (int e = 0; e < E; ++e) sum[e] = 0.f;
          before = false;
        }
      }
    }
  }
  if (open && before) {
#pragma unroll
    for (int e = 0; e < E; ++e) head.sum[w][lane * E + e] = sum[e];
  }
  if (lane == 0) head.passes[w] = open && before;
  __syncthreads();
  if (w == 0 && has_head && l.token(key_at(begin))) {  // a run that came from before the workgroup
    float t[E];
#pragma unroll
    for (int e = 0; e < E; ++e) t[e] = head.sum[0][lane * E + e];
    for (int i = 0; i + 1 < kSumWaves && head.passes[i]; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) t[e] += head.sum[i + 1][lane * E + e];
#pragma unroll
    for (int e = 0; e < E; ++e) partial[e] = t[e];
  }
  if (open && !before) {
    int i = w;
    do {
      if (++i == kSumWaves) break;
#pragma unroll
      for (int e = 0; e < E; ++e) sum[e] += head.sum[i][lane * E + e];
    } while (head.passes[i]);
    if (i < kSumWaves) {
      o.put(last, sum);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) partial[one + e] = sum[e];
    }
  }
}

// ------------------------------------------------------------------ the order of tokens within a workgroup
constexpr int kDigitBits = 9, kBins = 1 << kDigitBits;

// Ranks keys by digit, stably: thread `lane` of wave w holds the keys (w rounds + j) 64 + lane, j < rounds <= PER.  rank[j] becomes
// how many earlier keys of the wave have the same digit; mine[w][d] the wave's keys of digit d.  The wave's lanes with
// the same digit are found a bit at a time.
template <int PER> __device__ __forceinline__ void rank_digits(const int (&digit)[PER], const bool (&there)[PER], int rounds, int bits,
                                                               int* mine, int (&rank)[PER]) {
  const int lane = threadIdx.x % kWave;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (j >= rounds) break;
    uint64_t same = __ballot(there[j]);
    for (int k = 0; k < bits; ++k) {
      const bool set = (digit[j] >> k) & 1;
      const uint64_t with = __ballot(set);
      same &= set ? with : ~with;
    }
    const int below = __popcll(same & ((1ull << lane) - 1)), had = mine[digit[j]];
    rank[j] = had + below;
    __builtin_amdgcn_wave_barrier();  // all lanes have read before one of them writes
    if (there[j] && below == 0) mine[digit[j]] = had + __popcll(same);
    __builtin_amdgcn_wave_barrier();
  }
}
// The waves' keys of digit d, mine[w][d], become where the first of them goes, `next` being where the digit's first
// goes; returns where its next one will.
template <int WAVES> __device__ __forceinline__ int place_digit(int (*mine)[kBins], const int (&count)[WAVES], int d, int next) {
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    mine[i][d] = next;
    next += count[i];
  }
  return next;
}
// Exclusive sum of v over the workgroup's threads, and the whole sum; sums: an int for each wave.
template <int WAVES> __device__ __forceinline__ int sum_before(int v, int* sums, int& all) {
  const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
  int scan = v;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int up = __shfl_up(scan, o, kWave);
    scan += lane >= o ? up : 0;
  }
  if (lane == kWave - 1) sums[w] = scan;
  __syncthreads();
  int before = scan - v;
  all = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    before += i < w ? sums[i] : 0;
    all += sums[i];
  }
  return before;
}

// ------------------------------------------------------------------ few positions: one launch
// Workgroup g of G (for each 64 pieces of the rows) takes the tokens g, g + G, .. (up to kBins of them: frequent
// tokens are often neighbours), finds their positions among all ids, orders them by token in LDS, writes zeros
// to the rows of those that it has not found and adds up the others'.  384 x 256 of 1024 tokens 6.0 us: a chain of the ids'
// arrival, four barriers, the rows' arrival and a join (0.7 MB moved).  With each workgroup's tokens adjacent and its
// frequent ones one after the other it took 11.
constexpr int kFewPositions = 512, kFewPer = kFewPositions / kSumThreads;

template <typename TG, typename TO>
__global__ __launch_bounds__(kSumThreads) void embedding_few_kernel(Ids ids, int n, GradRows g, TO* out, int64_t out_rs, int D,
                                                                    int slices, int bits, float scale, bool add) {
  constexpr int E = kE<TG>;
  __shared__ Heads<TG> head;
  __shared__ int mine[kSumWaves][kBins];
  __shared__ int sums[kSumWaves];
  __shared__ uint16_t token[kFewPositions], at[kFewPositions];  // the found positions, by token
  __shared__ bool none[kBins];                                   // tokens that were not found
  const int tid = threadIdx.x, w = tid / kWave, lane = tid % kWave;
  const uint32_t G = gridDim.x / slices, group = blockIdx.x / slices;
  const int slice = blockIdx.x % slices, col = (slice * kWave + lane) * E;
  int digit[kFewPer], rank[kFewPer];
  bool there[kFewPer];
#pragma unroll
  for (int j = 0; j < kFewPer; ++j) {
    const int i = (w * kFewPer + j) * kWave + lane;
    digit[j] = i < n ? ids.key(i) : ids.V;
  }
#pragma unroll
  for (int i = 0; i < kSumWaves; ++i) mine[i][tid] = 0;  // kBins == kSumThreads
#pragma unroll
  for (int j = 0; j < kFewPer; ++j) {
    const uint32_t key = digit[j], r = key / G;
    there[j] = key < (uint32_t)ids.V && key - r * G == group;
    digit[j] = there[j] ? (int)r : 0;
  }
  __syncthreads();
  rank_digits<kFewPer>(digit, there, kFewPer, bits, mine[w], rank);
  __syncthreads();
  int each[kSumWaves], count = 0, found;
#pragma unroll
  for (int i = 0; i < kSumWaves; ++i) count += each[i] = mine[i][tid];
  place_digit<kSumWaves>(mine, each, tid, sum_before<kSumWaves>(count, sums, found));
  none[tid] = count == 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kFewPer; ++j) {
    if (!there[j]) continue;
    const int to = mine[w][digit[j]] + rank[j];
    token[to] = (uint16_t)digit[j], at[to] = (uint16_t)((w * kFewPer + j) * kWave + lane);
  }
  const Sums<TG, TO> o{static_cast<const TG*>(g.p) + col, g, out, out_rs, col, D, scale, add};
  if (!add) {
    const float zeros[E] = {};
    const int tokens = (int)((ids.V - group + G - 1) / G);
    for (int r = w; r < tokens; r += kSumWaves)
      if (none[r] && col < D) put_row<E, TO>(out + ((int64_t)r * G + group) * out_rs + col, zeros, 1.f, D - col, false);
  }
  __syncthreads();
  const int unit = (found + kSumWaves * kAhead - 1) / (kSumWaves * kAhead) * kAhead;
  add_up<false, TG, TO>(List{0, found, ids.V, unit, (uint32_t)n - 1}, [&](int64_t i) { return (int)(token[i] * G + group); }, [&](int64_t i) { return at[i]; }, o,
                              head, nullptr, 0);
}

// ------------------------------------------------------------------ many positions in the order of their tokens
// Stable radix passes over digits of up to kDigitBits bits of the token, least significant first.  A workgroup
// scatters its stretch of the list behind the keys of lower digits and those of the same digit in the stretches
// before, which a launch before has counted.  Up to kOneGroup positions are one workgroup's work: all passes in LDS, in one
// launch.
// Bound by latency: without zeros to write a count takes 3 us and a scatter 5 at 32768 positions (launch, ids, counts,
// stores); 98 MiB of zeros, which alone take 15, make two passes 9 us longer (all with the scatters; a third of them with the
// counts 11).  us a call of 32768 x 1024, 131072 x 1024 and 1048576 x 64 of 50304 tokens: one key a thread 45.1, 99, 223 (64
// groups), two 47.5, 97, 177, in up to 256 groups 169, in 512 229.  4096 positions of two passes: 19 us a call sorted by one
// workgroup, 27 in four launches; 8192 24 and 27; 16384 (16 keys a thread) 44 and 27.
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kMaxGroups = 256;    // workgroups of a pass, so that each may add all counts up by itself
constexpr int kOneKeyGroups = 64;  // up to so many take one key a thread in a round, more take two
constexpr int kCountAhead = 16;                           // keys or counts of a thread in flight
constexpr int kOnePer = 8, kOneGroup = kOnePer * kSortThreads;

// A pass' input: the caller's ids (first pass) or the keys and positions of the pass before.
struct SortIn {
  Ids ids;
  const int *keys, *pos;  // null: ids
  __device__ __forceinline__ int key(int64_t i) const { return keys ? keys[i] : ids.key(i); }
  __device__ __forceinline__ int position(int64_t i) const { return keys ? pos[i] : (int)i; }
};
struct Pass {
  int n, stretch, groups, shift, bits;
};

// Zeros for the weight's gradient, written by the workgroups of a sorting launch that have nothing to sort: these
// launches are short and leave most CUs idle.  Bytes [begin, end), kFillBytes a workgroup.
constexpr int kFillAhead = 4, kFillBytes = kFillAhead * kSortThreads * 16;
struct Fill {
  char* p;
  int64_t begin, end;
};
__device__ __forceinline__ void fill_part(const Fill& f, int64_t part) {
  typedef u32x4_t loose_t __attribute__((aligned(2)));
  const int64_t b = f.begin + part * kFillBytes;
#pragma unroll
  for (int u = 0; u < kFillAhead; ++u) {
    const int64_t i = b + (u * kSortThreads + (int)threadIdx.x) * 16;
    if (i + 16 <= f.end) *reinterpret_cast<loose_t*>(f.p + i) = u32x4_t{0, 0, 0, 0};
    else
      for (int64_t k = i; k < f.end; k += 2) *reinterpret_cast<uint16_t*>(f.p + k) = 0;
  }
}

__global__ __launch_bounds__(kSortThreads) void sort_one_kernel(Ids ids, int n, int passes, int bits, int* keys, int* pos, Fill fill) {
  __shared__ int sums[kSortWaves];
  __shared__ int mine[kSortWaves][kBins];  // a wave's keys of a digit, then where its first goes
  __shared__ int list[kOneGroup];
  __shared__ uint16_t place[kOneGroup];
  if (blockIdx.x > 0) {
    fill_part(fill, (int)blockIdx.x - 1);
    return;
  }
  const int tid = threadIdx.x, w = tid / kWave, lane = tid % kWave;
  const int per = (n + kSortThreads - 1) / kSortThreads;  // rounds of the keys that there are
  int key[kOnePer], at[kOnePer], digit[kOnePer], rank[kOnePer];
  bool there[kOnePer];
#pragma unroll
  for (int j = 0; j < kOnePer; ++j) {
    at[j] = (w * per + j) * kWave + lane;
    there[j] = j < per && at[j] < n;
    key[j] = there[j] ? ids.key(at[j]) : 0;
  }
  for (int k = 0; k < passes; ++k) {
    for (int i = tid; i < kSortWaves * kBins; i += kSortThreads) mine[i / kBins][i % kBins] = 0;
#pragma unroll
    for (int j = 0; j < kOnePer; ++j) digit[j] = (key[j] >> (k * bits)) & ((1 << bits) - 1);
    __syncthreads();
    rank_digits<kOnePer>(digit, there, per, bits, mine[w], rank);
    __syncthreads();
    int each[kSortWaves] = {}, total = 0, all;
    if (tid < kBins)
#pragma unroll
      for (int i = 0; i < kSortWaves; ++i) total += each[i] = mine[i][tid];
    const int lower = sum_before<kSortWaves>(total, sums, all);
    if (tid < kBins) place_digit<kSortWaves>(mine, each, tid, lower);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kOnePer; ++j)
      if (there[j]) {
        const int to = mine[w][digit[j]] + rank[j];
        list[to] = key[j], place[to] = (uint16_t)at[j];
      }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kOnePer; ++j)
      if (there[j]) {
        const int i = (w * per + j) * kWave + lane;
        key[j] = list[i], at[j] = place[i];
      }
  }
#pragma unroll
  for (int j = 0; j < kOnePer; ++j)
    if (there[j]) {
      const int i = (w * per + j) * kWave + lane;
      keys[i] = key[j], pos[i] = at[j];
    }
}

template <int kPer> __global__ __launch_bounds__(kSortThreads) void sort_count_kernel(SortIn in, Pass p, int* counts) {
  constexpr int kTile = kPer * kSortThreads;
  __shared__ int count[kBins];
  const int tid = threadIdx.x;
  if (tid < kBins) count[tid] = 0;
  __syncthreads();
  const int64_t b = (int64_t)blockIdx.x * p.stretch, e = min(b + p.stretch, (int64_t)p.n);
  for (int64_t t = b; t < e; t += kTile) {
    int key[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int64_t i = t + j * kSortThreads + tid;
      key[j] = i < e ? in.key(i) : 0;
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (t + j * kSortThreads + tid < e) atomicAdd(&count[(key[j] >> p.shift) & ((1 << p.bits) - 1)], 1);
  }
  __syncthreads();
  if (tid < kBins) counts[blockIdx.x * kBins + tid] = count[tid];
}

template <int kPer>
__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(SortIn in, Pass p, const int* counts, int* keys, int* pos,
                                                                    Fill fill) {
  constexpr int kTile = kPer * kSortThreads;
  __shared__ int sums[kSortWaves];
  __shared__ int mine[kSortWaves][kBins];  // a wave's keys of a digit, then where its first goes
  if ((int)blockIdx.x >= p.groups) {
    fill_part(fill, (int)blockIdx.x - p.groups);
    return;
  }
  const int tid = threadIdx.x, w = tid / kWave, lane = tid % kWave;
  const int64_t b = (int64_t)blockIdx.x * p.stretch, e = min(b + p.stretch, (int64_t)p.n);
  int key[kPer], at[kPer];
  const auto load = [&](int64_t t) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int64_t i = t + (w * kPer + j) * kWave + lane;
      key[j] = i < e ? in.key(i) : 0;
      at[j] = i < e ? in.position(i) : -1;
    }
  };
  load(b);
  int before = 0, total = 0;  // keys of digit `tid`: in the stretches before, in all
  if (tid < kBins) {
    for (int g0 = 0; g0 < p.groups; g0 += kCountAhead) {
      int c[kCountAhead];
#pragma unroll
      for (int g = 0; g < kCountAhead; ++g) c[g] = counts[min(g0 + g, p.groups - 1) * kBins + tid];
#pragma unroll
      for (int g = 0; g < kCountAhead; ++g) {
        before += g0 + g < (int)blockIdx.x ? c[g] : 0;
        total += g0 + g < p.groups ? c[g] : 0;
      }
    }
  }
  int all;
  int next = sum_before<kSortWaves>(total, sums, all) + before;  // where the next key of digit `tid` goes
  for (int64_t t = b; t < e; t += kTile) {
    for (int i = tid; i < kSortWaves * kBins; i += kSortThreads) mine[i / kBins][i % kBins] = 0;
    __syncthreads();
    int digit[kPer], rank[kPer];
    bool there[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) there[j] = at[j] >= 0, digit[j] = (key[j] >> p.shift) & ((1 << p.bits) - 1);
    rank_digits<kPer>(digit, there, kPer, p.bits, mine[w], rank);
    __syncthreads();
    if (tid < kBins) {
      int each[kSortWaves];
#pragma unroll
      for (int i = 0; i < kSortWaves; ++i) each[i] = mine[i][tid];
      next = place_digit<kSortWaves>(mine, each, tid, next);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int to = mine[w][digit[j]] + rank[j];
      if (there[j] && (unsigned)to < (unsigned)p.n) keys[to] = key[j], pos[to] = at[j];  // (whatever the ids became since the count)
    }
    load(t + kTile);
    __syncthreads();
  }
}

// Zeros in all rows of a gradient whose rows are not adjacent.
template <typename T>
__global__ __launch_bounds__(256) void zero_rows_kernel(T* out, int64_t rs, int64_t rows, int D) {
  const uint32_t P = (D + kE<T> - 1) / kE<T>;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / P;
  const int col = kE<T> * (int)(i - row * P);
  if (row < rows) store_piece<T>(out + row * rs + col, u32x4_t{0, 0, 0, 0}, D - col);
}

// ------------------------------------------------------------------ sums of the sorted rows
// Bound by the rows of dy, each read once where it lies: 32768 x 1024 bf16 17.9 us (67 MB of rows and 20 of sums, 4.9 TB/s),
// 131072 x 2048 108 (537 MB, 5.2 with the sums; 149 with loads through the caches).  Eight rows ahead leave 6 waves a SIMD;
// 16 rows ahead 19.0.  Units of 8, 16 and 32 positions: 32768 x 1024 18.5, 17.9, 21.1; 131072 x 2048 and the join behind it
// 113 + 22, 112 + 14, 108 + 8.  A contiguous part of the groups for each XCD: 181 for 149.
struct Sorted {
  const int *keys, *pos;
  int n, V, unit;
};

template <bool STREAM, typename TG, typename TO>
__global__ __launch_bounds__(kSumThreads) void embedding_sum_kernel(Sorted s, GradRows g, TO* out, int64_t out_rs, float* partial,
                                                                    int D, int slices, float scale, bool add) {
  constexpr int E = kE<TG>;
  __shared__ Heads<TG> head;
  const int lane = threadIdx.x % kWave, slice = blockIdx.x % slices, col = (slice * kWave + lane) * E;
  const int64_t group = blockIdx.x / slices, one = (int64_t)slices * kWave * E;
  add_up<STREAM, TG, TO>(List{group * kSumWaves * s.unit, s.n, s.V, s.unit, (uint32_t)s.n - 1}, [&](int64_t i) { return s.keys[i]; },
                 [&](int64_t i) { return s.pos[i]; },
                 Sums<TG, TO>{static_cast<const TG*>(g.p) + col, g, out, out_rs, col, D, scale, add}, head,
                 partial + group * 2 * one + (slice * kWave + lane) * E, one);
}

// The runs that begin in one workgroup of the sums and end in a later one: the partial rows in their order.  The run's end is
// found 64 workgroups at a time, and its partial rows are shared by the waves: 4 us at 32768 positions of text, 8 where
// a quarter of 131072 is one token (726 when one wave added its partial rows one after the other).
template <typename TG, typename TO>
__global__ __launch_bounds__(kSumThreads) void embedding_join_kernel(Sorted s, TO* out, int64_t out_rs, const float* partial, int D,
                                                                     int slices, float scale, bool add) {
  constexpr int E = kE<TG>;
  __shared__ __attribute__((aligned(16))) float part[kSumWaves][kWave * E];
  const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
  const int64_t group = blockIdx.x / slices, per = (int64_t)s.unit * kSumWaves, begin = group * per, end = begin + per;
  if (end >= s.n) return;
  // all keys that most groups need at once: the run at the group's end, where it begins, how far it reaches
  const int key = s.keys[end], at_end = s.keys[end - 1], at_begin = begin > 0 ? s.keys[begin - 1] : -1;
  int64_t more = 1;  // groups behind this one that the run reaches
  const auto reach = [&] { return end + (more + lane) * per; };  // the first position behind the group that it may reach
  int reached = s.keys[min(reach(), (int64_t)s.n - 1)];
  if ((unsigned)key >= (unsigned)s.V || at_end != key || at_begin == key) return;  // none, or it began before
  for (;;) {
    const uint64_t ends = __ballot(reach() >= s.n || reached != key);
    if (ends) {
      more += __builtin_ctzll(ends);
      break;
    }
    more += kWave;
    reached = s.keys[min(reach(), (int64_t)s.n - 1)];
  }
  const int slice = blockIdx.x % slices, col = (slice * kWave + lane) * E;
  const int64_t one = (int64_t)slices * kWave * E, two = 2 * one;
  const float* p = partial + group * two + (slice * kWave + lane) * E;
  float sum[E] = {};
  const int64_t share = (more + kSumWaves - 1) / kSumWaves, u0 = w * share + 1, u1 = min(u0 + share, more + 1);
#pragma unroll 8
  for (int64_t u = u0; u < u1; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] += p[u * two + e];
#pragma unroll
  for (int e = 0; e < E; ++e) part[w][lane * E + e] = sum[e];
  __syncthreads();
  if (w != 0 || col >= D) return;
#pragma unroll
  for (int e = 0; e < E; ++e) sum[e] = p[one + e];
  for (int i = 0; i < kSumWaves; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] += part[i][lane * E + e];
  put_row<E, TO>(out + key * out_rs + col, sum, scale, D - col, add);
}

// ------------------------------------------------------------------ host side
int bit_length(int64_t v) {
  int n = 0;
  for (; v; v >>= 1) ++n;
  return n;
}

// Few positions beside little to fill with zeros: one launch, whose workgroups wait for all ids before they write.  us
// recorded, in one launch and sorted: 512 positions of text with 8 MiB of zeros 7.4 and 15.1, 32 MiB 13.9 and 17.2, 64 MiB 20.0 and
// 19.5, 98 MiB 25.2 and 23.6; of one token, whose rows one workgroup adds up, 18.6 and 14.2 with 8 MiB (1024: 40 and 14).
// Added to a given gradient, 512 positions here and 513 sorted: 50304 x 1024 7.6 and 14.3, 2^20 x 64 11.6 and 16.0; with more
// tokens than any vocabulary has the workgroups that find nothing cost more (2^22 x 64 30 and 16).
bool few_of(int64_t n, int64_t zeros) { return n <= kFewPositions && zeros <= (int64_t)48 << 20; }

// How a call's passes and workspace are cut.
struct Plan {
  int few_groups, few_bits;                   // few positions
  int passes, bits, keys, groups, stretch;    // sorting
  int slices, unit;
  bool stream;
  int64_t sum_groups;
  size_t list, counts, part;  // bytes of one list of n positions, of the counts, of the partial rows
  size_t bytes() const { return 4 * list + counts + part; }
};
Plan plan_of(int64_t n, int64_t V, int64_t D, int dtype) {
  Plan p{};
  const int E = 16 / hdcm_elt_size(dtype);
  p.slices = (int)((D + kWave * E - 1) / (kWave * E));
  // a round of workgroups, as far as their tokens are kSumWaves at least and kBins at most
  int64_t tokens = V * p.slices / 512;
  tokens = tokens < kSumWaves ? kSumWaves : tokens > kBins ? kBins : tokens;
  p.few_groups = (int)((V + tokens - 1) / tokens);
  p.few_bits = bit_length((V + p.few_groups - 1) / p.few_groups - 1);
  const int bits = bit_length(V);  // of the largest key, V
  p.passes = (bits + kDigitBits - 1) / kDigitBits;
  p.bits = (bits + p.passes - 1) / p.passes;
  p.keys = n <= kOneKeyGroups * kSortThreads ? 1 : 2;
  const int64_t tile = p.keys * kSortThreads, tiles = (n + tile - 1) / tile;
  p.stretch = (int)((tiles + kMaxGroups - 1) / kMaxGroups * tile);
  p.groups = (int)((n + p.stretch - 1) / p.stretch);
  // two workgroups a CU at least (32768 x 256: 32.8 us a call for 34.8); where there are many, longer units leave fewer partial rows
  const int64_t groups = (n + kAhead * kSumWaves - 1) / (kAhead * kSumWaves) * p.slices;
  p.unit = kAhead * (groups <= 512 ? 1 : groups < 8192 ? 2 : 4);
  p.stream = (n + V) * D * hdcm_elt_size(dtype) > kStreamBytes;
  p.sum_groups = (n + p.unit * kSumWaves - 1) / (p.unit * kSumWaves);
  const auto whole = [](size_t b) { return (b + 255) / 256 * 256; };
  p.list = whole((size_t)n * 4);
  p.counts = (size_t)p.groups * kBins * 4;
  p.part = whole((size_t)p.sum_groups * 2 * p.slices * kWave * E * 4);
  return p;
}

constexpr int64_t kMaxVocab = (int64_t)1 << 30, kMaxPositions = (int64_t)1 << 30, kMaxWidth = (int64_t)1 << 24;
// A launch has fewer than 2^32 threads.
bool fits(int64_t groups, int threads) { return groups < ((int64_t)1 << 32) / threads; }
int64_t pieces_of(int64_t rows, int64_t D, int dtype) { return rows * ((D * hdcm_elt_size(dtype) + 15) / 16); }

template <typename TG, typename TO>
void launch_few(const Plan& p, const Ids& ids, int n, const GradRows& g, void* out, int64_t out_rs, int64_t D, float scale, bool add,
                hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)p.few_groups * p.slices));
  HDCM_LAUNCH((embedding_few_kernel<TG, TO>), grid, dim3(kSumThreads), 0, stream, ids, n, g, (TO*)out, out_rs, (int)D, p.slices,
              p.few_bits, scale, add);
}

template <typename TG, typename TO>
void launch_sums(const Plan& p, const Sorted& s, const GradRows& g, void* out, int64_t out_rs, float* part, int64_t D, float scale,
                 bool add, hipStream_t stream) {
  const dim3 grid((unsigned)(p.sum_groups * p.slices));
  const auto sums = p.stream ? embedding_sum_kernel<true, TG, TO> : embedding_sum_kernel<false, TG, TO>;
  HDCM_LAUNCH(sums, grid, dim3(kSumThreads), 0, stream, s, g, (TO*)out, out_rs, part, (int)D, p.slices, scale, add);
  if (p.sum_groups > 1)
    HDCM_LAUNCH((embedding_join_kernel<TG, TO>), grid, dim3(kSumThreads), 0, stream, s, (TO*)out, out_rs, (const float*)part, (int)D,
                p.slices, scale, add);
}

// Zeros by a launch of their own: there is nothing to sort, or rows lie apart
void launch_zeros(void* dw, int64_t rs, int64_t V, int64_t D, int dtype, hipStream_t s) {
  const int E = 16 / hdcm_elt_size(dtype);
  const dim3 grid((unsigned)((V * ((D + E - 1) / E) + 255) / 256));
  if (dtype == HDCM_F32) HDCM_LAUNCH(zero_rows_kernel<float>, grid, dim3(256), 0, s, (float*)dw, rs, V, (int)D);
  else HDCM_LAUNCH(zero_rows_kernel<bf16_t>, grid, dim3(256), 0, s, (bf16_t*)dw, rs, V, (int)D);
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
  HDCM_CHECK_ARG(fits(pieces_of(rows, D, dtype) / (2 * kLookThreads) + 1, kLookThreads), HDCM_EUNSUPPORTED);
  hipStream_t s = (hipStream_t)stream;
  const auto go = [&](auto launch) { launch(ids, w, w_row_stride, out, out_row_stride, rows, V, D, scale, s); };
  if (dtype == HDCM_F32) id_bytes == 8 ? go(launch_lookup<float, int64_t>) : go(launch_lookup<float, int32_t>);
  else id_bytes == 8 ? go(launch_lookup<bf16_t, int64_t>) : go(launch_lookup<bf16_t, int32_t>);
  return hdcm_launch_status();
}

extern "C" size_t hdcm_embedding_grad_workspace_bytes(int64_t B, int64_t L, int64_t V, int64_t D, int dtype) {
  if (B <= 0 || L <= 0 || V <= 0 || D <= 0 || L > kMaxPositions / B || V > kMaxVocab || D > kMaxWidth) return 0;
  return few_of(B * L, V * D * 4) ? 0 : plan_of(B * L, V, D, dtype).bytes();
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
  const bool few = !none && few_of(B * L, accumulate ? 0 : V * D * hdcm_elt_size(dw_dtype));
  if (!none) p = plan_of(B * L, V, D, dtype);
  const bool apart = dw_row_stride != D && V > 1;  // rows of dw are not adjacent
  const int64_t zeros = accumulate || apart ? 0 : V * D * hdcm_elt_size(dw_dtype);
  HDCM_CHECK_ARG(none || (few ? fits((int64_t)p.few_groups * p.slices, kSumThreads)
                              : fits(p.sum_groups * p.slices, kSumThreads) && fits(p.groups + zeros / kFillBytes + 1, kSortThreads)),
                 HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(few || accumulate || !(none || apart) || fits(pieces_of(V, D, dw_dtype) / 256 + 1, 256), HDCM_EUNSUPPORTED);
  if (!none && !few) {
    HDCM_CHECK_ARG(ws && ws_bytes >= p.bytes(), HDCM_EWORKSPACE);
    HDCM_CHECK_ARG(hdcm_aligned16(ws), HDCM_EALIGN);
  }
  if (none) {
    launch_zeros(dw, dw_row_stride, V, D, dw_dtype, s);
    return hdcm_launch_status();
  }
  const int n = (int)(B * L);
  const Ids keys_of{ids, id_bytes, (int)V, (int)padding_idx};
  const GradRows g{dy, dy_batch_stride, dy_row_stride, (uint32_t)(B > 1 ? L : 0)};
  if (few) {
    const auto go = [&](auto launch) { launch(p, keys_of, n, g, dw, dw_row_stride, D, scale, accumulate != 0, s); };
    if (dtype == HDCM_F32) dw_dtype == HDCM_F32 ? go(launch_few<float, float>) : go(launch_few<float, bf16_t>);
    else dw_dtype == HDCM_F32 ? go(launch_few<bf16_t, float>) : go(launch_few<bf16_t, bf16_t>);
    return hdcm_launch_status();
  }
  char* at = (char*)ws;
  int* lists[4];
  for (int i = 0; i < 4; ++i, at += p.list) lists[i] = (int*)at;
  int* counts = (int*)at;
  float* part = (float*)(at + p.counts);
  // the zeros go with the sorting launches: with all scatters alike
  if (!accumulate && apart) launch_zeros(dw, dw_row_stride, V, D, dw_dtype, s);
  const auto fill_of = [&](int k, int n) {
    const auto upto = [&](int i) { return i == n ? zeros : zeros / n * i / 16 * 16; };
    return Fill{(char*)dw, upto(k), upto(k + 1)};
  };
  const auto grid = [&](int groups, const Fill& f) { return dim3((unsigned)(groups + (f.end - f.begin + kFillBytes - 1) / kFillBytes)); };
  SortIn in{keys_of, nullptr, nullptr};
  if (n <= kOneGroup) {
    const Fill f = fill_of(0, 1);
    HDCM_LAUNCH(sort_one_kernel, grid(1, f), dim3(kSortThreads), 0, s, keys_of, n, p.passes, p.bits, lists[0], lists[1], f);
    in.keys = lists[0], in.pos = lists[1];
  } else {
    const auto count = p.keys == 1 ? sort_count_kernel<1> : sort_count_kernel<2>;
    const auto scatter = p.keys == 1 ? sort_scatter_kernel<1> : sort_scatter_kernel<2>;
    for (int k = 0; k < p.passes; ++k) {
      int *keys = lists[2 * (k & 1)], *pos = lists[2 * (k & 1) + 1];
      const Pass pass{n, p.stretch, p.groups, k * p.bits, p.bits};
      const Fill f = fill_of(k, p.passes);
      HDCM_LAUNCH(count, dim3(p.groups), dim3(kSortThreads), 0, s, in, pass, counts);
      HDCM_LAUNCH(scatter, grid(p.groups, f), dim3(kSortThreads), 0, s, in, pass, (const int*)counts, keys, pos, f);
      in.keys = keys, in.pos = pos;
    }
  }
  const Sorted sorted{in.keys, in.pos, n, (int)V, p.unit};
  const auto go = [&](auto launch) { launch(p, sorted, g, dw, dw_row_stride, part, D, scale, accumulate != 0, s); };
  if (dtype == HDCM_F32) dw_dtype == HDCM_F32 ? go(launch_sums<float, float>) : go(launch_sums<float, bf16_t>);
  else dw_dtype == HDCM_F32 ? go(launch_sums<bf16_t, float>) : go(launch_sums<bf16_t, bf16_t>);
  return hdcm_launch_status();
}
