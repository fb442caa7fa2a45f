// The global norm of many tensors and their scaling by it: what a training step does between its backward and
// its optimizer (torch.nn.utils.clip_grad_norm_; the reference trains without).
//   norm:   sqrt(sum x^2) over all elements of all tensors, or max |x|
//   scale:  x *= min(1, max_norm / (norm + 1e-6))
// A list of tensors goes to one launch as a table in the kernel's arguments; every workgroup takes one stretch
// of one tensor.  Squares are added in 64 bits: exact for bf16 and fp32 inputs, no square overflows or vanishes,
// and the sum's rounding is that of the result.  Every sum has a fixed order.
#include "hdcm_common.h"

using namespace hdcm;

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kAhead = 8;         // 16-byte loads of a thread in flight
constexpr int kSomeTensors = 32, kManyTensors = 320;  // of a launch: a table of many still fits 4 KB of arguments
constexpr uint32_t kIsF32 = 1u << 31;
constexpr int64_t kMaxCount = (int64_t)1 << 30;  // elements of an entry; a longer tensor has several

// Entry i: `size` elements (and, in the highest bit, their type) at the address hi[i] : lo[i].  Arrays of words, for the
// lanes of a wave to read.
template <int N> struct Table {
  static constexpr int kRows = (N + kWave - 1) / kWave;
  uint32_t lo[N], hi[N], size[N];  // entries behind the last have size 0
  uint32_t before[kRows];          // workgroups of the entries before every kWave-th; all bits behind the last
};

// A workgroup's stretch: `count` elements from `data` on.
struct Stretch {
  void* data;
  uint32_t count;
  bool f32;
};
// log2 of the elements in a stretch of 2^bits bytes
__host__ __device__ __forceinline__ int stretch_shift(int bits, bool f32) { return f32 ? bits - 2 : bits - 1; }

// Every wave looks its workgroup's entry up: the workgroups of the kWave entries among which it is are added up over the
// lanes.
template <int N> __device__ __forceinline__ Stretch stretch_of(const Table<N>& t, int bits, uint32_t group) {
  const int lane = threadIdx.x % kWave;
  int row = 0;
#pragma unroll
  for (int r = 1; r < Table<N>::kRows; ++r) row = group >= t.before[r] ? r : row;
  const int i = row * kWave + lane;
  const uint32_t size = i < N ? t.size[i] : 0;
  const int shift = stretch_shift(bits, size & kIsF32);
  const uint32_t groups = ((size & ~kIsF32) + (1u << shift) - 1) >> shift;
  uint32_t up_to = groups;  // of the lanes up to this one
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint32_t up = __shfl_up(up_to, o, kWave);
    up_to += lane >= o ? up : 0;
  }
  const uint64_t behind = __ballot(group - t.before[row] < up_to);  // its first lane has the entry
  Stretch s{nullptr, 0, false};
  if (!behind) return s;
  const int at = __builtin_ctzll(behind);
  const uint32_t first = __builtin_amdgcn_readlane(up_to - groups, at), whole = __builtin_amdgcn_readlane(size, at);
  s.f32 = whole & kIsF32;
  const uint32_t begin = (group - t.before[row] - first) << stretch_shift(bits, s.f32);
  s.data = (char*)((uint64_t)t.hi[row * kWave + at] << 32 | t.lo[row * kWave + at]) + ((uint64_t)begin << (s.f32 ? 2 : 1));
  s.count = min((whole & ~kIsF32) - begin, 1u << stretch_shift(bits, s.f32));
  return s;
}

template <typename T> struct Loose;  // 16 bytes at the type's own alignment: tensors may be slices of a buffer
template <> struct Loose<bf16_t> {
  typedef u32x4_t type __attribute__((aligned(2)));
};
template <> struct Loose<float> {
  typedef u32x4_t type __attribute__((aligned(4)));
};
// STREAM: past the caches
template <typename T, bool STREAM> __device__ __forceinline__ u32x4_t load_piece(const T* p) {
  const auto q = reinterpret_cast<const typename Loose<T>::type*>(p);
  return STREAM ? __builtin_nontemporal_load(q) : *q;
}
template <typename T, bool STREAM> __device__ __forceinline__ void store_piece(T* p, u32x4_t v) {
  const auto q = reinterpret_cast<typename Loose<T>::type*>(p);
  if constexpr (STREAM) __builtin_nontemporal_store(v, q);
  else *q = v;
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

// The norm's accumulator: a sum of squares, or the largest magnitude by its bits (those of a NaN are above all).
template <bool MAX> struct Acc;
template <> struct Acc<false> {
  double v = 0.0;
  __device__ __forceinline__ void take(float x) { v = fma((double)x, (double)x, v); }
  __device__ __forceinline__ void join(double o) { v += o; }
  __device__ __forceinline__ double part() const { return v; }
  __device__ __forceinline__ void join_part(double p) { v += p; }
  __device__ __forceinline__ float norm() const { return (float)sqrt(v); }
};
template <> struct Acc<true> {
  uint32_t v = 0;
  __device__ __forceinline__ void take(float x) { v = max(v, __float_as_uint(x) & 0x7fffffffu); }
  __device__ __forceinline__ void join(uint32_t o) { v = max(v, o); }
  __device__ __forceinline__ double part() const { return __longlong_as_double((int64_t)v); }
  __device__ __forceinline__ void join_part(double p) { v = max(v, (uint32_t)__double_as_longlong(p)); }
  __device__ __forceinline__ float norm() const { return __uint_as_float(v); }
};
// The workgroup's threads as one, in every thread
template <int WAVES, typename A> __device__ __forceinline__ void join_threads(A& a) {
  __shared__ decltype(a.v) each[WAVES];
#pragma unroll
  for (int o = kWave / 2; o >= 1; o >>= 1) a.join(__shfl_xor(a.v, o, kWave));
  if (threadIdx.x % kWave == 0) each[threadIdx.x / kWave] = a.v;
  __syncthreads();
  a.v = each[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) a.join(each[i]);
}

template <typename T, bool STREAM, typename A> __device__ __forceinline__ void norm_of(const Stretch& s, A& a) {
  constexpr uint32_t E = 16 / sizeof(T);
  const T* p = static_cast<const T*>(s.data);
  const uint32_t pieces = s.count / E;
  for (uint32_t i0 = 0; i0 < pieces; i0 += kAhead * kThreads) {
    u32x4_t x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint32_t i = i0 + u * kThreads + threadIdx.x;
      x[u] = u32x4_t{0, 0, 0, 0};
      if (i < pieces) x[u] = load_piece<T, STREAM>(p + i * E);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      float v[E];
      values<T>(x[u], v);
#pragma unroll
      for (uint32_t e = 0; e < E; ++e) a.take(v[e]);
    }
  }
  const uint32_t i = pieces * E + threadIdx.x;
  if (i < s.count) a.take(to_f<T>(p[i]));
}

// Bound by its one read: 2.06 GB of bf16 303 us (6.8 TB/s; 342 through the caches), 0.38 GB 58.  The conversions to 64 bits and
// the multiply-adds fit beside it (128 KB a workgroup: the same).
template <bool MAX, bool STREAM, int N>
__global__ __launch_bounds__(kThreads) void norm_parts_kernel(Table<N> t, int bits, double* parts) {
  const Stretch s = stretch_of(t, bits, blockIdx.x);
  Acc<MAX> a;
  if (s.f32) norm_of<float, STREAM>(s, a);
  else norm_of<bf16_t, STREAM>(s, a);
  join_threads<kWaves>(a);
  if (threadIdx.x == 0) parts[blockIdx.x] = a.part();
}

// The norm from the workgroups' parts
template <bool MAX, int THREADS> __device__ __forceinline__ float join_parts(const double* parts, int64_t n) {
  constexpr int U = 8;
  Acc<MAX> a;
  for (int64_t i0 = 0; i0 < n; i0 += U * THREADS) {
    double v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * THREADS + (int)threadIdx.x;
      v[u] = i < n ? parts[i] : 0.0;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) a.join_part(v[u]);
  }
  join_threads<THREADS / kWave>(a);
  return a.norm();
}

// 31000 parts 9 us, 5800 4.7: a chain of their arrival and two reductions.
constexpr int kJoinThreads = 1024;
template <bool MAX> __global__ __launch_bounds__(kJoinThreads) void norm_join_kernel(const double* parts, int64_t n, float* norm) {
  const float v = join_parts<MAX, kJoinThreads>(parts, n);
  if (threadIdx.x == 0) *norm = v;
}

template <typename T, bool STREAM> __device__ __forceinline__ void scale_of(const Stretch& s, float factor) {
  constexpr uint32_t E = 16 / sizeof(T);
  T* p = static_cast<T*>(s.data);
  const uint32_t pieces = s.count / E;
  for (uint32_t i0 = 0; i0 < pieces; i0 += kAhead * kThreads) {
    u32x4_t x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint32_t i = i0 + u * kThreads + threadIdx.x;
      if (i < pieces) x[u] = load_piece<T, STREAM>(p + i * E);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint32_t i = i0 + u * kThreads + threadIdx.x;
      float v[E];
      values<T>(x[u], v);
#pragma unroll
      for (uint32_t e = 0; e < E; ++e) v[e] *= factor;
      const uint4 r = pack16<T>(v);
      if (i < pieces) store_piece<T, STREAM>(p + i * E, u32x4_t{r.x, r.y, r.z, r.w});
    }
  }
  const uint32_t i = pieces * E + threadIdx.x;
  if (i < s.count) p[i] = from_f<T>(to_f<T>(p[i]) * factor);
}

// Where the norm comes from: given, or joined from its parts by every workgroup (the first writes it).
enum From { kGiven, kParts2, kPartsMax };

// Nothing is read or written where the factor is 1 (4.4 us for 5800 workgroups; 7.0 with the table's entry looked up
// first).  0.76 GB of fp32 285 us: 5.3 TB/s of reads and writes (315 through the caches); 4.2 MB 4.3.
template <int FROM, bool STREAM, int N>
__global__ __launch_bounds__(kThreads) void scale_kernel(Table<N> t, int bits, float* norm, const double* parts, int n_parts,
                                                         float max_norm) {
  float total;
  if constexpr (FROM == kGiven) {
    total = *norm;
  } else {
    total = join_parts<FROM == kPartsMax, kThreads>(parts, n_parts);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
  }
  const float ratio = max_norm / (total + 1e-6f), factor = ratio > 1.f ? 1.f : ratio;  // a NaN stays one
  if (factor == 1.f) return;
  const Stretch s = stretch_of(t, bits, blockIdx.x);
  if (s.f32) scale_of<float, STREAM>(s, factor);
  else scale_of<bf16_t, STREAM>(s, factor);
}

// ------------------------------------------------------------------ host side
int check_tensors(const hdcm_tensor* t, int64_t n) {
  HDCM_CHECK_ARG(n >= 0 && (t || n == 0), HDCM_EINVAL);
  for (int64_t i = 0; i < n; ++i) {
    HDCM_CHECK_ARG(t[i].dtype == HDCM_F32 || t[i].dtype == HDCM_BF16, HDCM_EUNSUPPORTED);
    HDCM_CHECK_ARG(t[i].count >= 0 && (t[i].data || t[i].count == 0), HDCM_EINVAL);
    HDCM_CHECK_ARG((uintptr_t)t[i].data % hdcm_elt_size(t[i].dtype) == 0, HDCM_EALIGN);
  }
  return HDCM_OK;
}

// Small lists are cut finer, into more workgroups: 4.2 MB scaled in 4.3 us instead of 7.2, its norm's parts 3.8 for 4.4.
constexpr int64_t kSmallBytes = (int64_t)16 << 20;

// What a list comes to.  Elements that are read (and written) once go past the caches where they are more than the
// caches hold of them until they are used again.
struct Size {
  int64_t entries = 0, groups = 0, bytes = 0;
  int bits = 0;  // a workgroup takes 2^bits bytes of a tensor
  bool stream() const { return bytes > kStreamBytes; }
  static constexpr int64_t kStreamBytes = (int64_t)128 << 20;
};
Size size_of(const hdcm_tensor* t, int64_t n) {
  Size s;
  for (int64_t i = 0; i < n; ++i) s.bytes += t[i].count * hdcm_elt_size(t[i].dtype);
  s.bits = s.bytes <= kSmallBytes ? 14 : 16;
  for (int64_t i = 0; i < n; ++i) {
    const int shift = stretch_shift(s.bits, t[i].dtype == HDCM_F32);  // entries hold whole stretches
    s.entries += (t[i].count + kMaxCount - 1) / kMaxCount;
    s.groups += (t[i].count + (1 << shift) - 1) >> shift;
  }
  return s;
}

// Calls launch(table, workgroups) for the tensors in their order, as many to a table as it holds.
template <int N, typename F> void each_table(const hdcm_tensor* t, int64_t n, int bits, F launch) {
  Table<N> table;
  int held = 0;
  uint32_t groups = 0;
  const auto flush = [&] {
    for (int i = held; i < N; ++i) table.lo[i] = table.hi[i] = table.size[i] = 0;
    for (int r = (held + kWave - 1) / kWave; r < Table<N>::kRows; ++r) table.before[r] = ~0u;
    if (groups) launch(table, groups);
    held = 0, groups = 0;
  };
  for (int64_t i = 0; i < n; ++i) {
    const bool f32 = t[i].dtype == HDCM_F32;
    uint64_t data = (uint64_t)(uintptr_t)t[i].data;
    for (int64_t left = t[i].count; left > 0; left -= kMaxCount, data += (uint64_t)kMaxCount << (f32 ? 2 : 1)) {
      const uint32_t count = (uint32_t)(left < kMaxCount ? left : kMaxCount);
      if (held % kWave == 0) table.before[held / kWave] = groups;
      table.lo[held] = (uint32_t)data, table.hi[held] = (uint32_t)(data >> 32);
      table.size[held] = count | (f32 ? kIsF32 : 0);
      groups += (count + (1u << stretch_shift(bits, f32)) - 1) >> stretch_shift(bits, f32);
      if (++held == N || groups >= 1u << 23) flush();  // (a launch has fewer than 2^32 threads)
    }
  }
  flush();
}
// The table for a list: a short one costs less to hand over.
template <typename F> void each_table(const hdcm_tensor* t, int64_t n, const Size& size, F launch) {
  if (size.entries <= kSomeTensors) each_table<kSomeTensors>(t, n, size.bits, launch);
  else each_table<kManyTensors>(t, n, size.bits, launch);
}

template <bool MAX> void launch_parts(const hdcm_tensor* t, int64_t n, const Size& size, double* parts, hipStream_t s) {
  each_table(t, n, size, [&](const auto& table, uint32_t groups) {
    constexpr int N = sizeof(table.lo) / sizeof(table.lo[0]);
    const auto kernel = size.stream() ? norm_parts_kernel<MAX, true, N> : norm_parts_kernel<MAX, false, N>;
    HDCM_LAUNCH(kernel, dim3(groups), dim3(kThreads), 0, s, table, size.bits, parts);
    parts += groups;
  });
}
template <bool MAX> void launch_norm(const hdcm_tensor* t, int64_t n, const Size& size, float* norm, double* parts, hipStream_t s) {
  launch_parts<MAX>(t, n, size, parts, s);
  HDCM_LAUNCH(norm_join_kernel<MAX>, dim3(1), dim3(kJoinThreads), 0, s, (const double*)parts, size.groups, norm);
}
template <int FROM>
void launch_scale(const hdcm_tensor* t, int64_t n, const Size& size, float* norm, const double* parts, float max_norm, hipStream_t s) {
  each_table(t, n, size, [&](const auto& table, uint32_t groups) {
    constexpr int N = sizeof(table.lo) / sizeof(table.lo[0]);
    const auto kernel = size.stream() ? scale_kernel<FROM, true, N> : scale_kernel<FROM, false, N>;
    HDCM_LAUNCH(kernel, dim3(groups), dim3(kThreads), 0, s, table, size.bits, norm, parts, (int)size.groups, max_norm);
  });
}

int check_norm(const hdcm_tensor* t, int64_t n, int norm, const float* out, const void* ws, size_t ws_bytes, Size& size) {
  const int st = check_tensors(t, n);
  if (st) return st;
  HDCM_CHECK_ARG(norm == HDCM_NORM_2 || norm == HDCM_NORM_MAX, HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(out, HDCM_EINVAL);
  size = size_of(t, n);
  const size_t need = (size_t)size.groups * sizeof(double);
  HDCM_CHECK_ARG(need == 0 || (ws && ws_bytes >= need), HDCM_EWORKSPACE);
  HDCM_CHECK_ARG(need == 0 || ((uintptr_t)ws & 7u) == 0, HDCM_EALIGN);
  return HDCM_OK;
}

// Parts that every workgroup of the scaling joins by itself, a launch less; more are joined by a launch between.
constexpr int64_t kOwnParts = 1024;

}  // namespace

extern "C" size_t hdcm_grad_norm_workspace_bytes(const hdcm_tensor* tensors, int64_t n) {
  return check_tensors(tensors, n) == HDCM_OK ? (size_t)size_of(tensors, n).groups * sizeof(double) : 0;
}

extern "C" int hdcm_grad_norm(const hdcm_tensor* tensors, int64_t n, int norm, float* out, void* ws, size_t ws_bytes, void* stream) {
  Size size;
  const int st = check_norm(tensors, n, norm, out, ws, ws_bytes, size);
  if (st) return st;
  if (norm == HDCM_NORM_2) launch_norm<false>(tensors, n, size, out, (double*)ws, (hipStream_t)stream);
  else launch_norm<true>(tensors, n, size, out, (double*)ws, (hipStream_t)stream);
  return hdcm_launch_status();
}

extern "C" int hdcm_grad_scale(const hdcm_tensor* tensors, int64_t n, const float* norm, float max_norm, void* stream) {
  const int st = check_tensors(tensors, n);
  if (st) return st;
  HDCM_CHECK_ARG(norm && max_norm >= 0.f, HDCM_EINVAL);
  const Size size = size_of(tensors, n);
  if (size.groups == 0) return HDCM_OK;
  launch_scale<kGiven>(tensors, n, size, const_cast<float*>(norm), nullptr, max_norm, (hipStream_t)stream);
  return hdcm_launch_status();
}

extern "C" int hdcm_clip_grad_norm(const hdcm_tensor* tensors, int64_t n, int norm, float max_norm, float* out, void* ws,
                                   size_t ws_bytes, void* stream) {
  Size size;
  const int st = check_norm(tensors, n, norm, out, ws, ws_bytes, size);
  if (st) return st;
  HDCM_CHECK_ARG(max_norm >= 0.f, HDCM_EINVAL);
  hipStream_t s = (hipStream_t)stream;
  double* parts = (double*)ws;
  const bool max = norm == HDCM_NORM_MAX;
  if (size.groups == 0 || size.groups > kOwnParts) {
    max ? launch_norm<true>(tensors, n, size, out, parts, s) : launch_norm<false>(tensors, n, size, out, parts, s);
    launch_scale<kGiven>(tensors, n, size, out, nullptr, max_norm, s);
  } else if (max) {
    launch_parts<true>(tensors, n, size, parts, s);
    launch_scale<kPartsMax>(tensors, n, size, out, parts, max_norm, s);
  } else {
    launch_parts<false>(tensors, n, size, parts, s);
    launch_scale<kParts2>(tensors, n, size, out, parts, max_norm, s);
  }
  return hdcm_launch_status();
}
