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
constexpr int kAhead = 8;                   // 16-byte loads of a thread in flight
constexpr int64_t kStretchBytes = 65536;    // of a tensor, for one workgroup
constexpr int kMaxTensors = 224;            // of a launch: its table stays inside 4 KB of arguments
constexpr uint32_t kIsF32 = 1u << 31;
constexpr int64_t kMaxCount = (int64_t)1 << 30;  // elements of an entry; a longer tensor has several

// Entry i: `count` elements at `data` for the workgroups [first[i], first[i + 1]).
struct Table {
  void* data[kMaxTensors];
  uint32_t count[kMaxTensors];  // and the type, in the highest bit
  uint32_t first[kMaxTensors];
  int n;
};

// A workgroup's stretch: elements [begin, end) of the tensor at data.
struct Stretch {
  void* data;
  uint32_t begin, end;
  bool f32;
};
__device__ __forceinline__ Stretch stretch_of(const Table& t, uint32_t group) {
  int lo = 0, hi = t.n;  // the last entry that begins at or before the group
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= group) lo = mid;
    else hi = mid;
  }
  Stretch s;
  s.data = t.data[lo];
  s.f32 = t.count[lo] & kIsF32;
  const uint32_t per = (uint32_t)(kStretchBytes / (s.f32 ? 4 : 2)), count = t.count[lo] & ~kIsF32;
  s.begin = (group - t.first[lo]) * per;
  s.end = min(s.begin + per, count);
  return s;
}

template <typename T> struct Loose;  // 16 bytes at the type's own alignment: tensors may be slices of a buffer
template <> struct Loose<bf16_t> {
  typedef u32x4_t type __attribute__((aligned(2)));
};
template <> struct Loose<float> {
  typedef u32x4_t type __attribute__((aligned(4)));
};
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
};
template <> struct Acc<true> {
  uint32_t v = 0;
  __device__ __forceinline__ void take(float x) { v = max(v, __float_as_uint(x) & 0x7fffffffu); }
  __device__ __forceinline__ void join(uint32_t o) { v = max(v, o); }
};
template <typename A> __device__ __forceinline__ void join_lanes(A& a) {
#pragma unroll
  for (int o = kWave / 2; o >= 1; o >>= 1) a.join(__shfl_xor(a.v, o, kWave));
}
// The workgroup's threads as one, in thread 0
template <int WAVES, typename A> __device__ __forceinline__ void join_threads(A& a) {
  __shared__ decltype(a.v) each[WAVES];
  join_lanes(a);
  if (threadIdx.x % kWave == 0) each[threadIdx.x / kWave] = a.v;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int i = 1; i < WAVES; ++i) a.join(each[i]);
}

template <typename T, typename A> __device__ __forceinline__ void norm_of(const Stretch& s, A& a) {
  constexpr int E = 16 / sizeof(T);
  const T* p = static_cast<const T*>(s.data) + s.begin;
  const uint32_t n = s.end - s.begin, pieces = n / E;
  for (uint32_t i0 = 0; i0 < pieces; i0 += kAhead * kThreads) {
    u32x4_t x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint32_t i = i0 + u * kThreads + threadIdx.x;
      x[u] = u32x4_t{0, 0, 0, 0};
      if (i < pieces) x[u] = *reinterpret_cast<const typename Loose<T>::type*>(p + (int64_t)i * E);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      float v[E];
      values<T>(x[u], v);
#pragma unroll
      for (int e = 0; e < E; ++e) a.take(v[e]);
    }
  }
  const uint32_t i = pieces * E + threadIdx.x;
  if (i < n) a.take(to_f<T>(p[i]));
}

template <bool MAX>
__global__ __launch_bounds__(kThreads) void norm_parts_kernel(Table t, double* parts) {
  const Stretch s = stretch_of(t, blockIdx.x);
  Acc<MAX> a;
  if (s.f32) norm_of<float>(s, a);
  else norm_of<bf16_t>(s, a);
  join_threads<kWaves>(a);
  if (threadIdx.x == 0) parts[blockIdx.x] = MAX ? __longlong_as_double((int64_t)a.v) : (double)a.v;
}

constexpr int kJoinThreads = 1024;
template <bool MAX>
__global__ __launch_bounds__(kJoinThreads) void norm_join_kernel(const double* parts, int64_t n, float* norm) {
  Acc<MAX> a;
  for (int64_t i = threadIdx.x; i < n; i += kJoinThreads) {
    if constexpr (MAX) a.join((uint32_t)__double_as_longlong(parts[i]));
    else a.join(parts[i]);
  }
  join_threads<kJoinThreads / kWave>(a);
  if (threadIdx.x == 0) {
    if constexpr (MAX) *norm = __uint_as_float(a.v);
    else *norm = (float)sqrt(a.v);
  }
}

template <typename T> __device__ __forceinline__ void scale_of(const Stretch& s, float factor) {
  constexpr int E = 16 / sizeof(T);
  T* p = static_cast<T*>(s.data) + s.begin;
  const uint32_t n = s.end - s.begin, pieces = n / E;
  for (uint32_t i0 = 0; i0 < pieces; i0 += kAhead * kThreads) {
    u32x4_t x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint32_t i = i0 + u * kThreads + threadIdx.x;
      if (i < pieces) x[u] = *reinterpret_cast<const typename Loose<T>::type*>(p + (int64_t)i * E);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint32_t i = i0 + u * kThreads + threadIdx.x;
      float v[E];
      values<T>(x[u], v);
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] *= factor;
      const uint4 r = pack16<T>(v);
      if (i < pieces) *reinterpret_cast<typename Loose<T>::type*>(p + (int64_t)i * E) = u32x4_t{r.x, r.y, r.z, r.w};
    }
  }
  const uint32_t i = pieces * E + threadIdx.x;
  if (i < n) p[i] = from_f<T>(to_f<T>(p[i]) * factor);
}

// Nothing is read or written where the factor is 1.
__global__ __launch_bounds__(kThreads) void scale_kernel(Table t, const float* norm, float max_norm) {
  const float ratio = max_norm / (*norm + 1e-6f), factor = ratio > 1.f ? 1.f : ratio;  // a NaN stays one
  if (factor == 1.f) return;
  const Stretch s = stretch_of(t, blockIdx.x);
  if (s.f32) scale_of<float>(s, factor);
  else scale_of<bf16_t>(s, factor);
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
uint32_t groups_of(int64_t count, int dtype) {
  return (uint32_t)((count * hdcm_elt_size(dtype) + kStretchBytes - 1) / kStretchBytes);
}

// Calls launch(table, workgroups) for the tensors in their order, as many to a table as it holds.
template <typename F> void each_table(const hdcm_tensor* t, int64_t n, F launch) {
  Table table;
  table.n = 0;
  uint32_t groups = 0;
  const auto flush = [&] {
    if (table.n) launch(table, groups);
    table.n = 0, groups = 0;
  };
  for (int64_t i = 0; i < n; ++i) {
    char* data = (char*)t[i].data;
    const int e = hdcm_elt_size(t[i].dtype);
    for (int64_t left = t[i].count; left > 0; left -= kMaxCount, data += kMaxCount * e) {
      const int64_t count = left < kMaxCount ? left : kMaxCount;
      table.data[table.n] = data;
      table.count[table.n] = (uint32_t)count | (t[i].dtype == HDCM_F32 ? kIsF32 : 0);
      table.first[table.n] = groups;
      groups += groups_of(count, t[i].dtype);
      if (++table.n == kMaxTensors || groups >= 1u << 24) flush();
    }
  }
  flush();
}

int64_t parts_of(const hdcm_tensor* t, int64_t n) {
  int64_t parts = 0;
  each_table(t, n, [&](const Table&, uint32_t groups) { parts += groups; });
  return parts;
}

template <bool MAX> void launch_norm(const hdcm_tensor* t, int64_t n, float* norm, double* parts, hipStream_t s) {
  int64_t done = 0;
  each_table(t, n, [&](const Table& table, uint32_t groups) {
    HDCM_LAUNCH(norm_parts_kernel<MAX>, dim3(groups), dim3(kThreads), 0, s, table, parts + done);
    done += groups;
  });
  HDCM_LAUNCH(norm_join_kernel<MAX>, dim3(1), dim3(kJoinThreads), 0, s, (const double*)parts, done, norm);
}

}  // namespace

extern "C" size_t hdcm_grad_norm_workspace_bytes(const hdcm_tensor* tensors, int64_t n) {
  return check_tensors(tensors, n) == HDCM_OK ? (size_t)parts_of(tensors, n) * sizeof(double) : 0;
}

extern "C" int hdcm_grad_norm(const hdcm_tensor* tensors, int64_t n, int norm, float* out, void* ws, size_t ws_bytes, void* stream) {
  const int st = check_tensors(tensors, n);
  if (st) return st;
  HDCM_CHECK_ARG(norm == HDCM_NORM_2 || norm == HDCM_NORM_MAX, HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(out, HDCM_EINVAL);
  const size_t need = (size_t)parts_of(tensors, n) * sizeof(double);
  HDCM_CHECK_ARG(need == 0 || (ws && ws_bytes >= need), HDCM_EWORKSPACE);
  HDCM_CHECK_ARG(need == 0 || ((uintptr_t)ws & 7u) == 0, HDCM_EALIGN);
  if (norm == HDCM_NORM_2) launch_norm<false>(tensors, n, out, (double*)ws, (hipStream_t)stream);
  else launch_norm<true>(tensors, n, out, (double*)ws, (hipStream_t)stream);
  return hdcm_launch_status();
}

extern "C" int hdcm_grad_scale(const hdcm_tensor* tensors, int64_t n, const float* norm, float max_norm, void* stream) {
  const int st = check_tensors(tensors, n);
  if (st) return st;
  HDCM_CHECK_ARG(norm && max_norm >= 0.f, HDCM_EINVAL);
  if (parts_of(tensors, n) == 0) return HDCM_OK;
  each_table(tensors, n, [&](const Table& table, uint32_t groups) {
    HDCM_LAUNCH(scale_kernel, dim3(groups), dim3(kThreads), 0, (hipStream_t)stream, table, norm, max_norm);
  });
  return hdcm_launch_status();
}
