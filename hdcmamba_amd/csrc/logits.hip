// From logits to the next tokens of a batch of sequences (no counterpart in the reference, whose
// generate samples on the host side of torch, train.py:139-151):
//   process:  z = seen ? (l > 0 ? l / r : l r) : l;  count > 0: z -= f count, z -= p;  z += bias;
//             out = allowed ? z : -inf
//   select:   t = z / T, token = the lowest index of the largest t + noise, and
//             logprob = t[token] - log sum exp t, in one read and without writing z
//   history:  seen and count per (sequence, token): an int16 whose sign bit marks the prompt's
//             tokens and whose low 15 bits count the token in the output (at most 32767)
// Every step of z is one fp32 operation with its own rounding (no contraction), so process and
// select agree bit for bit with the formula evaluated operation by operation.
#include "hdcm_common.h"

using namespace hdcm;

namespace {

constexpr float kInf = __builtin_inff();
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// Eight consecutive values of a row as they lie in memory, at the type's own alignment (rows of an odd
// vocabulary start anywhere).
template <typename T> struct Run {
  u32x4_t v[sizeof(T) / 2];
};
template <typename T> __device__ __forceinline__ Run<T> load_run(const T* p) {
  typedef u32x4_t run2_t __attribute__((aligned(2)));
  typedef u32x4_t run4_t __attribute__((aligned(4)));
  Run<T> r;
  if constexpr (sizeof(T) == 2) {
    r.v[0] = *reinterpret_cast<const run2_t*>(p);
  } else {
    r.v[0] = *reinterpret_cast<const run4_t*>(p);
    r.v[1] = *reinterpret_cast<const run4_t*>(p + 4);
  }
  return r;
}
// The end of a row: n < 8 values, zero bits behind them.
template <typename T> __device__ __forceinline__ Run<T> load_end(const T* p, int n) {
  Run<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = u32x4_t{0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) {
      if constexpr (sizeof(T) == 2) r.v[0][e / 2] |= (uint32_t)(uint16_t)p[e] << (16 * (e & 1));
      else r.v[e / 4][e & 3] = __float_as_uint(p[e]);
    }
  return r;
}
__device__ __forceinline__ void values(const Run<bf16_t>& r, float* z) {
#pragma unroll
  for (int e = 0; e < 4; ++e) z[2 * e] = __uint_as_float(r.v[0][e] << 16), z[2 * e + 1] = __uint_as_float(r.v[0][e] & 0xffff0000u);
}
__device__ __forceinline__ void values(const Run<float>& r, float* z) {
#pragma unroll
  for (int e = 0; e < 4; ++e) z[e] = __uint_as_float(r.v[0][e]), z[4 + e] = __uint_as_float(r.v[1][e]);
}
template <typename T> __device__ __forceinline__ void store8(T* row, int v, int V, const float* z);
template <> __device__ __forceinline__ void store8<bf16_t>(bf16_t* row, int v, int V, const float* z) {
  typedef u32x4_t run_t __attribute__((aligned(2)));
  if (v + 8 <= V) {
    *reinterpret_cast<run_t*>(row + v) = u32x4_t{pack_bf16x2(z[0], z[1]), pack_bf16x2(z[2], z[3]), pack_bf16x2(z[4], z[5]),
                                                 pack_bf16x2(z[6], z[7])};
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (v + e < V) row[v + e] = f2bf(z[e]);
  }
}
template <> __device__ __forceinline__ void store8<float>(float* row, int v, int V, const float* z) {
  typedef u32x4_t run_t __attribute__((aligned(4)));
  if (v + 8 <= V) {
    u32x4_t a, b;
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = __float_as_uint(z[e]), b[e] = __float_as_uint(z[4 + e]);
    *reinterpret_cast<run_t*>(row + v) = a;
    *reinterpret_cast<run_t*>(row + v + 4) = b;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (v + e < V) row[v + e] = z[e];
  }
}

// What a row's controls come to: row pointers (null where there is none) and its penalties.
struct RowControls {
  const int16_t* history;
  const void* bias;
  const uint8_t* mask;
  bool bias_f32;
  float r, f, p;
};
__device__ __forceinline__ RowControls row_controls(const hdcm_logits_controls& c, int64_t b) {
  RowControls o;
  o.r = c.repetition ? c.repetition[b] : c.repetition_all;
  o.f = c.frequency ? c.frequency[b] : c.frequency_all;
  o.p = c.presence ? c.presence[b] : c.presence_all;
  // a row without penalties does not read its history
  const bool none = o.r == 1.f && o.f == 0.f && o.p == 0.f;
  o.history = c.history && !none ? c.history + b * c.history_row_stride : nullptr;
  o.bias_f32 = c.bias_dtype == HDCM_F32;
  o.bias = c.bias ? (o.bias_f32 ? (const void*)((const float*)c.bias + b * c.bias_row_stride)
                                : (const void*)((const bf16_t*)c.bias + b * c.bias_row_stride))
                  : nullptr;
  o.mask = c.mask ? (const uint8_t*)(c.mask + b * c.mask_row_stride) : nullptr;
  return o;
}

// Eight logits from column v (a multiple of 8) on and what their controls hold: all loads first, converted
// only in z(), so that none waits for another.
template <typename T> struct Eight {
  Run<T> l;
  Run<int16_t> h;
  Run<bf16_t> b16;
  Run<float> b32, noise;
  uint32_t mask;
  int n;  // columns inside the row
  __device__ __forceinline__ void load(const T* row, const RowControls& c, const float* nrow, int v, int V) {
    n = min(8, V - v);
    if (n == 8) {
      l = load_run(row + v);
      if (c.history) h = load_run(c.history + v);
      if (c.bias && c.bias_f32) b32 = load_run((const float*)c.bias + v);
      if (c.bias && !c.bias_f32) b16 = load_run((const bf16_t*)c.bias + v);
      if (nrow) noise = load_run(nrow + v);
    } else {
      l = load_end(row + v, n);
      if (c.history) h = load_end(c.history + v, n);
      if (c.bias && c.bias_f32) b32 = load_end((const float*)c.bias + v, n);
      if (c.bias && !c.bias_f32) b16 = load_end((const bf16_t*)c.bias + v, n);
      if (nrow) noise = load_end(nrow + v, n);
    }
    if (c.mask) mask = c.mask[v / 8];  // bit v % 32 of word v / 32, little endian
  }
  // the processed logits; -inf behind the row's end
  __device__ __forceinline__ void z(const RowControls& c, float* z) const {
#pragma clang fp contract(off)
    values(l, z);
    if (c.history && (h.v[0][0] | h.v[0][1] | h.v[0][2] | h.v[0][3])) {  // most tokens were never seen
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t t = (h.v[0][e / 2] >> (16 * (e & 1))) & 0xffffu, count = t & 0x7fffu;
        if (t) z[e] = z[e] > 0.f ? z[e] / c.r : z[e] * c.r;
        z[e] = z[e] - (count ? c.f * (float)count : 0.f);  // an infinite penalty bans what the output holds, no more
        z[e] = z[e] - (count ? c.p : 0.f);
      }
    }
    if (c.bias) {
      float b[8];
      if (c.bias_f32) values(b32, b);
      else values(b16, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = z[e] + b[e];
    }
    const uint32_t allowed = (c.mask ? mask : 0xffu) & (n < 8 ? (1u << n) - 1 : 0xffu);
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = (allowed >> e) & 1 ? z[e] : -kInf;
  }
};

// Bound by its one pass: 64 x 50277 bf16 with history, a shared bias and masks (20 MB) 8.1 us (from HBM 9.6), of which 2
// are a launch: 63 % of a copy's rate, since odd rows make the 16-byte accesses straddle their lines; one sequence 3.4 us
// recorded.
constexpr int kProcThreads = 256;

template <typename T>
__global__ __launch_bounds__(kProcThreads) void logits_process_kernel(const T* logits, int64_t l_rs, hdcm_logits_controls ctl,
                                                                      T* out, int64_t o_rs, int64_t B, int V) {
  const int v = 8 * (blockIdx.x * kProcThreads + threadIdx.x);
  if (v >= V) return;
  for (int64_t b = blockIdx.y; b < B; b += gridDim.y) {
    const RowControls c = row_controls(ctl, b);
    Eight<T> x;
    x.load(logits + b * l_rs, c, nullptr, v, V);
    float z[8];
    x.z(c, z);
    store8<T>(out + b * o_rs, v, V, z);
  }
}

// ------------------------------------------------------------------ choice of the token
// The best candidate (its t + noise, index and t) and the running maximum and sum of exp(t - max).
struct Pick {
  float best, t, max, sum;
  int at;
};
constexpr int kNoToken = 0x7fffffff;
__device__ __forceinline__ Pick no_pick() { return {-kInf, -kInf, -kInf, 0.f, kNoToken}; }

// Maximum and minimum over the 64 lanes on DPP lane moves (the steps of wave_total; a lane without a
// source keeps its own value), read into a wave-uniform scalar.
__device__ __forceinline__ float wave_max(float v) {
#define HDCM_STEP(CTRL, ROWS)                                                                                         \
  v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), CTRL, ROWS, 0xf, false)));
  HDCM_STEP(0xB1, 0xf) HDCM_STEP(0x4E, 0xf) HDCM_STEP(0x141, 0xf) HDCM_STEP(0x140, 0xf) HDCM_STEP(0x142, 0xa) HDCM_STEP(0x143, 0xc)
#undef HDCM_STEP
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ int wave_min(int v) {
#define HDCM_STEP(CTRL, ROWS) v = min(v, __builtin_amdgcn_update_dpp(v, v, CTRL, ROWS, 0xf, false));
  HDCM_STEP(0xB1, 0xf) HDCM_STEP(0x4E, 0xf) HDCM_STEP(0x141, 0xf) HDCM_STEP(0x140, 0xf) HDCM_STEP(0x142, 0xa) HDCM_STEP(0x143, 0xc)
#undef HDCM_STEP
  return __builtin_amdgcn_readlane(v, 63);
}
// The lanes' picks as one (in every lane): ties of `best` go to the lowest index.
__device__ __forceinline__ Pick merge_lanes(const Pick& a) {
  Pick o;
  o.max = wave_max(a.max);
  const float ref = o.max == -kInf ? 0.f : o.max;
  o.sum = wave_total(a.sum * fexp(a.max - ref));
  o.best = wave_max(a.best);
  o.at = wave_min(a.best == o.best ? a.at : kNoToken);
  const uint64_t owner = __ballot(a.best == o.best && a.at == o.at);  // one lane, or (no token) all
  o.t = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(a.t), owner ? __builtin_ctzll(owner) : 0));
  return o;
}
__device__ __forceinline__ void write_pick(const Pick& a, int64_t* token, float* logprob) {
  // nothing allowed (or only NaN): no token
  const bool none = a.at == kNoToken;
  *token = none ? -1 : a.at;
  *logprob = none ? -kInf : (a.t - a.max) - logf(a.sum);  // of large logits: no rounding at their magnitude
}

constexpr int kPickThreads = 512;
constexpr int kPickWaves = kPickThreads / kWave;

// Workgroup (s, b) takes part s of gridDim.x of row b, in whole groups of eight columns.  One pass: the
// eight values' maximum moves the running one, and only a maximum above the best so far is looked
// up.  128 x 50304 fp32 with history, biases and noise (90 MB) 20.4 us: the read.  16 x 50304 bf16 with
// history and masks 6.4 us recorded (7.6 with every input from HBM), two launches and their latency: a row on one
// workgroup of 1024 threads, without a join, takes 9.8 us at one sequence, in parts 4.9.
template <typename T>
__global__ __launch_bounds__(kPickThreads) void token_select_kernel(const T* logits, int64_t l_rs, hdcm_logits_controls ctl,
                                                                    const float* temperature, float temperature_all,
                                                                    const float* noise, int64_t n_rs, int V, int part,
                                                                    Pick* ws, int64_t* tokens, float* logprobs) {
#pragma clang fp contract(off)
  __shared__ Pick picks[kPickWaves];
  const int64_t b = blockIdx.y;
  const RowControls c = row_controls(ctl, b);
  const float temp = temperature ? temperature[b] : temperature_all;
  const bool greedy = !(temp > 0.f);
  const T* row = logits + b * l_rs;
  const float* nrow = noise && !greedy ? noise + b * n_rs : nullptr;
  const int v0 = blockIdx.x * part, v1 = min(v0 + part, V);
  Pick a = no_pick();
  for (int v = v0 + 8 * threadIdx.x; v < v1; v += 8 * kPickThreads) {
    Eight<T> x;
    x.load(row, c, nrow, v, V);
    float t[8], n[8];
    x.z(c, t);
    if (!greedy && temp != 1.f) {
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = t[e] / temp;
    }
    const float top = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
    float best = top;
    if (nrow) {
      values(x.noise, n);
#pragma unroll
      for (int e = 0; e < 8; ++e) n[e] = t[e] + n[e];
      best = fmaxf(fmaxf(fmaxf(n[0], n[1]), fmaxf(n[2], n[3])), fmaxf(fmaxf(n[4], n[5]), fmaxf(n[6], n[7])));
    }
    if (best > a.best) {  // a thread's columns ascend, so a tie keeps the lower one; -inf and NaN are no candidates
      a.best = best;
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if ((nrow ? n[e] : t[e]) == best) a.at = v + e, a.t = t[e];
    }
    const float m = fmaxf(a.max, top), ref = m == -kInf ? 0.f : m;
    float s = a.sum * fexp(a.max - ref);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += fexp(t[e] - ref);
    a.sum = s, a.max = m;
  }
  a = merge_lanes(a);
  const int w = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  if (lane == 0) picks[w] = a;
  __syncthreads();
  if (w != 0) return;
  a = merge_lanes(lane < kPickWaves ? picks[lane] : no_pick());
  if (lane != 0) return;
  if (gridDim.x == 1) write_pick(a, tokens + b, logprobs + b);
  else ws[b * gridDim.x + blockIdx.x] = a;
}

// The parts of a row, at most a wave's lanes.
__global__ __launch_bounds__(kWave) void token_select_join_kernel(const Pick* ws, int parts, int64_t* tokens, float* logprobs) {
  const int64_t b = blockIdx.x;
  const Pick a = merge_lanes((int)threadIdx.x < parts ? ws[b * parts + threadIdx.x] : no_pick());
  if (threadIdx.x == 0) write_pick(a, tokens + b, logprobs + b);
}

// Parts of a row: enough workgroups for the CUs, each with a full pass of its threads at least.
int select_parts(int64_t B, int64_t V) {
  const int64_t full = (V + 8 * kPickThreads - 1) / (8 * kPickThreads), want = (1024 + B - 1) / B;
  const int64_t n = full < want ? full : want;
  return (int)(n < kWave ? n : kWave);
}

// ------------------------------------------------------------------ token history
constexpr int kHistThreads = 512;
constexpr int kHistSlice = 8 * kHistThreads;  // tokens of a row per workgroup

// Calls f with the ids[0..n) that lie in [v0, v0 + size), less v0; eight loads of a thread in flight.
template <typename F>
__device__ __forceinline__ void each_id(const int64_t* ids, int64_t n, int v0, int size, F f) {
  constexpr int U = 8;
  for (int64_t i0 = 0; i0 < n; i0 += U * kHistThreads) {
    int64_t id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * kHistThreads + threadIdx.x;
      id[u] = ids[i < n ? i : n - 1];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t at = (uint64_t)id[u] - (uint64_t)v0;
      if (i0 + u * kHistThreads + threadIdx.x < n && at < (uint64_t)size) f((int)at);
    }
  }
}

// 16 x 50304 with 8448 ids a row 3.9 us recorded (5.4 from HBM), 1 x 50304 with 200 3.1: a launch, the
// ids' latency (each of a row's 13 slices reads all of them) and the table's one write.
// Workgroup (s, b) counts slice s of row b in LDS from all of the row's ids, then writes the slice, eight
// entries a thread: no atomics on the table, every entry written once.  keep: on top of what the
// table holds.
__global__ __launch_bounds__(kHistThreads) void token_history_kernel(int16_t* table, int64_t rs, const int64_t* prompt,
                                                                     int64_t p_rs, const int64_t* p_len, int64_t P,
                                                                     const int64_t* output, int64_t o_rs,
                                                                     const int64_t* o_len, int64_t O, int V, bool keep) {
  typedef u32x4_t run_t __attribute__((aligned(2)));
  __shared__ __attribute__((aligned(16))) uint32_t cell[kHistSlice];  // bit 31: in the prompt; below: the count
  const int64_t b = blockIdx.y;
  const int v0 = blockIdx.x * kHistSlice, n = min(kHistSlice, V - v0), i0 = 8 * threadIdx.x;
  int16_t* row = table + b * rs + v0;
  uint32_t h[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (keep) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t t = i0 + e < n ? (uint16_t)row[i0 + e] : 0u;
      h[e] = (t & 0x7fffu) | (t >> 15) << 31;
    }
  }
  u32x4_t* mine = reinterpret_cast<u32x4_t*>(cell + i0);
  mine[0] = u32x4_t{h[0], h[1], h[2], h[3]};
  mine[1] = u32x4_t{h[4], h[5], h[6], h[7]};
  __syncthreads();
  const int64_t np = p_len ? min(max(p_len[b], (int64_t)0), P) : P, no = o_len ? min(max(o_len[b], (int64_t)0), O) : O;
  each_id(prompt + b * p_rs, np, v0, n, [&](int at) { atomicOr(&cell[at], 0x80000000u); });
  each_id(output + b * o_rs, no, v0, n, [&](int at) { atomicAdd(&cell[at], 1u); });
  __syncthreads();
  u32x4_t o;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x4_t c = mine[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) h[4 * i + e] = min(c[e] & 0x7fffffffu, 0x7fffu) | (c[e] >> 31) << 15;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = h[2 * e] | h[2 * e + 1] << 16;
  if (i0 + 8 <= n) {
    *reinterpret_cast<run_t*>(row + i0) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i0 + e < n) row[i0 + e] = (int16_t)h[e];
  }
}

// A few tokens per row, one thread each row, in order (so a token that comes twice is counted twice
// without atomics): 2.1 us for 64 rows, an empty kernel's time.
__global__ __launch_bounds__(kWave) void token_append_kernel(int16_t* table, int64_t rs, const int64_t* tokens, int64_t t_rs,
                                                             const int64_t* lengths, int64_t T, int64_t B, int V) {
  const int64_t b = (int64_t)blockIdx.x * kWave + threadIdx.x;
  if (b >= B) return;
  const int64_t n = lengths ? min(max(lengths[b], (int64_t)0), T) : T;
  for (int64_t i = 0; i < n; ++i) {
    const int64_t t = tokens[b * t_rs + i];
    if (t < 0 || t >= V) continue;
    const uint16_t h = (uint16_t)table[b * rs + t];
    if ((h & 0x7fffu) != 0x7fffu) table[b * rs + t] = (int16_t)(h + 1);
  }
}

constexpr int64_t kMaxVocab = (int64_t)1 << 30, kMaxRows = 65535;
constexpr int64_t kMaxIds = (int64_t)1 << 30;  // of a row: a count of them and of what the table holds stays below bit 31

int check_controls(const hdcm_logits_controls* c, int64_t B, int64_t V) {
  HDCM_CHECK_ARG(c, HDCM_EINVAL);
  HDCM_CHECK_ARG(!c->history || c->history_row_stride >= V || B <= 1, HDCM_EINVAL);
  HDCM_CHECK_ARG(!c->bias || c->bias_row_stride >= V || c->bias_row_stride == 0, HDCM_EINVAL);
  HDCM_CHECK_ARG(!c->bias || c->bias_dtype == HDCM_F32 || c->bias_dtype == HDCM_BF16, HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(!c->mask || c->mask_row_stride >= (V + 31) / 32 || c->mask_row_stride == 0, HDCM_EINVAL);
  return HDCM_OK;
}

}  // namespace

extern "C" int hdcm_logits_process(const void* logits, int64_t logits_row_stride, const hdcm_logits_controls* controls, void* out,
                                   int64_t out_row_stride, int64_t B, int64_t V, int dtype, void* stream) {
  HDCM_CHECK_ARG(dtype == HDCM_F32 || dtype == HDCM_BF16, HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(B >= 0 && V >= 0, HDCM_EINVAL);
  if (B == 0 || V == 0) return HDCM_OK;
  HDCM_CHECK_ARG(logits && out, HDCM_EINVAL);
  HDCM_CHECK_ARG(B == 1 || (logits_row_stride >= V && out_row_stride >= V), HDCM_EINVAL);
  HDCM_CHECK_ARG(V <= kMaxVocab, HDCM_EUNSUPPORTED);
  const int st = check_controls(controls, B, V);
  if (st) return st;
  const dim3 grid((unsigned)((V + 8 * kProcThreads - 1) / (8 * kProcThreads)), (unsigned)(B < kMaxRows ? B : kMaxRows));
  hipStream_t s = (hipStream_t)stream;
  if (dtype == HDCM_F32)
    HDCM_LAUNCH(logits_process_kernel<float>, grid, dim3(kProcThreads), 0, s, (const float*)logits, logits_row_stride,
                *controls, (float*)out, out_row_stride, B, (int)V);
  else
    HDCM_LAUNCH(logits_process_kernel<bf16_t>, grid, dim3(kProcThreads), 0, s, (const bf16_t*)logits, logits_row_stride,
                *controls, (bf16_t*)out, out_row_stride, B, (int)V);
  return hdcm_launch_status();
}

extern "C" size_t hdcm_token_select_workspace_bytes(int64_t B, int64_t V) {
  if (B <= 0 || V <= 0) return 0;
  const int parts = select_parts(B, V);
  return parts > 1 ? (size_t)B * parts * sizeof(Pick) : 0;
}

extern "C" int hdcm_token_select(const void* logits, int64_t logits_row_stride, const hdcm_logits_controls* controls,
                                 const float* temperature, float temperature_all, const float* noise,
                                 int64_t noise_row_stride, int64_t* tokens, float* logprobs, void* ws, size_t ws_bytes,
                                 int64_t B, int64_t V, int dtype, void* stream) {
  HDCM_CHECK_ARG(dtype == HDCM_F32 || dtype == HDCM_BF16, HDCM_EUNSUPPORTED);
  HDCM_CHECK_ARG(B >= 0 && V > 0, HDCM_EINVAL);
  if (B == 0) return HDCM_OK;
  HDCM_CHECK_ARG(logits && tokens && logprobs, HDCM_EINVAL);
  HDCM_CHECK_ARG(B == 1 || (logits_row_stride >= V && (!noise || noise_row_stride >= V)), HDCM_EINVAL);
  HDCM_CHECK_ARG(V <= kMaxVocab && B <= kMaxRows, HDCM_EUNSUPPORTED);
  const int st = check_controls(controls, B, V);
  if (st) return st;
  const int parts = select_parts(B, V);
  HDCM_CHECK_ARG(parts == 1 || (ws && ws_bytes >= hdcm_token_select_workspace_bytes(B, V)), HDCM_EWORKSPACE);
  HDCM_CHECK_ARG(parts == 1 || ((uintptr_t)ws & 3u) == 0, HDCM_EALIGN);
  const int part = (int)((V + 8 * parts - 1) / (8 * parts)) * 8;
  const dim3 grid((unsigned)parts, (unsigned)B);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == HDCM_F32)
    HDCM_LAUNCH(token_select_kernel<float>, grid, dim3(kPickThreads), 0, s, (const float*)logits, logits_row_stride, *controls,
                temperature, temperature_all, noise, noise_row_stride, (int)V, part, (Pick*)ws, tokens, logprobs);
  else
    HDCM_LAUNCH(token_select_kernel<bf16_t>, grid, dim3(kPickThreads), 0, s, (const bf16_t*)logits, logits_row_stride,
                *controls, temperature, temperature_all, noise, noise_row_stride, (int)V, part, (Pick*)ws, tokens, logprobs);
  if (parts > 1)
    HDCM_LAUNCH(token_select_join_kernel, dim3((unsigned)B), dim3(kWave), 0, s, (const Pick*)ws, parts, tokens, logprobs);
  return hdcm_launch_status();
}

extern "C" int hdcm_token_history_fill(int16_t* table, int64_t table_row_stride, const int64_t* prompt,
                                       int64_t prompt_row_stride, const int64_t* prompt_lengths, int64_t P,
                                       const int64_t* output, int64_t output_row_stride, const int64_t* output_lengths,
                                       int64_t O, int64_t B, int64_t V, void* stream) {
  HDCM_CHECK_ARG(B >= 0 && V >= 0 && P >= 0 && O >= 0, HDCM_EINVAL);
  if (B == 0 || V == 0) return HDCM_OK;
  HDCM_CHECK_ARG(table && (prompt || P == 0) && (output || O == 0), HDCM_EINVAL);
  HDCM_CHECK_ARG(B == 1 || (table_row_stride >= V && prompt_row_stride >= P && output_row_stride >= O), HDCM_EINVAL);
  HDCM_CHECK_ARG(V <= kMaxVocab && B <= kMaxRows && P <= kMaxIds && O <= kMaxIds, HDCM_EUNSUPPORTED);
  const dim3 grid((unsigned)((V + kHistSlice - 1) / kHistSlice), (unsigned)B);
  HDCM_LAUNCH(token_history_kernel, grid, dim3(kHistThreads), 0, (hipStream_t)stream, table, table_row_stride, prompt,
              prompt_row_stride, prompt_lengths, P, output, output_row_stride, output_lengths, O, (int)V, false);
  return hdcm_launch_status();
}

extern "C" int hdcm_token_history_append(int16_t* table, int64_t table_row_stride, const int64_t* tokens,
                                         int64_t tokens_row_stride, const int64_t* lengths, int64_t T, int64_t B, int64_t V,
                                         void* stream) {
  HDCM_CHECK_ARG(B >= 0 && V >= 0 && T >= 0, HDCM_EINVAL);
  if (B == 0 || V == 0 || T == 0) return HDCM_OK;
  HDCM_CHECK_ARG(table && tokens, HDCM_EINVAL);
  HDCM_CHECK_ARG(B == 1 || (table_row_stride >= V && tokens_row_stride >= T), HDCM_EINVAL);
  HDCM_CHECK_ARG(V <= kMaxVocab && B <= kMaxRows && T <= kMaxIds, HDCM_EUNSUPPORTED);
  hipStream_t s = (hipStream_t)stream;
  // Up to 16 tokens a row (a step, or a few accepted drafts) touch single entries, one round trip each; more are counted
  // slice by slice, which reads and writes the whole table.  us recorded for 1, 8, 16 and 24 tokens of 50304, single and
  // by slices: 1 row 1.8, 3.2, 5.1, 6.9 and 3.6; 16 rows 1.8, 3.4, 5.7, 7.8 and 3.9; 64 rows 1.8, 4.0, 6.7, 9.2 and 8.1;
  // 256 rows 2.1, 4.1, 6.9, 9.3 and 22.
  if (T <= 16)
    HDCM_LAUNCH(token_append_kernel, dim3((unsigned)((B + kWave - 1) / kWave)), dim3(kWave), 0, s, table, table_row_stride,
                tokens, tokens_row_stride, lengths, T, B, (int)V);
  else
    HDCM_LAUNCH(token_history_kernel, dim3((unsigned)((V + kHistSlice - 1) / kHistSlice), (unsigned)B), dim3(kHistThreads), 0,
                s, table, table_row_stride, (const int64_t*)nullptr, (int64_t)0, (const int64_t*)nullptr, (int64_t)0, tokens,
                tokens_row_stride, lengths, T, (int)V, true);
  return hdcm_launch_status();
}
