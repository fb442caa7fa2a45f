// From logits to the next tokens of a batch of sequences (no counterpart in the reference, whose
// generate samples on the host side of torch, train.py:139-151):
//   process:  z = seen ? (l > 0 ? l / r : l r) : l;  z -= f count;  z -= p [count > 0];  z += bias;
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

// Eight values of a row from column v on at the type's own alignment (rows of an odd vocabulary start
// anywhere); `pad` past the row's V columns.
template <typename T> __device__ __forceinline__ void load8(const T* row, int v, int V, float pad, float* z);
template <> __device__ __forceinline__ void load8<bf16_t>(const bf16_t* row, int v, int V, float pad, float* z) {
  typedef u32x4_t run_t __attribute__((aligned(2)));
  if (v + 8 <= V) {
    const u32x4_t a = *reinterpret_cast<const run_t*>(row + v);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      z[2 * e] = __uint_as_float(a[e] << 16);
      z[2 * e + 1] = __uint_as_float(a[e] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = v + e < V ? bf2f(row[v + e]) : pad;
  }
}
template <> __device__ __forceinline__ void load8<float>(const float* row, int v, int V, float pad, float* z) {
  typedef u32x4_t run_t __attribute__((aligned(4)));
  if (v + 8 <= V) {
    const u32x4_t a = *reinterpret_cast<const run_t*>(row + v), b = *reinterpret_cast<const run_t*>(row + v + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = __uint_as_float(a[e]), z[4 + e] = __uint_as_float(b[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = v + e < V ? row[v + e] : pad;
  }
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

// z of eight logits from column v (a multiple of 8) on; columns past V become -inf.
template <typename T>
__device__ __forceinline__ void process8(const T* row, const RowControls& c, int v, int V, float* z) {
#pragma clang fp contract(off)
  load8<T>(row, v, V, -kInf, z);
  if (c.history) {
    typedef u32x4_t run_t __attribute__((aligned(2)));
    u32x4_t h = {0, 0, 0, 0};
    if (v + 8 <= V) {
      h = *reinterpret_cast<const run_t*>(c.history + v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (v + e < V) h[e / 2] |= (uint32_t)(uint16_t)c.history[v + e] << (16 * (e & 1));
    }
    if (h[0] | h[1] | h[2] | h[3]) {  // most tokens were never seen
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t t = (h[e / 2] >> (16 * (e & 1))) & 0xffffu, count = t & 0x7fffu;
        if (t) z[e] = z[e] > 0.f ? z[e] / c.r : z[e] * c.r;
        z[e] = z[e] - c.f * (float)count;
        z[e] = z[e] - (count ? c.p : 0.f);
      }
    }
  }
  if (c.bias) {
    float b[8];
    if (c.bias_f32) load8<float>((const float*)c.bias, v, V, 0.f, b);
    else load8<bf16_t>((const bf16_t*)c.bias, v, V, 0.f, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = z[e] + b[e];
  }
  if (c.mask) {
    const uint32_t m = c.mask[v / 8];  // bit v % 32 of word v / 32, little endian
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = (m >> e) & 1 ? z[e] : -kInf;
  }
}

constexpr int kProcThreads = 256;

template <typename T>
__global__ __launch_bounds__(kProcThreads) void logits_process_kernel(const T* logits, int64_t l_rs, hdcm_logits_controls ctl,
                                                                      T* out, int64_t o_rs, int64_t B, int V) {
  const int v = 8 * (blockIdx.x * kProcThreads + threadIdx.x);
  if (v >= V) return;
  for (int64_t b = blockIdx.y; b < B; b += gridDim.y) {
    const RowControls c = row_controls(ctl, b);
    float z[8];
    process8<T>(logits + b * l_rs, c, v, V, z);
    store8<T>(out + b * o_rs, v, V, z);
  }
}

// ------------------------------------------------------------------ choice of the token
// The best candidate (its t + noise, index and t) and the running maximum and sum of exp(t - max).
struct Pick {
  float best, t, max, sum;
  int at;
};
__device__ __forceinline__ Pick no_pick() { return {-kInf, -kInf, -kInf, 0.f, 0x7fffffff}; }
__device__ __forceinline__ void merge(Pick& a, const Pick& b) {
  if (b.best > a.best || (b.best == a.best && b.at < a.at)) a.best = b.best, a.at = b.at, a.t = b.t;
  const float m = fmaxf(a.max, b.max), ref = m == -kInf ? 0.f : m;
  a.sum = a.sum * fexp(a.max - ref) + b.sum * fexp(b.max - ref);
  a.max = m;
}
__device__ __forceinline__ Pick merge_lanes(Pick a) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const Pick b = {__shfl_xor(a.best, o, kWave), __shfl_xor(a.t, o, kWave), __shfl_xor(a.max, o, kWave),
                    __shfl_xor(a.sum, o, kWave), __shfl_xor(a.at, o, kWave)};
    merge(a, b);
  }
  return a;
}
__device__ __forceinline__ void write_pick(const Pick& a, int64_t* token, float* logprob) {
  // nothing allowed (or only NaN): no token
  const bool none = a.at == 0x7fffffff;
  *token = none ? -1 : a.at;
  *logprob = none ? -kInf : a.t - (a.max + logf(a.sum));
}

constexpr int kPickThreads = 512;
constexpr int kPickWaves = kPickThreads / kWave;

// Workgroup (s, b) takes part s of gridDim.x of row b, in whole groups of eight columns.
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
    float t[8], n[8];
    process8<T>(row, c, v, V, t);
    if (!greedy && temp != 1.f) {
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] = t[e] / temp;
    }
    if (nrow) load8<float>(nrow, v, V, 0.f, n);
    float m = a.max;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = nrow ? t[e] + n[e] : t[e];
      // a thread's columns ascend, so a tie keeps the lower one; -inf and NaN are no candidates
      if (x > a.best) a.best = x, a.at = v + e, a.t = t[e];
      m = fmaxf(m, t[e]);
    }
    const float ref = m == -kInf ? 0.f : m;
    float s = a.sum * fexp(a.max - ref);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += fexp(t[e] - ref);
    a.sum = s, a.max = m;
  }
  a = merge_lanes(a);
  if (threadIdx.x % kWave == 0) picks[threadIdx.x / kWave] = a;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < kPickWaves; ++w) merge(a, picks[w]);
  if (gridDim.x == 1) write_pick(a, tokens + b, logprobs + b);
  else ws[b * gridDim.x + blockIdx.x] = a;
}

// The parts of a row in order, one wave per row.
__global__ __launch_bounds__(kWave) void token_select_join_kernel(const Pick* ws, int parts, int64_t* tokens, float* logprobs) {
  const int64_t b = blockIdx.x;
  Pick a = no_pick();
  for (int s = threadIdx.x; s < parts; s += kWave) merge(a, ws[b * parts + s]);
  a = merge_lanes(a);
  if (threadIdx.x == 0) write_pick(a, tokens + b, logprobs + b);
}

int select_parts(int64_t B, int64_t V) {
  const int64_t most = (V + 8191) / 8192;
  return B >= 256 ? 1 : (int)most;
}

// ------------------------------------------------------------------ token history
constexpr int kHistThreads = 256;
constexpr int kHistSlice = 4096;  // tokens of a row per workgroup

// Workgroup (s, b) counts slice s of row b in LDS from all of the row's ids, then writes the slice: no
// atomics on the table, every entry written once.  keep: on top of what the table holds.
__global__ __launch_bounds__(kHistThreads) void token_history_kernel(int16_t* table, int64_t rs, const int64_t* prompt,
                                                                     int64_t p_rs, const int64_t* p_len, int64_t P,
                                                                     const int64_t* output, int64_t o_rs,
                                                                     const int64_t* o_len, int64_t O, int V, bool keep) {
  __shared__ uint32_t cell[kHistSlice];  // bit 31: in the prompt; below: the count
  const int64_t b = blockIdx.y;
  const int v0 = blockIdx.x * kHistSlice, n = min(kHistSlice, V - v0);
  int16_t* row = table + b * rs + v0;
  for (int i = threadIdx.x; i < n; i += kHistThreads) {
    const uint32_t h = keep ? (uint16_t)row[i] : 0u;
    cell[i] = (h & 0x7fffu) | (h >> 15) << 31;
  }
  __syncthreads();
  const int64_t np = p_len ? min(max(p_len[b], (int64_t)0), P) : P, no = o_len ? min(max(o_len[b], (int64_t)0), O) : O;
  for (int64_t i = threadIdx.x; i < np; i += kHistThreads) {
    const uint64_t at = (uint64_t)(prompt[b * p_rs + i] - v0);
    if (at < (uint64_t)n) atomicOr(&cell[at], 0x80000000u);
  }
  for (int64_t i = threadIdx.x; i < no; i += kHistThreads) {
    const uint64_t at = (uint64_t)(output[b * o_rs + i] - v0);
    if (at < (uint64_t)n) atomicAdd(&cell[at], 1u);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kHistThreads) {
    const uint32_t h = cell[i];
    row[i] = (int16_t)(min(h & 0x7fffffffu, 0x7fffu) | (h >> 31) << 15);
  }
}

// A few tokens per row, one thread each row, in order.
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
  HDCM_CHECK_ARG(V <= kMaxVocab && B <= kMaxRows && P < ((int64_t)1 << 31) && O < ((int64_t)1 << 31), HDCM_EUNSUPPORTED);
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
  HDCM_CHECK_ARG(V <= kMaxVocab && B <= kMaxRows && T < ((int64_t)1 << 31), HDCM_EUNSUPPORTED);
  hipStream_t s = (hipStream_t)stream;
  // up to 16 tokens a row (a step, or a few accepted drafts) touch single entries; more are counted slice by slice
  if (T <= 16)
    HDCM_LAUNCH(token_append_kernel, dim3((unsigned)((B + kWave - 1) / kWave)), dim3(kWave), 0, s, table, table_row_stride,
                tokens, tokens_row_stride, lengths, T, B, (int)V);
  else
    HDCM_LAUNCH(token_history_kernel, dim3((unsigned)((V + kHistSlice - 1) / kHistSlice), (unsigned)B), dim3(kHistThreads), 0,
                s, table, table_row_stride, (const int64_t*)nullptr, (int64_t)0, (const int64_t*)nullptr, (int64_t)0, tokens,
                tokens_row_stride, lengths, T, (int)V, true);
  return hdcm_launch_status();
}
