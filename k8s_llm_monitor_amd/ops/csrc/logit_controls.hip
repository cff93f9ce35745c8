// Controls of logits ahead of the sampler: penalties for repeated tokens, biases, allowed-token masks - in one pass.
//
//   seen in prompt or answer:  x <- x > 0 ? x / repetition : x * repetition
//   x <- x - frequency * count - presence * [count > 0]     count: how often the answer has the token
//   x <- x + bias;   not allowed: -inf
//
// The history is read where it lies, in pages of token ids beside the KV cache's (the same block tables), so a sequence's
// controls need nothing that a scheduler would have to keep in step.  Vocabulary parts are workgroups: each holds one word per token of
// its part in LDS - count (20 bits), a prompt bit, the number of the token's bias entry (11 bits) -, scans the row's history with integer LDS
// atomics (any order, same result), then makes its one pass over the logits, which it has asked for ahead of the history; only tokens with
// a word take the long way.  32-bit arithmetic, one rounding to the output's type at the end.
//
// Bound by memory - the logits in and out, a bit a token of the mask - and the chain in front of them: 64 rows of 128256 in bf16, 34 MB:
// 10.4 us, 3.3 TB/s (a large copy moves 5.1), of which the launch, the history's two trips and the LDS words are about 4.
#include "common.h"

namespace k8sllm {

constexpr int kLcThreads = 1024;
constexpr uint32_t kLcPrompt = 1u << 20, kLcCount = kLcPrompt - 1;
constexpr int kLcBias = 21;  // first bit of the bias entry's number

struct LogitControls {
  const float* params;    // [slots][3]: repetition, presence, frequency
  const int* info;        // [slots][2]: tokens of the prompt, whether the mask counts
  const int* bias_ids;    // [slots][n_bias], < 0: none
  const float* bias_vals;
  const uint32_t* masks;  // [slots][words], bit v % 32 of word v / 32: token v is allowed
  int slots, n_bias, words;
  const int* rows;        // [B]: the row's slot, < 0: no controls
  const int* tokens;      // [pages][16]
  int pages;
  const int* table;
  long table_stride;
  int table_width;
  const int* lens;
};

// 8 logits in a row, as loaded
template <typename T>
struct LcGroup {
  static constexpr int N = sizeof(T) / 2;
  uint4 w[N];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void get(float* x) const {
    if constexpr (N == 1) {
      unpack8(w[0], x);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[4 * i] = __uint_as_float(w[i].x);
        x[4 * i + 1] = __uint_as_float(w[i].y);
        x[4 * i + 2] = __uint_as_float(w[i].z);
        x[4 * i + 3] = __uint_as_float(w[i].w);
      }
    }
  }
};

__device__ __forceinline__ float lc_get(const bf16_t* p) { return bf2f(*p); }
__device__ __forceinline__ float lc_get(const float* p) { return *p; }
__device__ __forceinline__ void lc_put(bf16_t* p, float x) { *p = f2bf(x); }
__device__ __forceinline__ void lc_put(float* p, float x) { *p = x; }
__device__ __forceinline__ void lc_put8(bf16_t* p, const float* x) { *reinterpret_cast<uint4*>(p) = pack8(x); }
__device__ __forceinline__ void lc_put8(float* p, const float* x) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}

constexpr int kLcGroups = 2;  // of a thread: parts of at most 16384 tokens

// grid (parts, rows); dynamic LDS: `chunk` words (a multiple of 256, at most 8 * kLcGroups * kLcThreads)
template <typename TI, typename TO>
__global__ __launch_bounds__(kLcThreads) void logit_controls_kernel(TO* out, long out_stride, const TI* in, long in_stride, int V, int chunk,
                                                                    const LogitControls c) {
  extern __shared__ __attribute__((aligned(16))) uint32_t s_word[];
  const int b = blockIdx.y, tid = threadIdx.x;
  const TI* x = in + (long)b * in_stride;
  TO* y = out + (long)b * out_stride;
  // a row begins anywhere (an odd vocabulary): its groups of 8 begin where loads of 16 bytes do, the first part's first group ahead of the row
  const int ahead = (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(TI);  // tokens ahead of the first such place
  const int base = blockIdx.x * chunk + (ahead ? ahead - 8 : 0);
  const int lo = max(base, 0), hi = min(V, base + chunk);
  const bool vout = ((uintptr_t)(y + ahead) & 15) == 0;  // uniform
  int slot = c.rows[b];
  if (slot >= c.slots) slot = -1;
  if (slot < 0 && (const void*)x == (const void*)y) return;
  // What does not hang on one another is asked for together: the history's first 4096 tokens, the slot's numbers, the logits
  const int* bt = c.table + (long)b * c.table_stride;
  const int width = c.table_width * 16, t0 = tid * 4;
  auto history = [&](int t) {
    const int page = bt[t >> 4];
    return page >= 0 && page < c.pages ? *reinterpret_cast<const int4*>(c.tokens + (long)page * 16 + (t & 15)) : make_int4(-1, -1, -1, -1);
  };
  int4 first = make_int4(-1, -1, -1, -1);
  if (t0 < width) first = history(t0);
  const int len = min(c.lens[b], width);
  int prompt = 0, entry = -1;
  float rep = 1.f, pres = 0.f, freq = 0.f;
  bool masked = false;
  const uint32_t* mask = c.masks;
  const int* bi = c.bias_ids;
  if (slot >= 0) {
    prompt = c.info[2 * slot];
    masked = c.info[2 * slot + 1] != 0;
    rep = c.params[3 * slot];
    pres = c.params[3 * slot + 1];
    freq = c.params[3 * slot + 2];
    mask += (long)slot * c.words;
    bi += (long)slot * c.n_bias;
    if (tid < c.n_bias) entry = bi[tid];
  }
  LcGroup<TI> g[kLcGroups];
#pragma unroll
  for (int i = 0; i < kLcGroups; ++i) {
    const int v = base + (i * kLcThreads + tid) * 8;
    if (v >= 0 && v + 8 <= hi) g[i].load(x + v);
  }
  if (slot >= 0) {
    for (int i = tid * 4; i < chunk; i += kLcThreads * 4) *reinterpret_cast<uint4*>(s_word + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    // bias entries beside the history: of several with one token the first counts, the one with the largest n_bias - j
    for (int j = tid; j < c.n_bias; j += kLcThreads) {
      const int v = j == tid ? entry : bi[j];
      if (v < lo || v >= hi) continue;
      const uint32_t mine = (uint32_t)(c.n_bias - j);
      uint32_t* p = &s_word[v - base];
      uint32_t had = *p;
      while ((had >> kLcBias) < mine) {  // ends: another's write either leaves a larger number or the compare succeeds
        const uint32_t now = atomicCAS(p, had, (had & (kLcPrompt | kLcCount)) | mine << kLcBias);
        if (now == had) break;
        had = now;
      }
    }
    for (int t = t0; t < len; t += kLcThreads * 4) {
      const int4 q = t == t0 ? first : history(t);
      const int id[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (t + j < len && id[j] >= lo && id[j] < hi) {
          if (t + j < prompt) atomicOr(&s_word[id[j] - base], kLcPrompt);
          else atomicAdd(&s_word[id[j] - base], 1u);
        }
    }
    __syncthreads();
  }
  const float* bv = c.bias_vals + (long)max(slot, 0) * c.n_bias;
  const float inv = 1.f / rep;  // one rounding more, half a step of 32 bits (a quotient for each token of a row's frequent ones is what the slowest workgroups would spend their time on)
  auto one = [&](float f, uint32_t w) {
    const float count = (float)(w & kLcCount);
    if (w & (kLcPrompt | kLcCount)) f *= f > 0.f ? inv : rep;
    if (w & kLcCount) f = f - freq * count - pres;
    if (w >> kLcBias) f += bv[c.n_bias - (int)(w >> kLcBias)];
    return f;
  };
#pragma unroll
  for (int i = 0; i < kLcGroups; ++i) {
    const int v = base + (i * kLcThreads + tid) * 8;
    if (v >= hi) break;
    if (v >= 0 && v + 8 <= hi) {
      float f[8];
      g[i].get(f);
      if (slot >= 0) {
        uint32_t ok = 0xffu;
        if (masked) ok = (uint32_t)((((uint64_t)mask[(v + 7) >> 5] << 32) | mask[v >> 5]) >> (v & 31));
        const uint4 p = *reinterpret_cast<const uint4*>(s_word + v - base), q = *reinterpret_cast<const uint4*>(s_word + v - base + 4);
        const uint32_t w[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (w[j]) f[j] = one(f[j], w[j]);
          if (!((ok >> j) & 1)) f[j] = -INFINITY;
        }
      }
      if (vout) {
        lc_put8(y + v, f);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) lc_put(y + v + j, f[j]);
      }
    } else {  // a row's ends
      for (int j = max(v, 0); j < min(v + 8, hi); ++j) {
        float f = lc_get(x + j);
        const uint32_t w = slot >= 0 ? s_word[j - base] : 0u;
        if (w) f = one(f, w);
        if (masked && !((mask[j >> 5] >> (j & 31)) & 1)) f = -INFINITY;
        lc_put(y + j, f);
      }
    }
  }
}

// Token ids into their pages; a row whose input is the token that the step before sampled (src >= 0) takes it from there.
__global__ __launch_bounds__(256) void cache_tokens_kernel(int* __restrict__ tokens, int pages, const int* __restrict__ ids,
                                                           const int* __restrict__ slots, const int* __restrict__ src,
                                                           const int* __restrict__ prev, int n_prev, int n) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int slot = slots[i];
  if (slot < 0 || (slot >> 4) >= pages) return;
  const int r = src != nullptr ? src[i] : -1;
  tokens[slot] = r >= 0 && r < n_prev ? prev[r] : ids[i];
}

}  // namespace k8sllm

using namespace k8sllm;

// dtypes: 0 bf16 -> bf16, 1 fp32 -> fp32, 2 bf16 -> fp32
extern "C" int k8sllm_logit_controls(void* out, long out_stride, const void* in, long in_stride, int types, int B, int V, const float* params,
                                     const int* info, const int* bias_ids, const float* bias_vals, const void* masks, int slots, int n_bias,
                                     int words, const int* rows, const int* tokens, int pages, const int* table, long table_stride,
                                     int table_width, const int* lens, hipStream_t s) {
  if (B <= 0 || V <= 0) return 0;
  if (n_bias > 2046 || (long)table_width * 16 >= (1 << 20) || B > 65535) return -2;
  const LogitControls c{params, info, bias_ids, bias_vals, (const uint32_t*)masks, slots, n_bias, words, rows, tokens, pages, table, table_stride,
                        table_width, lens};
  // two workgroups a CU where rows x parts allow, parts of 2 K to 16 K tokens (8 to 64 KB of LDS)
  const int n = V + 7;  // a row's groups may begin up to 7 tokens ahead of it
  int parts = (n + 16383) / 16384;
  const int want = (512 + B - 1) / B, most = (n + 2047) / 2048;
  parts = parts > (want < most ? want : most) ? parts : (want < most ? want : most);
  const int chunk = ((n + parts - 1) / parts + 255) & ~255;
  parts = (n + chunk - 1) / chunk;
  const dim3 grid(parts, B);
  const size_t lds = (size_t)chunk * 4;
#define K8S_LC(TI, TO)                                                                                                                  \
  hipLaunchKernelGGL((logit_controls_kernel<TI, TO>), grid, dim3(kLcThreads), lds, s, (TO*)out, out_stride, (const TI*)in, in_stride, V, chunk, c)
  if (types == 0) K8S_LC(bf16_t, bf16_t);
  else if (types == 1) K8S_LC(float, float);
  else if (types == 2) K8S_LC(bf16_t, float);
  else return -1;
#undef K8S_LC
  return (int)hipGetLastError();
}

extern "C" int k8sllm_cache_tokens(int* tokens, int pages, const int* ids, const int* slots, const int* src, const int* prev, int n_prev, int n,
                                   hipStream_t s) {
  if (n <= 0) return 0;
  hipLaunchKernelGGL(cache_tokens_kernel, dim3((n + 255) / 256), dim3(256), 0, s, tokens, pages, ids, slots, src, prev, n_prev, n);
  return (int)hipGetLastError();
}
