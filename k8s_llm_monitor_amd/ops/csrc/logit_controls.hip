// Controls of logits ahead of the sampler: penalties for repeated tokens, biases, allowed-token masks - in one pass.
//
//   seen in prompt or answer:  x <- x > 0 ? x / repetition : x * repetition
//   x <- x - frequency * count - presence * [count > 0]     count: how often the answer has the token
//   x <- x + bias;   not allowed: -inf
//
// The history is read where it lies, in pages of token ids beside the KV cache's (the same block tables), so a sequence's
// controls need nothing that a scheduler would have to keep in step.  Vocabulary parts are workgroups: each holds one word per token of its part in
// LDS - count (20 bits), a prompt bit, the number of the token's bias entry (11 bits) - scans the row's history with integer LDS
// atomics (any order, same result), then makes its one pass over the logits; only tokens with a word take the long way.  Bound by memory: the logits in and out,
// and a bit a token of the mask.  32-bit arithmetic, one rounding to the output's type at the end.
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

template <typename T>
__device__ __forceinline__ void lc_load(const T* p, float* x, bool vec) {  // 8 in a row
  if constexpr (sizeof(T) == 2) {
    if (vec) {
      unpack8(*reinterpret_cast<const uint4*>(p), x);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = bf2f(p[j]);
    }
  } else {
    if (vec) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = p[j];
    }
  }
}

template <typename T>
__device__ __forceinline__ void lc_store(T* p, const float* x, bool vec) {
  if constexpr (sizeof(T) == 2) {
    if (vec) {
      *reinterpret_cast<uint4*>(p) = pack8(x);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = f2bf(x[j]);
    }
  } else {
    if (vec) {
      *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = x[j];
    }
  }
}

// grid (parts, rows); dynamic LDS: `chunk` words (a multiple of 256)
template <typename TI, typename TO>
__global__ __launch_bounds__(kLcThreads) void logit_controls_kernel(TO* out, long out_stride, const TI* in, long in_stride, int V, int chunk,
                                                                    const LogitControls c) {
  extern __shared__ __attribute__((aligned(16))) uint32_t s_word[];
  const int b = blockIdx.y, tid = threadIdx.x;
  const int lo = blockIdx.x * chunk, hi = min(V, lo + chunk);
  const TI* x = in + (long)b * in_stride;
  TO* y = out + (long)b * out_stride;
  const bool vin = ((uintptr_t)x & 15) == 0, vout = ((uintptr_t)y & 15) == 0;  // uniform; lo is a multiple of 256
  int slot = c.rows[b];
  if (slot >= c.slots) slot = -1;
  if (slot < 0) {
    if ((const void*)x == (const void*)y) return;
    for (int v = lo + tid * 8; v < hi; v += kLcThreads * 8) {
      if (v + 8 <= hi) {
        float f[8];
        lc_load(x + v, f, vin);
        lc_store(y + v, f, vout);
      } else {
        for (int j = v; j < hi; ++j) {
          if constexpr (sizeof(TI) == 2 && sizeof(TO) == 2) y[j] = x[j];
          else if constexpr (sizeof(TI) == 2) y[j] = bf2f(x[j]);
          else y[j] = x[j];
        }
      }
    }
    return;
  }
  for (int i = tid * 4; i < chunk; i += kLcThreads * 4) *reinterpret_cast<uint4*>(s_word + i) = make_uint4(0, 0, 0, 0);
  __syncthreads();
  // the bias entries first: of several with one token the first counts, the largest n_bias - j
  const int* bi = c.bias_ids + (long)slot * c.n_bias;
  for (int j = tid; j < c.n_bias; j += kLcThreads) {
    const int v = bi[j];
    if (v >= lo && v < hi) atomicMax(&s_word[v - lo], (uint32_t)(c.n_bias - j) << kLcBias);
  }
  __syncthreads();
  const int len = min(c.lens[b], c.table_width * 16), prompt = c.info[2 * slot];
  const int* bt = c.table + (long)b * c.table_stride;
  for (int t = tid * 4; t < len; t += kLcThreads * 4) {
    const int page = bt[t >> 4];
    if (page < 0 || page >= c.pages) continue;
    const int4 q = *reinterpret_cast<const int4*>(c.tokens + (long)page * 16 + (t & 15));
    const int id[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (t + j < len && id[j] >= lo && id[j] < hi) {
        if (t + j < prompt) atomicOr(&s_word[id[j] - lo], kLcPrompt);
        else atomicAdd(&s_word[id[j] - lo], 1u);
      }
  }
  __syncthreads();
  const float rep = c.params[3 * slot], pres = c.params[3 * slot + 1], freq = c.params[3 * slot + 2];
  const bool masked = c.info[2 * slot + 1] != 0;
  const uint32_t* mask = c.masks + (long)slot * c.words;
  const float* bv = c.bias_vals + (long)slot * c.n_bias;
  auto one = [&](float f, uint32_t w) {
    const float count = (float)(w & kLcCount);
    if (w & (kLcPrompt | kLcCount)) f = f > 0.f ? f / rep : f * rep;
    if (w & kLcCount) f = f - freq * count - pres;
    if (w >> kLcBias) f += bv[c.n_bias - (int)(w >> kLcBias)];
    return f;
  };
  for (int v = lo + tid * 8; v < hi; v += kLcThreads * 8) {
    const uint32_t ok = masked ? mask[v >> 5] >> (v & 31) : 0xffu;  // v is a multiple of 8
    if (v + 8 <= hi) {
      float f[8];
      lc_load(x + v, f, vin);
      const uint4 a = *reinterpret_cast<const uint4*>(s_word + v - lo), d = *reinterpret_cast<const uint4*>(s_word + v - lo + 4);
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, d.x, d.y, d.z, d.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (w[j]) f[j] = one(f[j], w[j]);
        if (!((ok >> j) & 1)) f[j] = -INFINITY;
      }
      lc_store(y + v, f, vout);
    } else {
      for (int j = v; j < hi; ++j) {
        float f;
        if constexpr (sizeof(TI) == 2) f = bf2f(x[j]);
        else f = x[j];
        const uint32_t w = s_word[j - lo];
        if (w) f = one(f, w);
        if (!((ok >> (j - v)) & 1)) f = -INFINITY;
        if constexpr (sizeof(TO) == 2) y[j] = f2bf(f);
        else y[j] = f;
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
  int parts = (V + 16383) / 16384;
  const int want = (512 + B - 1) / B, most = (V + 2047) / 2048;
  parts = parts > (want < most ? want : most) ? parts : (want < most ? want : most);
  const int chunk = ((V + parts - 1) / parts + 255) & ~255;
  parts = (V + chunk - 1) / chunk;
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
