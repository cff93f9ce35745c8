// New tokens' keys and values into the 8-bit pages (kv8.h).
//
// One wave per (window of W rows, kv head).  It owns the runs that start in its window - a run: rows whose slots follow one another inside one
// page, at most 16 - and holds such a run whole in registers (keys: a lane has one token's D / 4 dims, values: a lane has D / 64 dims of
// all 16 tokens, so that both leave in 16-byte stores and V needs no transposing through LDS), which is what the scale, a maximum over
// the run, asks for.  The rows of a call that belong to one page follow one another; a run that starts inside a page finds that
// page's scale and earlier tokens, whose codes are rounded anew if the scale grows.
//
// Bound by memory at prefill: per row and kv head 4 D bytes in, 2 D out.
#include "kv8.h"

namespace k8sllm {

template <int D, int W>
__global__ __launch_bounds__(256) void kv8_write_kernel(const bf16_t* __restrict__ qkv, long stride, const int* __restrict__ slots,
                                                        uint8_t* __restrict__ k_codes, uint8_t* __restrict__ v_codes,
                                                        float* __restrict__ scales, int T, int Hq, int Hkv, int pages) {
  constexpr int KD = D / 4;    // dims a lane holds of a key
  constexpr int VD = D / 64;   // dims a lane holds of the values
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int t0 = (blockIdx.x * 4 + wave) * W, h = blockIdx.y;
  if (t0 >= T) return;
  // lane l: the slot of row t0 - 1 + l
  const int at = t0 - 1 + lane;
  const int mine = lane < W + 17 && at >= 0 && at < T ? slots[at] : -1;
  for (int i = 0; i < W; ++i) {
    const int slot = __builtin_amdgcn_readlane(mine, i + 1);
    if (slot < 0) continue;
    const int off = slot & (kPage - 1), page = slot >> 4;
    if ((off != 0 && __builtin_amdgcn_readlane(mine, i) == slot - 1) || page >= pages) continue;  // inside a run, or no such page
    const uint64_t next = __builtin_amdgcn_ballot_w64(mine == slot + (lane - i - 1)) >> (i + 1);
    const int len = min(kPage - off, (int)__builtin_ctzll(~next));
    const bf16_t* row = qkv + (long)(t0 + i) * stride;
    const long tile = ((long)page * Hkv + h);

    // keys: lane = (token, run of dims)
    const int tok = lane & 15, kg = lane >> 4, r = tok - off;
    const bool in = r >= 0 && r < len;
    float kx[KD], amax = 0.f;
    {
      const bf16_t* p = row + (long)(in ? r : 0) * stride + (Hq + h) * D + kg * KD;
#pragma unroll
      for (int j = 0; j < KD; j += 8) unpack8(*reinterpret_cast<const uint4*>(p + j), kx + j);
#pragma unroll
      for (int j = 0; j < KD; ++j) amax = fmaxf(amax, in ? kv8_finite(kx[j]) : 0.f);
    }
    // values: lane = dims VD * lane .., every token of the page
    float vx[VD][kPage], vmax = 0.f;
    {
      const bf16_t* p = row + (Hq + Hkv + h) * D + VD * lane;
#pragma unroll
      for (int t = 0; t < kPage; ++t) {
        const bool have = t >= off && t < off + len;  // uniform
        if constexpr (VD == 2) {
          const uint32_t w = have ? *reinterpret_cast<const uint32_t*>(p + (long)(t - off) * stride) : 0u;
          vx[0][t] = lo_bf(w);
          vx[1][t] = hi_bf(w);
          vmax = fmaxf(vmax, fmaxf(kv8_finite(vx[0][t]), kv8_finite(vx[1][t])));
        } else {
          vx[0][t] = have ? bf2f(p[(long)(t - off) * stride]) : 0.f;
          vmax = fmaxf(vmax, kv8_finite(vx[0][t]));
        }
      }
    }
    float* sp = scales + tile * 2;
    const float k_old = off ? sp[0] : 0.f, v_old = off ? sp[1] : 0.f;
    const float ks = fmaxf(kv8_scale(wave_max(amax)), k_old), vs = fmaxf(kv8_scale(wave_max(vmax)), v_old);

    uint8_t* kp = k_codes + tile * (kPage * D) + (kg * kPage + tok) * KD;
    if (in) {
      const float inv = kv8_inverse(ks);
#pragma unroll
      for (int j = 0; j < KD; j += 16) {
        u32x4 w;
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = kv8_codes(kx[j + 4 * q], kx[j + 4 * q + 1], kx[j + 4 * q + 2], kx[j + 4 * q + 3], inv);
        *reinterpret_cast<u32x4*>(kp + j) = w;
      }
    } else if (tok < off && ks != k_old) {
      const float ratio = k_old * kv8_inverse(ks);
#pragma unroll
      for (int j = 0; j < KD; j += 16) {
        u32x4 w = *reinterpret_cast<const u32x4*>(kp + j);
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = kv8_again(w[q], ratio);
        *reinterpret_cast<u32x4*>(kp + j) = w;
      }
    }
    uint8_t* vp = v_codes + tile * (kPage * D) + (long)VD * lane * kPage;
    const float inv = kv8_inverse(vs), ratio = v_old * inv;
    const bool whole = off == 0 && len == kPage;  // uniform
#pragma unroll
    for (int d = 0; d < VD; ++d) {
      u32x4 w;
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = kv8_codes(vx[d][4 * q], vx[d][4 * q + 1], vx[d][4 * q + 2], vx[d][4 * q + 3], inv);
      if (!whole) {  // what the page held: earlier tokens, and whatever lies behind the run
        const u32x4 had = *reinterpret_cast<const u32x4*>(vp + d * kPage);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t before = kv8_below(off, q), upto = kv8_below(off + len, q);
          const uint32_t again = vs != v_old ? kv8_again(had[q], ratio) : had[q];
          w[q] = (again & before) | (w[q] & upto & ~before) | (had[q] & ~upto);
        }
      }
      *reinterpret_cast<u32x4*>(vp + d * kPage) = w;
    }
    if (lane == 0) *reinterpret_cast<f32x2*>(sp) = f32x2{ks, vs};
  }
}

}  // namespace k8sllm

using namespace k8sllm;

extern "C" int k8sllm_kv8_write(const void* qkv, long stride, const int* slots, void* k, void* v, float* scales, int T, int Hq, int Hkv, int D,
                                int pages, hipStream_t s) {
  if (T <= 0) return 0;
  const bool few = T <= 512;
  const int W = few ? 1 : 4;
  const dim3 grid((unsigned)((T + 4 * W - 1) / (4 * W)), (unsigned)Hkv);
#define K8S_KV8W(DD, WW)                                                                                                       \
  hipLaunchKernelGGL((kv8_write_kernel<DD, WW>), grid, dim3(256), 0, s, (const bf16_t*)qkv, stride, slots, (uint8_t*)k, (uint8_t*)v, scales, \
                     T, Hq, Hkv, pages)
  if (D == 128) {
    if (few) K8S_KV8W(128, 1); else K8S_KV8W(128, 4);
  } else if (D == 64) {
    if (few) K8S_KV8W(64, 1); else K8S_KV8W(64, 4);
  } else {
    return -1;
  }
#undef K8S_KV8W
  return (int)hipGetLastError();
}
