// New tokens' keys and values into the 8-bit pages (kv8.h).
//
// One wave per (window of W rows, kv head).  It owns the runs that start in its window - a run: rows whose slots follow one another inside one
// page, at most 16 - and holds such a run whole in registers, which is what the scale, a maximum over the run, asks for: keys 8 dims of a token
// a lane, whole rows to a load; values D / 64 dims of all 16 tokens a lane, so that a dim's 16 codes leave in one store without a
// transpose through LDS.  The rows of a call that belong to one page follow one another; a run that starts inside a page finds that
// page's scale and earlier tokens, whose codes are rounded anew if the scale grows.
//
// Magnitudes are compared as the 16-bit patterns that they are, two to an instruction, and v_cvt_scalef32_pk_fp8_bf16 takes packed bf16 and the
// scale: about 130 instructions a run (in 32-bit arithmetic 1000, which took longer than the memory: 28 us for the figure below).
// Bound by memory at prefill: per row and kv head 4 D bytes in, 2 D out; 16 k rows x 8 heads x 128 dims, 98 MB: 19.3 us, 5.1 TB/s (a large copy
// moves 5.1).
#include "kv8.h"

namespace k8sllm {

template <int D, int W>
__global__ __launch_bounds__(256) void kv8_write_kernel(const bf16_t* __restrict__ qkv, long stride, const int* __restrict__ slots,
                                                        uint8_t* __restrict__ k_codes, uint8_t* __restrict__ v_codes,
                                                        float* __restrict__ scales, int T, int Hq, int Hkv, int pages) {
  constexpr int KP = D / 8, KT = 64 / KP, KN = kPage / KT;  // keys: 8-dim pieces of a token, tokens at a time, times
  constexpr int RP = KP / 4;                                // pieces of a run of dims
  constexpr int VD = D / 64;                                // dims a lane holds of the values
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  // neighbouring waves: neighbouring heads of the same rows
  const int unit = blockIdx.x * 4 + wave, t0 = unit / Hkv * W, h = unit % Hkv;
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

    // keys: lane = 8 dims of a token, KT tokens at a time.  Places outside the run hold one of its rows (which changes no maximum).
    const int piece = lane % KP;
    uint4 kx[KN];
#pragma unroll
    for (int n = 0; n < KN; ++n) {
      const int r = min(max(n * KT + lane / KP - off, 0), len - 1);
      kx[n] = *reinterpret_cast<const uint4*>(row + (long)r * stride + (Hq + h) * D + piece * 8);
    }
    // values: lane = dims VD * lane .., every token of the page; packed in pairs, D = 128: two dims, D = 64: one and zero
    uint32_t vx[kPage];
    {
      const bf16_t* p = row + (Hq + Hkv + h) * D + VD * lane;
#pragma unroll
      for (int t = 0; t < kPage; ++t) {
        const bf16_t* pt = p + (long)min(max(t - off, 0), len - 1) * stride;
        if constexpr (VD == 2) vx[t] = *reinterpret_cast<const uint32_t*>(pt);
        else vx[t] = *pt;
      }
    }
    // magnitudes as 16-bit patterns, two at a time; one that is not finite sends the wave the long way
    uint32_t km = 0, vm = 0;
#pragma unroll
    for (int n = 0; n < KN; ++n) km = kv8_max_bits(kv8_max_bits(kv8_max_bits(kv8_max_bits(km, kx[n].x), kx[n].y), kx[n].z), kx[n].w);
#pragma unroll
    for (int t = 0; t < kPage; ++t) vm = kv8_max_bits(vm, vx[t]);
    const uint32_t both = kv8_max_bits(km, vm);
    if (__builtin_amdgcn_ballot_w64((both & 0xffffu) >= 0x7f80u || both >= 0x7f800000u)) {
      km = vm = 0;
#pragma unroll
      for (int n = 0; n < KN; ++n)
        km = kv8_max_bits(kv8_max_bits(kv8_max_bits(kv8_max_bits(km, kv8_finite_bits(kx[n].x)), kv8_finite_bits(kx[n].y)), kv8_finite_bits(kx[n].z)),
                          kv8_finite_bits(kx[n].w));
#pragma unroll
      for (int t = 0; t < kPage; ++t) vm = kv8_max_bits(vm, kv8_finite_bits(vx[t]));
    }
    const float amax = fmaxf(lo_bf(km), hi_bf(km)), vmax = fmaxf(lo_bf(vm), hi_bf(vm));
    float* sp = scales + tile * 2;
    const float k_old = off ? sp[0] : 0.f, v_old = off ? sp[1] : 0.f;
    const float ks = fmaxf(kv8_scale(wave_max(amax)), k_old), vs = fmaxf(kv8_scale(wave_max(vmax)), v_old);

    uint8_t* kp = k_codes + tile * (kPage * D) + (piece / RP) * (kPage * RP * 8) + (piece % RP) * 8;
    const float k_ratio = k_old * kv8_inverse(ks);
#pragma unroll
    for (int n = 0; n < KN; ++n) {
      const int tok = n * KT + lane / KP, r = tok - off;
      uint2* dst = reinterpret_cast<uint2*>(kp + tok * (RP * 8));
      if (r >= 0 && r < len) {
        *dst = make_uint2(kv8_codes_bf16(kx[n].x, kx[n].y, ks), kv8_codes_bf16(kx[n].z, kx[n].w, ks));
      } else if (r < 0 && ks != k_old) {
        const uint2 had = *dst;
        *dst = make_uint2(kv8_again(had.x, k_ratio), kv8_again(had.y, k_ratio));
      }
    }
    uint8_t* vp = v_codes + tile * (kPage * D) + (long)VD * lane * kPage;
    const float v_ratio = v_old * kv8_inverse(vs);
    const bool whole = off == 0 && len == kPage;  // uniform
#pragma unroll
    for (int d = 0; d < VD; ++d) {
      u32x4 w;
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // tokens 4 q .. 4 q + 3 of the dim: its halves of two words each
        const uint32_t half = d ? 0x07060302u : 0x05040100u;
        w[q] = kv8_codes_bf16(__builtin_amdgcn_perm(vx[4 * q + 1], vx[4 * q], half), __builtin_amdgcn_perm(vx[4 * q + 3], vx[4 * q + 2], half), vs);
      }
      if (!whole) {  // what the page held: earlier tokens, and whatever lies behind the run
        const u32x4 had = *reinterpret_cast<const u32x4*>(vp + d * kPage);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t before = kv8_below(off, q), upto = kv8_below(off + len, q);
          const uint32_t again = vs != v_old ? kv8_again(had[q], v_ratio) : had[q];
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
  // rows a wave: few rows are sequences' next tokens as often as not, each a run of its own (W = 2, 40 rows: 3.9 us, 16: 7.0); many are
  // prompts, whose runs are 16 long, and waves that own none still cost their dispatch (16384 rows: W = 2 70 us, 8 27.6, 16 20.9;
  // 2048 rows: 8 6.5, 16 7.5)
  const int W = T <= 512 ? 2 : T <= 4096 ? 8 : 16;
  const dim3 grid((unsigned)(((long)((T + W - 1) / W) * Hkv + 3) / 4));
#define K8S_KV8W(DD, WW)                                                                                                       \
  hipLaunchKernelGGL((kv8_write_kernel<DD, WW>), grid, dim3(256), 0, s, (const bf16_t*)qkv, stride, slots, (uint8_t*)k, (uint8_t*)v, scales, \
                     T, Hq, Hkv, pages)
#define K8S_KV8W_D(DD)                                                                    \
  if (W == 2) K8S_KV8W(DD, 2); else if (W == 8) K8S_KV8W(DD, 8); else K8S_KV8W(DD, 16)
  if (D == 128) {
    K8S_KV8W_D(128);
  } else if (D == 64) {
    K8S_KV8W_D(64);
  } else {
    return -1;
  }
#undef K8S_KV8W_D
#undef K8S_KV8W
  return (int)hipGetLastError();
}
