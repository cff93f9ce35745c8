// Single-token attention over the 8-bit pages (kv8.h), split over the context.
//
//   scores  S[t][h]   = K[t][:] . Q[h][:]            A = K   (16 tokens x 32 dims per v_mfma_f32_16x16x32_bf16)
//   output  O^T[d][h] = sum_t V^T[d][t] P^T[t][h]    A = V^T (16 dims  x 32 tokens)
//
// Columns are the G <= 16 query heads of a kv head.  Codes become bf16 in registers, two to a v_cvt_scalef32_pk_bf16_fp8 with the
// page's scale in the instruction: exact, so the products are those of a bf16 cache that holds the rounded values.
//
// A wave takes 64 tokens = 4 pages a step: 16-byte loads only, 16 KB of codes at D = 128.  Score tile i's row r is token 4 i + (r & 3) of page
// r >> 2: a lane's k-group kg then holds page kg's tokens in order over the four tiles, which is what the PV operand wants beside V's natural
// 16-byte rows (page kg's 16 tokens of a dim = the k-group's 8 tokens of two MFMA steps).  Each lane so needs two scales a step, of
// page col >> 2 for K and of page kg for V.
// Two buffers a wave: step c + 2's loads fly while step c + 1 is multiplied; page numbers are fetched a turn earlier still.  (Three or four
// buffers, or eight waves a workgroup, were slower or the same: registers then halve the waves of a SIMD, or joins begin later.)
//
// Work: grid (S splits, Hkv, batch), four waves of 64 tokens a workgroup and step, running maximum and sum per wave; a sequence that
// fits one split is finished there, else fp32 partials are joined by the last split to arrive (a counter per sequence and kv head, data
// written through and read past the XCD's L2) or, without counters, by a second launch.
//
// FUSED (the decode step, D = 128): q, k and v of the new token are the sum of the qkv projection's split-K slabs, rounded to bf16, q and k
// rotated.  The split that holds the sequence's end rounds k and v to the page's codes, attends to them from registers and, when all its
// waves have read their pages, writes them; if the page's scale grows it rounds the earlier tokens' codes anew, for its own products too: the
// answer is that of the write and the attention one after the other.  (The rotation's products are rounded one by one here; rotations that fuse them into
// the sums, as rope_and_cache's does, give the next bf16 number now and then.)
//
// Bound by memory: 64 x ~1.7 k tokens, 8 kv heads, 231 MB: 43 us, 5.3 TB/s (the same kernel without its products 41 to 43; a large sum reads 6.0);
// 8 x 31 k tokens, 512 MB: 93 us; over the bf16 cache the first takes 79 us.  One sequence of 1.7 k tokens: 10 us, of one token 6.7,
// a launch that does nothing 3 to 4.
#include "kv8.h"

namespace k8sllm {

struct Kv8Decode {
  bf16_t* out;
  long out_stride;  // < 0: fragment-packed (common.h act_index)
  float *part_o, *part_ml;  // [B][Hq][S][D], [B][Hq][S][2]
  const bf16_t* q;
  long q_stride;
  uint8_t *k, *v;
  float* scales;
  const int* table;
  long table_stride;
  int table_width;
  const int* lens;
  int B, Hq, Hkv, G, S, pages;
  float scale_log2;
  int* ctr;  // [B][Hkv], zero between launches; nullptr: a second launch joins the splits
  // FUSED
  const float* slabs;  // [nslabs][B][(Hq + 2 Hkv) * D]
  int nslabs;
  const int* positions;
  const float* cos_sin;  // [max_pos][D]
  int max_pos;
  const int* slots;  // [B], < 0: no write; nullptr: none
};

constexpr int kStep = 64;   // tokens of a wave's step
constexpr int kChunk = 256;  // of a workgroup's

__device__ __forceinline__ void kv8_range(int n, int S, int split, int* c0, int* c1, int* valid) {
  const int chunks = (n + kChunk - 1) / kChunk;
  const int per = (chunks + S - 1) / S;
  *c0 = split * per;
  *c1 = min(chunks, *c0 + per);
  *valid = (chunks + per - 1) / per;
}

template <int D>
struct Kv8Tiles {  // a wave's step, as loaded
  u32x4 k[4][D / 64];
  u32x4 v[D / 16];
  float ks, vs;
};

// Joins the `valid` splits' partials of the heads of (b, kvh): weights in s_w [16][64], then every thread its (head, dim) items.
template <int D, bool PAST>
__device__ __forceinline__ void kv8_join(const Kv8Decode& a, int b, int kvh, int valid, float* s_w) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  auto get = [](const float* p) {
    if constexpr (PAST) return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    else return *p;
  };
  for (int h = wave; h < a.G; h += 4) {
    const long ph = ((long)b * a.Hq + kvh * a.G + h) * a.S;
    const float m = lane < valid ? get(a.part_ml + (ph + lane) * 2) : -1e30f, l = lane < valid ? get(a.part_ml + (ph + lane) * 2 + 1) : 0.f;
    const float mm = wave_max(m);
    const float w = lane < valid ? __builtin_amdgcn_exp2f(m - mm) : 0.f;
    const float lw = wave_sum(w * l);
    s_w[h * 64 + lane] = w / lw;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.G * D; i += 256) {
    const int h = i / D, d = i - h * D;
    const float* po = a.part_o + ((long)b * a.Hq + kvh * a.G + h) * a.S * D + d;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    int p = 0;
    for (; p + 4 <= valid; p += 4)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] += s_w[h * 64 + p + j] * get(po + (long)(p + j) * D);
    for (; p < valid; ++p) s[0] += s_w[h * 64 + p] * get(po + (long)p * D);
    a.out[act_index(b, (kvh * a.G + h) * D + d, a.out_stride)] = f2bf((s[0] + s[1]) + (s[2] + s[3]));
  }
}

template <int D, bool FUSED>
__global__ __launch_bounds__(256, 2) void kv8_decode_kernel(const Kv8Decode a) {
  constexpr int KD = D / 4, KS = D / 32, KW = D / 64, DT = D / 16;
  __shared__ float s_max[4][16], s_sum[4][16];
  __shared__ __attribute__((aligned(16))) float s_o[4][16][D + 4];  // + 4: the 16 heads' rows start in different banks
  __shared__ __attribute__((aligned(16))) bf16_t s_q[FUSED ? 16 : 1][D];
  __shared__ __attribute__((aligned(16))) bf16_t s_kv[FUSED ? 2 : 1][D];        // the new token's k, v
  __shared__ __attribute__((aligned(16))) uint8_t s_code[FUSED ? 2 : 1][D];    // its codes
  __shared__ int s_last;

  const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z, G = a.G;
  const int len = min(a.lens[b], a.table_width * kPage);
  // (asked for together: each would be a trip to memory of its own where it is used)
  int slot = FUSED && a.slots != nullptr ? a.slots[b] : -1;
  const int position = FUSED ? a.positions[b] : 0;
  if (len <= 0) {  // an empty row (a graph bucket's slack): zeros
    if (split == 0)
      for (int i = threadIdx.x; i < G * D; i += 256) a.out[act_index(b, kvh * G * D + i, a.out_stride)] = 0;
    return;
  }
  int c0, c1, valid;
  kv8_range(len, a.S, split, &c0, &c1, &valid);
  if (c0 >= c1) return;  // uniform
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int col = lane & 15, kg = lane >> 4;
  const int cached = FUSED ? len - 1 : len;
  const bool owns_new = FUSED && c1 == (len + kChunk - 1) / kChunk;
  const int* bt = a.table + (long)b * a.table_stride;
  const int last_page = (len - 1) >> 4;

  // page numbers of the wave's step: K's (page col >> 2) and V's (page kg).  Ones past the end are the last page's; those outside the
  // cache are held to its ends where they are used (here that would be waiting for them).
  auto pages_of = [&](int c, int* pk, int* pv) {
    const int p0 = (c * kChunk + wave * kStep) >> 4;
    *pk = bt[min(p0 + (col >> 2), last_page)];
    *pv = bt[min(p0 + kg, last_page)];
  };
  auto issue = [&](Kv8Tiles<D>& t, int c, int pk, int pv) {
    const bool real = c < c1;  // uniform
    const long kt = (long)min(max(pk, 0), a.pages - 1) * a.Hkv + kvh, vt = (long)min(max(pv, 0), a.pages - 1) * a.Hkv + kvh;
    t.ks = a.scales[kt * 2];
    t.vs = a.scales[vt * 2 + 1];
    const uint8_t* kp = a.k + kt * (kPage * D) + (real ? (kg * kPage + (col & 3)) * KD : 0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int w = 0; w < KW; ++w) t.k[i][w] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kp + 4 * i * KD + 16 * w));
    const uint8_t* vp = a.v + vt * (kPage * D) + (real ? col * kPage : 0);
#pragma unroll
    for (int d = 0; d < DT; ++d) t.v[d] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(vp + d * 16 * kPage));
  };
  bf16x8 qf[KS];
  const int hc = min(col, G - 1);
  if constexpr (!FUSED) {
    const bf16_t* qp = a.q + (long)b * a.q_stride + (long)(kvh * G + hc) * D + KD * kg;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const bf16x8*>(qp + 8 * s);
  }
  // FUSED: thread's item of the new token's row - 4 rotary pairs of a head: its first four slabs and angles are asked for ahead of the pages
  constexpr int HALF = D / 2, QP = HALF / 4;
  const int cols = (a.Hq + 2 * a.Hkv) * D, items = (G + 2) * QP;
  const long slab = (long)a.B * cols;
  const float *row = nullptr, *cs = nullptr;
  f32x4 early[FUSED ? 10 : 1];
  auto column = [&](int it) {
    const int h = it / QP;  // h < G: a query head, G: k, G + 1: v
    return (h < G ? kvh * G + h : h == G ? a.Hq + kvh : a.Hq + a.Hkv + kvh) * D + (it % QP) * 4;
  };
  auto ask = [&](int it) {
    const float* p = row + column(it);
    const float* q = cs + (it % QP) * 4;
    early[8] = *reinterpret_cast<const f32x4*>(q);
    early[9] = *reinterpret_cast<const f32x4*>(q + HALF);
#pragma unroll
    for (int z = 0; z < 4; ++z) {
      const float* pz = p + min(z, a.nslabs - 1) * slab;
      early[2 * z] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(pz));
      early[2 * z + 1] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(pz + HALF));
    }
  };
  if constexpr (FUSED) {
    row = a.slabs + (long)b * cols;
    cs = a.cos_sin + (long)min(max(position, 0), a.max_pos - 1) * D;
    ask(min((int)threadIdx.x, items - 1));
    __builtin_amdgcn_sched_barrier(0);
  }
  // Loads return in order and the compiler counts them, so every path through the loop issues the same ones: behind the last step all lanes
  // read one place of the last page.  A buffer's page numbers are asked for behind its data, a turn before they are used.
  Kv8Tiles<D> t0, t1;
  int k0, v0, k1, v1, kn, vn;
  pages_of(c0, &k0, &v0);
  pages_of(c0 + 1, &k1, &v1);
  pages_of(c0 + 2, &kn, &vn);
  issue(t0, c0, k0, v0);
  k0 = kn, v0 = vn;
  pages_of(c0 + 3, &kn, &vn);
  __builtin_amdgcn_sched_barrier(0);  // t0's loads stay ahead of t1's, here as in the loop
  issue(t1, c0 + 1, k1, v1);
  k1 = kn, v1 = vn;
  __builtin_amdgcn_sched_barrier(0);
  auto refill = [&](Kv8Tiles<D>& t, int c, int& pk, int& pv) {
    issue(t, c, pk, pv);
    pages_of(c + 2, &pk, &pv);
  };

  float k_old = 0.f, v_old = 0.f, k_new = 0.f, v_new = 0.f;
  if constexpr (FUSED) {
    if (slot >= a.pages * kPage) slot = -1;
    if (owns_new && slot >= 0 && (slot & (kPage - 1))) {
      const float* sp = a.scales + ((long)(slot >> 4) * a.Hkv + kvh) * 2;
      k_old = sp[0];
      v_old = sp[1];
    }
    for (int it = threadIdx.x; it < items; it += 256) {
      if (it >= 256) ask(it);
      const int h = it / QP, p = (it % QP) * 4;
      f32x4 x1 = {0.f, 0.f, 0.f, 0.f}, x2 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int z = 0; z < 4; ++z)
        if (z < a.nslabs) {
          x1 += early[2 * z];
          x2 += early[2 * z + 1];
        }
      for (int z = 4; z < a.nslabs; ++z) {
        const float* pz = row + column(it) + z * slab;
        x1 += __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(pz));
        x2 += __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(pz + HALF));
      }
      const f32x4 cc = early[8], ss = early[9];
      bf16_t* dst = h < G ? s_q[h] : s_kv[h - G];
      float lo[4], hi[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x = bf2f(f2bf(x1[j])), y = bf2f(f2bf(x2[j]));
        if (h <= G) {  // each product rounded by itself: the page's scale, a threshold on these, is then what elementwise code finds
          const float o1 = __fsub_rn(__fmul_rn(x, cc[j]), __fmul_rn(y, ss[j])), o2 = __fadd_rn(__fmul_rn(y, cc[j]), __fmul_rn(x, ss[j]));
          x = o1;
          y = o2;
        }
        lo[j] = x;
        hi[j] = y;
      }
      *reinterpret_cast<uint2*>(dst + p) = make_uint2(pack2(lo[0], lo[1]), pack2(lo[2], lo[3]));
      *reinterpret_cast<uint2*>(dst + HALF + p) = make_uint2(pack2(hi[0], hi[1]), pack2(hi[2], hi[3]));
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const bf16x8*>(&s_q[hc][KD * kg + 8 * s]);
    if (owns_new) {  // uniform: the new token's scales and codes, in every wave; wave 0 leaves what they stand for
      // lanes 0..31: 4 dims of k each, 32..63: of v
      const int d = (lane & 31) * 4;
      const uint2 raw = *reinterpret_cast<const uint2*>(&s_kv[lane >> 5][d]);
      const float x[4] = {lo_bf(raw.x), hi_bf(raw.x), lo_bf(raw.y), hi_bf(raw.y)};
      float m = fmaxf(fmaxf(kv8_finite(x[0]), kv8_finite(x[1])), fmaxf(kv8_finite(x[2]), kv8_finite(x[3])));
      const float mk = wave_max(lane < 32 ? m : 0.f), mv = wave_max(lane < 32 ? 0.f : m);
      k_new = fmaxf(kv8_scale(mk), k_old);
      v_new = fmaxf(kv8_scale(mv), v_old);
      const float s = lane < 32 ? k_new : v_new;
      const uint32_t w = kv8_codes(x[0], x[1], x[2], x[3], kv8_inverse(s));
      const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false), hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true);
      __syncthreads();
      if (wave == 0) {
        *reinterpret_cast<uint32_t*>(&s_code[lane >> 5][d]) = w;
        *reinterpret_cast<bf16x4*>(&s_kv[lane >> 5][d]) = bf16x4{lo[0], lo[1], hi[0], hi[1]};
      }
    }
  } else {  // q has arrived before the loop, whose first wait for it would else stand for every load in flight
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" ::"v"(qf[s]));
  }

  float m = -1e30f, l = 0.f;  // of head `col`
  f32x4 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto compute = [&](Kv8Tiles<D>& t, int c) {
    const int tok0 = c * kChunk + wave * kStep;
    const int left = cached - tok0;  // tokens of this step (uniform)
    f32x4 s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < KS; ++j)
        s[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv8_values(t.k[i][j >> 1][2 * (j & 1)], t.k[i][j >> 1][2 * (j & 1) + 1], t.ks), qf[j], s[i],
                                                       0, 0, 0);
    }
    if (left < kStep) {  // scores past the end leave, and so do the codes behind them: what a page holds there may be anything
      const int mine = left - 16 * kg;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[i][r] = 4 * i + r < mine ? s[i][r] : -INFINITY;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int w = 0; w < 4; ++w) t.v[d][w] &= kv8_below(mine, w);
      if (mine <= 0) t.vs = 1.f;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[i][r] *= a.scale_log2;
        mx = fmaxf(mx, s[i][r]);
      }
    mx = xor32_max_f(xor16_max(mx));
    const float mnew = fmaxf(m, mx), alpha = __builtin_amdgcn_exp2f(m - mnew);
    float ls = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[i][r] = __builtin_amdgcn_exp2f(s[i][r] - mnew);
        ls += s[i][r];
      }
    l = l * alpha + xor32_sum_f(xor16_sum(ls));
    m = mnew;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] *= alpha;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 p;  // probabilities as bf16, the sum above in fp32: half a bf16 step each, as over the bf16 cache
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = (__bf16)s[2 * h + (j >> 2)][j & 3];
#pragma unroll
      for (int d = 0; d < DT; ++d)
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv8_values(t.v[d][2 * h], t.v[d][2 * h + 1], t.vs), p, o[d], 0, 0, 0);
    }
  };
  // the new token's page has grown a scale: the earlier tokens count as what their codes will stand for
  const bool grew = FUSED && __builtin_amdgcn_readfirstlane(owns_new && k_old > 0.f && (k_new != k_old || v_new != v_old));
  auto renew = [&](Kv8Tiles<D>& t, int c) {
    const int p0 = (c * kChunk + wave * kStep) >> 4;
    if (p0 + (col >> 2) == last_page && k_new != k_old) {
      const float ratio = k_old * kv8_inverse(k_new);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int w = 0; w < KW; ++w)
#pragma unroll
          for (int j = 0; j < 4; ++j) t.k[i][w][j] = kv8_again(t.k[i][w][j], ratio);
      t.ks = k_new;
    }
    if (p0 + kg == last_page && v_new != v_old) {
      const float ratio = v_old * kv8_inverse(v_new);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) t.v[d][j] = kv8_again(t.v[d][j], ratio);
      t.vs = v_new;
    }
  };
  int c = c0;
  for (; c + 1 < c1; c += 2) {  // (no way out in the middle: it would join the loop's head with fewer loads behind it)
    compute(t0, c);
    refill(t0, c + 2, k0, v0);
    __builtin_amdgcn_sched_barrier(0);
    if (FUSED && grew && c + 2 == c1) renew(t1, c + 1);
    compute(t1, c + 1);
    refill(t1, c + 3, k1, v1);
    __builtin_amdgcn_sched_barrier(0);
  }
  if (c < c1) {
    if (FUSED && grew) renew(t0, c);
    compute(t0, c);
  }

  if constexpr (FUSED) {
    if (owns_new && wave == 0) {  // the new token, from the numbers that its codes stand for (this wave wrote them)
      float sc = 0.f;
#pragma unroll 8
      for (int j = 0; j < KD; ++j) sc += bf2f(s_q[hc][kg * KD + j]) * bf2f(s_kv[0][kg * KD + j]);
      sc = xor32_sum_f(xor16_sum(sc)) * a.scale_log2;
      const float mnew = fmaxf(m, sc), alpha = __builtin_amdgcn_exp2f(m - mnew);
      const float e = __builtin_amdgcn_exp2f(sc - mnew), p = bf2f(f2bf(e));
      l = l * alpha + e;
      m = mnew;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[d][r] = o[d][r] * alpha + p * bf2f(s_kv[1][16 * d + 4 * kg + r]);
    }
  }

  // ---- the four waves' results: o[dt][r] = O^T[16 dt + 4 kg + r][col]
  if (lane < 16) {
    s_max[wave][lane] = m;
    s_sum[wave][lane] = l;
  }
  if (col < G)
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(&s_o[wave][col][16 * d + 4 * kg]) = o[d];
  __syncthreads();
  if constexpr (FUSED) {
    if (owns_new && slot >= 0) {  // every wave has its pages in registers by now: the page may change
      const int off = slot & (kPage - 1), tid = threadIdx.x;
      const long tile = (long)(slot >> 4) * a.Hkv + kvh;
      uint8_t *kp = a.k + tile * (kPage * D), *vp = a.v + tile * (kPage * D);
      if (tid < 64) {
        const int tok = tid & 15, run = tid >> 4;
        uint8_t* p = kp + (run * kPage + tok) * KD;
        if (tok == off) {
#pragma unroll
          for (int j = 0; j < KD; j += 16) *reinterpret_cast<u32x4*>(p + j) = *reinterpret_cast<const u32x4*>(&s_code[0][run * KD + j]);
        } else if (tok < off && k_new != k_old) {
          const float ratio = k_old * kv8_inverse(k_new);
#pragma unroll
          for (int j = 0; j < KD; j += 16) {
            u32x4 w = *reinterpret_cast<const u32x4*>(p + j);
#pragma unroll
            for (int q = 0; q < 4; ++q) w[q] = kv8_again(w[q], ratio);
            *reinterpret_cast<u32x4*>(p + j) = w;
          }
        }
        if (tid == 0) *reinterpret_cast<f32x2*>(a.scales + tile * 2) = f32x2{k_new, v_new};
      } else if (tid >= 128 && tid < 128 + D) {
        const int d = tid - 128;
        uint8_t* p = vp + d * kPage;
        if (off && v_new != v_old) {
          const float ratio = v_old * kv8_inverse(v_new);
          const u32x4 had = *reinterpret_cast<const u32x4*>(p);
          u32x4 w;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t before = kv8_below(off, q);
            w[q] = (kv8_again(had[q], ratio) & before) | (had[q] & ~before);
            if (q == off >> 2) w[q] = (w[q] & ~(0xffu << (8 * (off & 3)))) | ((uint32_t)s_code[1][d] << (8 * (off & 3)));
          }
          *reinterpret_cast<u32x4*>(p) = w;
        } else {
          p[off] = s_code[1][d];
        }
      }
    }
  }
  const bool merge = a.ctr != nullptr;
  for (int i = threadIdx.x; i < G * D; i += 256) {
    const int h = i / D, d = i - h * D;
    const float M = fmaxf(fmaxf(s_max[0][h], s_max[1][h]), fmaxf(s_max[2][h], s_max[3][h]));
    float acc = 0.f, L = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float e = __builtin_amdgcn_exp2f(s_max[w][h] - M);
      acc += e * s_o[w][h][d];
      L += e * s_sum[w][h];
    }
    if (valid == 1) {
      a.out[act_index(b, (kvh * G + h) * D + d, a.out_stride)] = f2bf(acc / L);
    } else {
      const long ph = ((long)b * a.Hq + kvh * G + h) * a.S + split;
      if (merge) {  // written through: another workgroup of this launch, maybe on another XCD, reads them
        __hip_atomic_store(a.part_o + ph * D + d, acc, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (d == 0) {
          __hip_atomic_store(a.part_ml + ph * 2, M, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          __hip_atomic_store(a.part_ml + ph * 2 + 1, L, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
      } else {
        a.part_o[ph * D + d] = acc;
        if (d == 0) {
          a.part_ml[ph * 2] = M;
          a.part_ml[ph * 2 + 1] = L;
        }
      }
    }
  }
  if (!merge || valid == 1) return;  // uniform
  // every wave's stores are out, then one lane takes a ticket; the last one joins and leaves the counter at zero
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    int* c = a.ctr + (long)b * gridDim.y + kvh;
    const int last = __hip_atomic_fetch_add(c, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == valid - 1;
    if (last) __hip_atomic_store(c, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = last;
  }
  __syncthreads();
  if (s_last) kv8_join<D, true>(a, b, kvh, valid, &s_o[0][0][0]);
}

// without counters: one workgroup per (kv head, sequence)
template <int D>
__global__ __launch_bounds__(256) void kv8_join_kernel(const Kv8Decode a) {
  __shared__ float s_w[16 * 64];
  const int kvh = blockIdx.x, b = blockIdx.y;
  const int len = min(a.lens[b], a.table_width * kPage);
  if (len <= 0) return;
  int c0, c1, valid;
  kv8_range(len, a.S, 0, &c0, &c1, &valid);
  if (valid > 1) kv8_join<D, false>(a, b, kvh, valid, s_w);
}

}  // namespace k8sllm

using namespace k8sllm;

// slabs != nullptr: the fused form (D = 128)
extern "C" int k8sllm_kv8_decode(void* out, long out_stride, float* part_o, float* part_ml, const void* q, long q_stride, void* k, void* v,
                                 float* scales, int pages, const int* table, long table_stride, int table_width, const int* lens, int B, int Hq,
                                 int Hkv, int D, int S, float scale, int* ctr, const float* slabs, int nslabs, const int* positions,
                                 const float* cos_sin, int max_pos, const int* slots, hipStream_t s) {
  if (B <= 0) return 0;
  const int G = Hq / Hkv;
  if (S < 1 || S > 64 || G < 1 || G > 16 || Hq % Hkv) return -2;
  const Kv8Decode a{(bf16_t*)out, out_stride, part_o, part_ml, (const bf16_t*)q, q_stride, (uint8_t*)k, (uint8_t*)v, scales, table, table_stride,
                    table_width, lens, B, Hq, Hkv, G, S, pages, scale * 1.4426950408889634f, S > 1 ? ctr : nullptr, slabs, nslabs, positions,
                    cos_sin, max_pos, slots};
  const dim3 grid(S, Hkv, B), block(256);
  if (slabs != nullptr) {
    if (D != 128) return -1;
    hipLaunchKernelGGL((kv8_decode_kernel<128, true>), grid, block, 0, s, a);
  } else if (D == 128) {
    hipLaunchKernelGGL((kv8_decode_kernel<128, false>), grid, block, 0, s, a);
  } else if (D == 64) {
    hipLaunchKernelGGL((kv8_decode_kernel<64, false>), grid, block, 0, s, a);
  } else {
    return -1;
  }
  if (S > 1 && ctr == nullptr) {
    if (D == 128)
      hipLaunchKernelGGL((kv8_join_kernel<128>), dim3(Hkv, B), block, 0, s, a);
    else
      hipLaunchKernelGGL((kv8_join_kernel<64>), dim3(Hkv, B), block, 0, s, a);
  }
  return (int)hipGetLastError();
}
