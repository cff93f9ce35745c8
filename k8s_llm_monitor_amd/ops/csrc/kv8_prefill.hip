// Causal attention of prompt chunks over the 8-bit pages (kv8.h): the queries are the new rows of the qkv buffer, all keys and values
// - what came before and the chunk itself, whole prompts too - are read from the pages, so that a prompt's answer does not depend on where it was cut
// (but for codes that become subnormal where a later chunk makes a page's scale grow) nor on what else is in the step.
//
// A workgroup takes one kv head and 256 (query row, head of the group) pairs, pair f = row * G + g, 32 to a wave: any group size fills
// the 32-column MFMAs, and the heads of a row share every K / V tile.  Products are in the swapped orientation
//   S^T[key][pair] = K Q^T,   O^T[dim][pair] += V^T P^T
// so running maximum, sum and the accumulator's rescale are lane-local but for one exchange of the wave's halves, and the score
// accumulator, rounded to bf16, is the second product's operand in place.
//
// Scores are v_mfma_scale_f32_32x32x64_f8f6f4 on the codes as they lie, with the page's scale as the operand's: K is staged without a
// conversion and read from LDS at half the bytes.  q is the sum of two e4m3 numbers (see there), so nothing of bf16's precision is lost; two
// products at twice the rate cost what one in bf16 does.  (In bf16, K converted on its way: 908 us for the first figure below, 835 so.)
// Probabilities as two e4m3 numbers would spare V's conversion but cost more in vector instructions than it does.
//
// Tiles of 64 keys (4 pages).  A thread loads 16 bytes of K codes and 16 of V codes a tile, a tile ahead of their way into LDS, where V
// becomes bf16 (8 conversions of two codes each, with the page's scale in them: exact); done by each wave for itself behind LDS it would be eight times
// that.  Staging goes between the wave's score products.  Four buffers of 24 KB (D = 128) and a barrier every other tile: waves drift apart by
// up to two tiles, and the second half of a tile - exponentials and the second product, both units at work - has priority over another
// wave's first, so that the two waves of a SIMD are in different halves more often than not (a barrier a tile, or no priority: 828 and
// 835 us for 807).  No unit alone bounds it: MFMAs are busy 56 % of the time and the vector
// units 61 %, LDS conflicts are 5 % (counters, 4096 rows behind 12 k).
//
// A V code that is NaN counts for rows that see its token and no others, though all rows of a tile multiply it (0 * NaN): the tile is
// staged with zero in its place, and the first such token of each dim is kept and put on the rows behind it at the end.
//
// Few rows (a short question behind a long conversation) leave most of the chip idle: the keys are then split S ways and fp32 partials
// joined by a second launch.
//
// Measured: 4096 rows behind 12 k tokens, 32 heads over 8: 807 to 859 us on two boxes, 1.12 to 1.19 PFLOP/s (a large bf16 library product: 1.36); 10 x up to 1124 rows
// behind 512: 222 to 234 us, 0.76 to 0.81; 45 rows behind 4 k tokens: 23 us.
#include <algorithm>

#include "kv8.h"

namespace k8sllm {

struct Kv8Prefill {
  bf16_t* out;
  long out_stride;
  const bf16_t* qkv;
  long qkv_stride;
  const int *cu, *ctx, *qb_seq, *qb_start;
  const uint8_t *k, *v;
  const float* scales;
  int pages;
  const int* table;
  long table_stride;
  int table_width, rows, seqs, Hq, Hkv, G, Z, S;
  float scale_log2;
  float *part_o, *part_ml;  // [S][rows][Hq][D], [S][rows][Hq][2]
};

constexpr int kTile = 64;
typedef int i32x8 __attribute__((ext_vector_type(8)));

template <int D>
__global__ __launch_bounds__(512, 2) void kv8_prefill_kernel(const Kv8Prefill a) {
  constexpr int KS = D / 64, DT = D / 32, KD = D / 4;
  constexpr int kHalf = kTile * D;  // elements of a K (or V) tile
  __shared__ __attribute__((aligned(16))) uint8_t s_k[4][kHalf];  // [4 pages][4 runs][16 tokens][D / 4], codes
  __shared__ uint32_t s_kscale[4][4];                             // the pages' scales as e8m0
  __shared__ __attribute__((aligned(16))) bf16_t s_v[4][kHalf];  // [4 pages][D][2 chunks of 8 tokens]
  __shared__ int s_nan[D];  // first token whose V code is NaN

  const int kvh = blockIdx.x, qb = blockIdx.y / a.Z, G = a.G;
  const int seq = a.qb_seq[qb];
  if (seq < 0 || seq >= a.seqs) return;
  const int qs = a.qb_start[qb], s0 = a.cu[seq], L = a.cu[seq + 1] - s0;
  const int pairs = min(128, L - qs) * G, f0 = (blockIdx.y % a.Z) * 256;
  if (qs < 0 || f0 >= pairs || s0 < 0 || s0 + L > a.rows) return;  // uniform
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, hh = lane >> 5;
  const int cst = __builtin_amdgcn_readfirstlane(max(0, min(a.ctx[seq], a.table_width * kPage - L)));  // keys never pass the table
  const int LK = min(cst + L, a.table_width * kPage), last_page = (LK - 1) >> 4;  // (a chunk longer than the table: its last rows see all of it)
  const int f = f0 + 32 * wave + r32;
  const bool mine = f < pairs;
  const int row = qs + (mine ? f / G : 0), hq = kvh * G + (mine ? f % G : 0);
  // (divisions are done in vector registers: what branches hang on goes back to scalar ones)
  const int wave_first = __builtin_amdgcn_readfirstlane(min(cst + qs + (f0 + 32 * wave) / G, LK - 1));  // the last key that the wave's first row sees
  const bool busy = f0 + 32 * wave < pairs;
  const int wave_last = cst + qs + (min(pairs, f0 + 32 * wave + 32) - 1) / G;
  const int tiles = (cst + qs + (min(pairs, f0 + 256) - 1) / G) / kTile + 1;
  const int per = (tiles + a.S - 1) / a.S;
  const int tb = __builtin_amdgcn_readfirstlane(blockIdx.z * per), te = __builtin_amdgcn_readfirstlane(min(tiles, tb + per));
  const int nt = __builtin_amdgcn_readfirstlane(busy ? min(te, wave_last / kTile + 1) : 0);  // the wave's tiles end here

  for (int i = tid; i < D; i += 512) s_nan[i] = 0x7fffffff;

  // ---- staging: thread = (page of the tile, 16 bytes of it); D = 128: all threads K and V, D = 64: the lower half K, the upper V
  constexpr bool BOTH = D == 128;
  const int piece = BOTH ? tid : tid & 255;
  const bool has_k = BOTH || wave < 4, has_v = BOTH || wave >= 4;  // uniform in a wave
  const int pg = piece / (D);  // page of the tile: D pieces of 16 bytes a page
  const int in = piece & (D - 1);
  // K piece: [run][half of its dims, D = 128][token]; the halves of a token's run change places from its eighth token on, so that sixteen lanes'
  // reads of one half meet all banks
  const int ktok = in & 15, kpart = in >> 4;  // 16-dim parts 0 .. D / 16 - 1: dims 16 kpart ..
  const int k_src = ((kpart * 16) / KD * kPage + ktok) * KD + (kpart * 16) % KD;
  int zero;  // in a vector register: page numbers and scales are loaded as vectors are, not by scalar loads, whose counter is LDS's
  asm("v_mov_b32 %0, 0" : "=v"(zero));
  const int* bt = a.table + (long)seq * a.table_stride + zero;
  auto page_of = [&](int t) { return min(max(bt[min(t * 4 + pg, last_page)], 0), a.pages - 1); };
  struct Raw {
    u32x4 k, v;
    float ks, vs;
  };
  auto fetch = [&](Raw& r, int page) {
    const long tile = (long)page * a.Hkv + kvh;
    if (has_k) r.k = *reinterpret_cast<const u32x4*>(a.k + tile * (kPage * D) + k_src);
    if (has_v) r.v = *reinterpret_cast<const u32x4*>(a.v + tile * (kPage * D) + in * kPage);
    r.ks = a.scales[tile * 2];
    r.vs = a.scales[tile * 2 + 1];
  };
  // Tile t's codes before they are converted: those behind the sequence's end, where a page holds anything, and NaN ones become zero
  auto settle = [&](Raw& r, int t) {
    if (!has_v) return;
    const int left = LK - (t * kTile + pg * kPage);
    if (__builtin_amdgcn_readfirstlane(left) < kPage) {
#pragma unroll
      for (int w = 0; w < 4; ++w) r.v[w] &= kv8_below(left, w);
      if (left <= 0) r.vs = 1.f;
    }
    uint32_t bad[4], any = 0;  // the high bit of each NaN code (0x7f, 0xff)
#pragma unroll
    for (int w = 0; w < 4; ++w) any |= bad[w] = ((r.v[w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    if (__builtin_amdgcn_ballot_w64(any != 0)) {
      if (any) {
        int first = 0;
#pragma unroll
        for (int w = 3; w >= 0; --w)
          if (bad[w]) first = 4 * w + (__builtin_ctz(bad[w]) >> 3);
        atomicMin(&s_nan[in], t * kTile + pg * kPage + first);
#pragma unroll
        for (int w = 0; w < 4; ++w) r.v[w] &= ~((bad[w] >> 7) * 0xffu);
      }
    }
  };
  auto stage = [&](const Raw& r, int t) {
    if (has_k) {
      *reinterpret_cast<u32x4*>(s_k[t & 3] + pg * (kPage * D) + (D == 128 ? k_src ^ ((ktok & 8) << 1) : k_src)) = r.k;
      if (in == 0) s_kscale[t & 3][pg] = __float_as_uint(r.ks) >> 23;
    }
    if (has_v) {
      // the 8 tokens of the accumulator's half hh: 0-3, 8-11 and 4-7, 12-15; the two chunks of a dim change places by its bit 3
      bf16_t* p = s_v[t & 3] + (pg * D + in) * 16;
      const int x = ((in >> 3) & 1) * 8;
      *reinterpret_cast<bf16x8*>(p + x) = kv8_values(r.v[0], r.v[2], r.vs);
      *reinterpret_cast<bf16x8*>(p + (8 - x)) = kv8_values(r.v[1], r.v[3], r.vs);
    }
  };

  // the first two tiles are on their way while q is prepared
  Raw r, r1;
  int next;
  {
    const int p0 = page_of(tb), p1 = page_of(tb + 1);
    next = page_of(tb + 2);
    fetch(r, p0);
    fetch(r1, p1);
  }

  // q as the sum of two e4m3 numbers, the second a sixteenth as large: a code's 4 bits and the 4 of what it leaves off are bf16's 8, so this
  // is q itself but for numbers below 2^-15 of the row's largest, which are off by 2^-22 of it
  i32x8 q_hi[KS], q_lo[KS];
  uint32_t qs_hi[KS];
  {
    const bf16_t* qp = a.qkv + (long)(s0 + row) * a.qkv_stride + hq * D + 32 * hh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      u32x4 x[4];
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = *reinterpret_cast<const u32x4*>(qp + 64 * ks + 8 * j);
#pragma unroll
        for (int w = 0; w < 4; ++w) m = kv8_max_bits(m, x[j][w]);
      }
      // (a row with infinities or NaN, which are NaN codes, answers NaN under any scale)
      const float amax = fminf(fmaxf(lo_bf(m), hi_bf(m)), 3.3895314e38f);
      const float sc = kv8_scale(xor32_max_f(amax)), sc_lo = sc * 0.0625f;
      qs_hi[ks] = __float_as_uint(sc) >> 23;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const uint32_t a0 = x[w >> 1][2 * (w & 1)], a1 = x[w >> 1][2 * (w & 1) + 1];
        const uint32_t hi = kv8_codes_bf16(a0, a1, sc);
        const f32x2 u = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, sc, false), v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, sc, true);
        s16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(s16x2{0, 0}, lo_bf(a0) - u[0], hi_bf(a0) - u[1], sc_lo, false);
        lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, lo_bf(a1) - v[0], hi_bf(a1) - v[1], sc_lo, true);
        q_hi[ks][w] = (int)hi;
        q_lo[ks][w] = __builtin_bit_cast(int, lo);
      }
    }
  }
  f32x16 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  float m = -1e30f, l = 0.f;

  // S^T of tile t, tile t + 2's conversions and LDS stores between its products: they are this wave's only other work then
  auto scores = [&](int t, f32x16 (&s)[2], Raw& r) {
    // key 32 i + r32: page 2 i + (r32 >> 4), token r32 & 15; dims 64 ks + 32 hh ..: runs of D / 4
    const uint8_t* kt = s_k[t & 3];
    i32x8 kf[KS][2];
    uint32_t sc[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int pg = 2 * i + (r32 >> 4), tok = r32 & 15;
      sc[i] = s_kscale[t & 3][pg];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const uint8_t* p = kt + pg * (kPage * D);
        u32x4 lo, hi;
        if constexpr (D == 128) {
          p += ((2 * ks + hh) * kPage + tok) * KD;
          const int x = (tok & 8) << 1;
          lo = *reinterpret_cast<const u32x4*>(p + x);
          hi = *reinterpret_cast<const u32x4*>(p + (16 - x));
        } else {
          p += (2 * hh * kPage + tok) * KD;
          lo = *reinterpret_cast<const u32x4*>(p);
          hi = *reinterpret_cast<const u32x4*>(p + kPage * KD);
        }
        kf[ks][i] = i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[i][r] = 0.f;
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" : "+v"(r.k), "+v"(r.v));  // (the conversions stay here and do not move ahead of the branch)
    stage(r, t + 2);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int part = 0; part < 2; ++part)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          s[i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kf[ks][i], part ? q_lo[ks] : q_hi[ks], s[i], 0, 0, 0, (int)sc[i], 0,
                                                                 (int)(part ? qs_hi[ks] - 4 : qs_hi[ks]));
    if constexpr (BOTH) {
#pragma unroll
      for (int n = 0; n < 4 * KS; ++n) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);    // a product
        __builtin_amdgcn_sched_group_barrier(0x2, 2, 0);    // vector instructions
        __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);  // an LDS store
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (t * kTile + kTile - 1 > wave_first) {  // keys past this lane's row (uniform branch)
      const int lim = min(cst + row, LK - 1) - t * kTile - 4 * hh;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[i][r] = 32 * i + (r & 3) + 8 * (r >> 2) > lim ? -INFINITY : s[i][r];
    }
  };
  auto products = [&](int t, f32x16 (&s)[2]) {
    const bf16_t* vt = s_v[t & 3];
    bf16x8 vf[2][2][DT];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const int dim = 32 * d + r32;
          vf[i][p][d] = *reinterpret_cast<const bf16x8*>(vt + ((2 * i + p) * D + dim) * 16 + (hh ^ ((dim >> 3) & 1)) * 8);
        }
    __builtin_amdgcn_sched_barrier(0);
    float mq[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      mq[c] = s[c >> 1][8 * (c & 1)];
#pragma unroll
      for (int r = 1; r < 8; ++r) mq[c] = fmaxf(mq[c], s[c >> 1][8 * (c & 1) + r]);
    }
    const float mt = xor32_max_f(fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3]))) * a.scale_log2;
    // the reference maximum moves only where a tile's passes it by 2^8: probabilities stay at most 256, the accumulator is rescaled rarely
    const float mnew = mt > m + 8.f ? mt : m;
    if (__builtin_amdgcn_ballot_w64(mnew != m) != 0) {
      const float alpha = __builtin_amdgcn_exp2f(m - mnew);
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
      m = mnew;
    }
    float rq[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        bf16x8 pb;  // probabilities rounded to bf16 for the product, summed in fp32
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][8 * p + j], a.scale_log2, -m));
          rq[2 * i + p] += e;
          pb[j] = (__bf16)e;
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[i][p][d], pb, o[d], 0, 0, 0);
      }
    l += xor32_sum_f((rq[0] + rq[1]) + (rq[2] + rq[3]));
  };

  if (tb < te) {
    __syncthreads();  // s_nan
    settle(r, tb);
    stage(r, tb);
    settle(r1, tb + 1);
    stage(r1, tb + 1);
    fetch(r, next);  // from here on r is the next tile to stage (behind the last one: later keys, or the last page again)
    next = page_of(tb + 3);
    for (int t = tb; t < te; ++t) {
      if (((t - tb) & 1) == 0) __syncthreads();
      settle(r, t + 2);
      if (t < nt) {
        f32x16 s[2];
        scores(t, s, r);
        fetch(r, next);
        next = page_of(t + 4);
        __builtin_amdgcn_s_setprio(1);
        products(t, s);
        __builtin_amdgcn_s_setprio(0);
      } else {
        stage(r, t + 2);
        fetch(r, next);
        next = page_of(t + 4);
      }
    }
    __syncthreads();  // s_nan
  }

  if (mine) {
    const int seen = cst + row;
    if (a.S > 1) {
      const long ph = ((long)blockIdx.z * a.rows + s0 + row) * a.Hq + hq;
      if (hh == 0) {
        a.part_ml[ph * 2] = m;
        a.part_ml[ph * 2 + 1] = l;
      }
      if (tb < te) {
        float* op = a.part_o + ph * D + 4 * hh;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            f32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = s_nan[32 * d + 8 * k + 4 * hh + j] <= seen ? __builtin_nanf("") : o[d][4 * k + j];
            *reinterpret_cast<f32x4*>(op + 32 * d + 8 * k) = v;
          }
      }
      return;
    }
    const float inv = 1.f / l;
    bf16_t* op = a.out + (long)(s0 + row) * a.out_stride + (long)hq * D + 4 * hh;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = s_nan[32 * d + 8 * k + 4 * hh + j] <= seen ? __builtin_nanf("") : o[d][4 * k + j] * inv;
        *reinterpret_cast<uint2*>(op + 32 * d + 8 * k) = make_uint2(pack2(x[0], x[1]), pack2(x[2], x[3]));
      }
  }
}

// Splits of (row, head), one wave each, of the rows that the q-blocks name.  Splits without a key for the row have l = 0 and hold nothing.
template <int D>
__global__ __launch_bounds__(256) void kv8_prefill_join_kernel(const Kv8Prefill a) {
  const int lane = threadIdx.x & 63, f = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int seq = a.qb_seq[blockIdx.y];
  if (seq < 0 || seq >= a.seqs) return;
  const int qs = a.qb_start[blockIdx.y], s0 = a.cu[seq], L = a.cu[seq + 1] - s0, row = qs + f / a.Hq;
  if (qs < 0 || f >= 128 * a.Hq || row >= L || s0 < 0 || s0 + L > a.rows) return;
  const long n = (long)a.rows * a.Hq, i = (long)(s0 + row) * a.Hq + f % a.Hq;
  const float m = lane < a.S ? a.part_ml[(lane * n + i) * 2] : -1e30f, l = lane < a.S ? a.part_ml[(lane * n + i) * 2 + 1] : 0.f;
  const float mm = wave_max(m);
  const float w = l != 0.f ? __builtin_amdgcn_exp2f(m - mm) : 0.f;
  const float inv = 1.f / wave_sum(w * l);
  const uint64_t have = __builtin_amdgcn_ballot_w64(l != 0.f);
  constexpr int E = D / 64;
  float acc[E] = {};
  for (int s = 0; s < a.S; ++s) {
    if (!((have >> s) & 1)) continue;
    const float ws = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), s));
    const float* p = a.part_o + (s * n + i) * D + E * lane;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += ws * p[e];
  }
  bf16_t* o = a.out + (i / a.Hq) * a.out_stride + (i % a.Hq) * D + E * lane;
  if constexpr (E == 2)
    *reinterpret_cast<uint32_t*>(o) = pack2(acc[0] * inv, acc[1] * inv);
  else
    o[0] = f2bf(acc[0] * inv);
}

}  // namespace k8sllm

using namespace k8sllm;

// Workgroups a q-block: no block has more rows than the call
static int prefill_z(int rows, int G) { return (std::min(128, rows) * G + 255) / 256; }

// How many ways the keys are split: where the rows make fewer than 256 workgroups, up to 32 splits of at least 4 tiles of the longest context
// that the block tables allow.  (A split's partials are 512 bytes a row and head out and in: 45 rows behind 4 k tokens, 32 heads: 16 splits
// of 5 tiles 17.5 + 4.0 us, 32 of 3 tiles 17.4 + 5.5.)
extern "C" int k8sllm_kv8_prefill_splits(int n_qblocks, int rows, int Hq, int Hkv, int table_width) {
  if (rows > 128L * n_qblocks) return 1;  // rows that no q-block names: partials are of all rows, and few of many would ask for gigabytes
  const int G = Hq / Hkv, Z = prefill_z(rows, G);
  const long groups = std::max(1L, std::min((long)n_qblocks * Z, (long)rows * G / 256 + n_qblocks) * Hkv);
  const long s = std::min((256 + groups - 1) / groups, (long)table_width * kPage / (4 * kTile));
  return (int)std::max(1L, std::min(s, 32L));
}

extern "C" int k8sllm_kv8_prefill(void* out, long out_stride, const void* qkv, long qkv_stride, const int* cu, const int* ctx, const int* qb_seq,
                                  const int* qb_start, int n_qblocks, int seqs, int rows, int Hq, int Hkv, int D, float scale, const void* k,
                                  const void* v, const float* scales, int pages, const int* table, long table_stride, int table_width, int S,
                                  float* part_o, float* part_ml, hipStream_t s) {
  if (n_qblocks <= 0 || rows <= 0) return 0;
  if (Hq % Hkv || S < 1 || S > 32) return -2;
  const int G = Hq / Hkv, Z = prefill_z(rows, G);
  const Kv8Prefill a{(bf16_t*)out, out_stride, (const bf16_t*)qkv, qkv_stride, cu, ctx, qb_seq, qb_start, (const uint8_t*)k, (const uint8_t*)v,
                     scales, pages, table, table_stride, table_width, rows, seqs, Hq, Hkv, G, Z, S, scale * 1.4426950408889634f, part_o, part_ml};
  const dim3 grid(Hkv, n_qblocks * Z, S);
  const dim3 joins((unsigned)((std::min(128, rows) * (long)Hq + 3) / 4), n_qblocks);
  if (D == 128) {
    hipLaunchKernelGGL((kv8_prefill_kernel<128>), grid, dim3(512), 0, s, a);
    if (S > 1) hipLaunchKernelGGL((kv8_prefill_join_kernel<128>), joins, dim3(256), 0, s, a);
  } else if (D == 64) {
    hipLaunchKernelGGL((kv8_prefill_kernel<64>), grid, dim3(512), 0, s, a);
    if (S > 1) hipLaunchKernelGGL((kv8_prefill_join_kernel<64>), joins, dim3(256), 0, s, a);
  } else {
    return -1;
  }
  return (int)hipGetLastError();
}
