// PyTorch bindings of the 8-bit KV cache and the logit controls: tensors are checked here, the work runs on the current stream of
// the tensors' device.
#include <torch/extension.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include <cmath>

extern "C" {
int k8sllm_reduce_slabs(void* out, const float* partial, int S, long n, hipStream_t s);
int k8sllm_rope_cache(void* qkv, long qkv_stride, const int* positions, const float* cos_sin, int max_pos, void* k_cache, void* v_cache,
                      const int* slot_mapping, long T, int Hq, int Hkv, int D, int block_size, int apply_rope, const float* partial, int S,
                      hipStream_t s);
int k8sllm_kv8_write(const void* qkv, long stride, const int* slots, void* k, void* v, float* scales, int T, int Hq, int Hkv, int D, int pages,
                     hipStream_t s);
int k8sllm_kv8_decode(void* out, long out_stride, float* part_o, float* part_ml, const void* q, long q_stride, void* k, void* v, float* scales,
                      int pages, const int* table, long table_stride, int table_width, const int* lens, int B, int Hq, int Hkv, int D, int S,
                      float scale, int* ctr, const float* slabs, int nslabs, const int* positions, const float* cos_sin, int max_pos,
                      const int* slots, hipStream_t s);
int k8sllm_kv8_prefill_splits(int n_qblocks, int rows, int Hq, int Hkv, int table_width);
int k8sllm_kv8_prefill(void* out, long out_stride, const void* qkv, long qkv_stride, const int* cu, const int* ctx, const int* qb_seq,
                       const int* qb_start, int n_qblocks, int seqs, int rows, int Hq, int Hkv, int D, float scale, const void* k, const void* v,
                       const float* scales, int pages, const int* table, long table_stride, int table_width, int S, float* part_o, float* part_ml,
                       hipStream_t s);
int k8sllm_logit_controls(void* out, long out_stride, const void* in, long in_stride, int types, int B, int V, const float* params,
                          const int* info, const int* bias_ids, const float* bias_vals, const void* masks, int slots, int n_bias, int words,
                          const int* rows, const int* tokens, int pages, const int* table, long table_stride, int table_width, const int* lens,
                          hipStream_t s);
int k8sllm_cache_tokens(int* tokens, int pages, const int* ids, const int* slots, const int* src, const int* prev, int n_prev, int n,
                        hipStream_t s);
}

namespace {

using torch::Tensor;

// The device of a call's tensors is made current for its duration
struct Call {
  c10::hip::HIPGuard guard;
  int dev;
  const char* what;
  Call(const Tensor& t, const char* w) : guard(check_gpu(t, w)), dev(t.get_device()), what(w) {}
  static c10::DeviceIndex check_gpu(const Tensor& t, const char* w) {
    TORCH_CHECK(t.is_cuda(), w, ": a GPU tensor is needed");
    return (c10::DeviceIndex)t.get_device();
  }
  hipStream_t stream() const { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)dev).stream(); }
  void typed(const Tensor& t, torch::ScalarType type, const char* n) const {
    TORCH_CHECK(t.is_cuda() && t.get_device() == dev, what, ": ", n, " must be on the same GPU");
    TORCH_CHECK(t.scalar_type() == type, what, ": ", n, " must be ", type, ", is ", t.scalar_type());
  }
  void whole(const Tensor& t, torch::ScalarType type, const char* n) const {
    typed(t, type, n);
    TORCH_CHECK(t.is_contiguous(), what, ": ", n, " must be contiguous");
  }
  // rows that 16-byte loads may read
  void rows(const Tensor& t, int64_t cols, const char* n) const {
    typed(t, torch::kBFloat16, n);
    TORCH_CHECK(t.dim() == 2 && t.size(1) >= cols && (t.stride(1) == 1 || t.size(0) == 0), what, ": ", n, " must be rows of at least ", cols);
    TORCH_CHECK((t.stride(0) % 8 == 0 || t.size(0) <= 1) && (uintptr_t)t.data_ptr() % 16 == 0, what, ": ", n,
                " must start at 16 bytes, its rows multiples of 8 elements apart");
  }
  void done(int rc) const { TORCH_CHECK(rc == 0, "k8sllm kernel launch failed: ", what, " rc=", rc); }
};

struct Heads {
  int Hq, Hkv, D;
  Heads(const Call& c, int64_t hq, int64_t hkv, int64_t d) : Hq((int)hq), Hkv((int)hkv), D((int)d) {
    TORCH_CHECK(d == 64 || d == 128, c.what, ": head size 64 or 128, is ", d);
    TORCH_CHECK(hkv >= 1 && hkv <= 65535 && hq >= hkv && hq % hkv == 0 && hq / hkv <= 16, c.what, ": 1 to 16 query heads a kv head, are ", hq, " over ",
                hkv);
  }
};

struct Cache {
  void *k, *v;
  float* scales;
  int pages;
  Cache(const Call& c, const Heads& h, const Tensor& k_, const Tensor& v_, const Tensor& s_) {
    c.whole(k_, torch::kFloat8_e4m3fn, "cache.k");
    c.whole(v_, torch::kFloat8_e4m3fn, "cache.v");
    c.whole(s_, torch::kFloat32, "cache.scales");
    TORCH_CHECK(k_.dim() == 5 && k_.size(1) == h.Hkv && k_.size(2) == 4 && k_.size(3) == 16 && k_.size(4) == h.D / 4, c.what,
                ": cache.k must be [pages, ", h.Hkv, ", 4, 16, ", h.D / 4, "], is ", k_.sizes());
    TORCH_CHECK(v_.dim() == 4 && v_.size(0) == k_.size(0) && v_.size(1) == h.Hkv && v_.size(2) == h.D && v_.size(3) == 16, c.what,
                ": cache.v must be [pages, ", h.Hkv, ", ", h.D, ", 16], is ", v_.sizes());
    TORCH_CHECK(s_.dim() == 3 && s_.size(0) == k_.size(0) && s_.size(1) == h.Hkv && s_.size(2) == 2, c.what, ": cache.scales must be [pages, ", h.Hkv,
                ", 2], is ", s_.sizes());
    TORCH_CHECK(k_.size(0) >= 1 && k_.size(0) < (1 << 27), c.what, ": 1 to 2^27 - 1 pages");
    k = k_.data_ptr();
    v = v_.data_ptr();
    scales = s_.data_ptr<float>();
    pages = (int)k_.size(0);
    TORCH_CHECK(((uintptr_t)k | (uintptr_t)v) % 16 == 0 && (uintptr_t)scales % 8 == 0, c.what, ": the cache must start at 16 bytes");
  }
};

struct Table {
  const int* p;
  long stride;
  int width;
  Table(const Call& c, const Tensor& t, int64_t rows) {
    c.typed(t, torch::kInt32, "block_tables");
    TORCH_CHECK(t.dim() == 2 && t.size(0) >= rows && t.size(1) >= 1 && t.size(1) < (1 << 26) && (t.stride(1) == 1 || t.size(1) == 1), c.what,
                ": block_tables must be [", rows, ", pages of a sequence]");
    p = t.data_ptr<int>();
    stride = t.stride(0);
    width = (int)t.size(1);
  }
};

void positive(const Call& c, double scale) { TORCH_CHECK(scale > 0 && std::isfinite(scale), c.what, ": scale must be positive, is ", scale); }

// Slab sum, rotation, write - nothing of it before every argument has been looked at
void kv8_write(Tensor qkv, c10::optional<Tensor> positions, c10::optional<Tensor> cos_sin, Tensor slots, Tensor k, Tensor v, Tensor scales,
               int64_t Hq, int64_t Hkv, int64_t D, bool apply_rope, c10::optional<Tensor> partial, int64_t nslabs) {
  Call c(qkv, "rope_and_cache_kv8");
  const Heads h(c, Hq, Hkv, D);
  c.rows(qkv, (Hq + 2 * Hkv) * D, "qkv");
  const Cache cache(c, h, k, v, scales);
  c.whole(slots, torch::kInt32, "slot_mapping");
  const int64_t T = qkv.size(0);
  TORCH_CHECK(slots.numel() >= T && T < (1LL << 30), c.what, ": a slot for each row");
  TORCH_CHECK(T * Hkv < (1LL << 31), c.what, ": rows times kv heads below 2^31");  // waves are numbered in 32 bits
  if (partial.has_value()) {
    c.whole(*partial, torch::kFloat32, "partial");
    TORCH_CHECK(qkv.size(1) == (Hq + 2 * Hkv) * D && qkv.is_contiguous() && nslabs >= 1 && nslabs < (1 << 20) &&
                    partial->numel() >= nslabs * qkv.numel() && (uintptr_t)partial->data_ptr() % 16 == 0, c.what,
                ": partial must hold nslabs x [T, (Hq + 2 Hkv) * D] from 16 bytes on, qkv be contiguous rows of that many columns");
  }
  if (apply_rope) {
    TORCH_CHECK(positions.has_value() && cos_sin.has_value(), c.what, ": positions and cos_sin are needed");
    c.whole(*positions, torch::kInt32, "positions");
    c.whole(*cos_sin, torch::kFloat32, "cos_sin");
    TORCH_CHECK(positions->numel() >= T && cos_sin->dim() == 2 && cos_sin->size(0) >= 1 && cos_sin->size(0) < (1LL << 31) && cos_sin->size(1) == D &&
                    (uintptr_t)cos_sin->data_ptr() % 16 == 0, c.what, ": positions [T] and cos_sin [positions, D], from 16 bytes on");
    TORCH_CHECK(T <= 1 || qkv.stride(0) >= (Hq + Hkv) * D, c.what, ": rows that are rotated in place must not overlap");
  }
  if (partial.has_value()) c.done(k8sllm_reduce_slabs(qkv.data_ptr(), partial->data_ptr<float>(), (int)nslabs, qkv.numel(), c.stream()));
  if (apply_rope)
    c.done(k8sllm_rope_cache(qkv.data_ptr(), qkv.stride(0), positions->data_ptr<int>(), cos_sin->data_ptr<float>(), (int)cos_sin->size(0), nullptr,
                             nullptr, nullptr, T, h.Hq, h.Hkv, h.D, 16, 1, nullptr, 0, c.stream()));
  c.done(k8sllm_kv8_write(qkv.data_ptr(), qkv.stride(0), slots.data_ptr<int>(), cache.k, cache.v, cache.scales, (int)T, h.Hq, h.Hkv, h.D,
                          cache.pages, c.stream()));
}

struct DecodeOut {
  long stride;
  DecodeOut(const Call& c, const Heads& h, const Tensor& out, int64_t B) {
    const int64_t n = (int64_t)h.Hq * h.D;
    c.typed(out, torch::kBFloat16, "out");
    if (out.dim() == 4) {
      TORCH_CHECK(n % 32 == 0 && out.is_contiguous() && out.size(1) * 32 == n && out.size(2) == 64 && out.size(3) == 8 && out.size(0) * 16 >= B,
                  c.what, ": a packed out must be [ceil(B / 16), Hq * D / 32, 64, 8]");
      stride = -(long)(n / 32);
    } else {
      TORCH_CHECK(out.dim() == 2 && out.stride(1) == 1 && out.size(0) >= B && out.size(1) == n && (out.stride(0) >= n || B <= 1), c.what,
                  ": out must be [B, Hq * D]");
      stride = B > 1 ? out.stride(0) : n;
    }
  }
};

int* decode_parts(const Call& c, const Heads& h, const Tensor& part_o, const Tensor& part_ml, const c10::optional<Tensor>& ctr, int64_t B, int64_t S) {
  TORCH_CHECK(S >= 1 && S <= 64, c.what, ": 1 to 64 splits");
  TORCH_CHECK(B <= 65535, c.what, ": at most 65535 rows");
  if (S == 1) return nullptr;
  c.whole(part_o, torch::kFloat32, "workspace[0]");
  c.whole(part_ml, torch::kFloat32, "workspace[1]");
  TORCH_CHECK(part_o.numel() >= B * h.Hq * S * h.D && part_ml.numel() >= B * h.Hq * S * 2, c.what, ": the workspace is too small for ", B, " rows x ",
              S, " splits");
  if (!ctr.has_value()) return nullptr;
  c.whole(*ctr, torch::kInt32, "workspace[2]");
  TORCH_CHECK(ctr->numel() >= B * h.Hkv, c.what, ": workspace[2] must hold a counter for each row and kv head");
  return ctr->data_ptr<int>();
}

void kv8_decode(Tensor out, Tensor q, Tensor k, Tensor v, Tensor scales, Tensor table, Tensor lens, Tensor part_o, Tensor part_ml,
                c10::optional<Tensor> ctr, int64_t Hq, int64_t Hkv, int64_t D, double scale, int64_t S) {
  Call c(q, "paged_decode_kv8");
  const Heads h(c, Hq, Hkv, D);
  positive(c, scale);
  c.whole(lens, torch::kInt32, "seq_lens");
  const int64_t B = lens.numel();
  c.rows(q, Hq * D, "q");
  TORCH_CHECK(q.size(0) >= B, c.what, ": a row of q for each sequence");
  const Cache cache(c, h, k, v, scales);
  const Table t(c, table, B);
  const DecodeOut o(c, h, out, B);
  int* counters = decode_parts(c, h, part_o, part_ml, ctr, B, S);
  c.done(k8sllm_kv8_decode(out.data_ptr(), o.stride, S > 1 ? part_o.data_ptr<float>() : nullptr, S > 1 ? part_ml.data_ptr<float>() : nullptr,
                           q.data_ptr(), q.stride(0), cache.k, cache.v, cache.scales, cache.pages, t.p, t.stride, t.width, lens.data_ptr<int>(),
                           (int)B, h.Hq, h.Hkv, h.D, (int)S, (float)scale, counters, nullptr, 0, nullptr, nullptr, 0, nullptr, c.stream()));
}

void kv8_decode_fused(Tensor out, Tensor slabs, int64_t nslabs, Tensor positions, Tensor cos_sin, c10::optional<Tensor> slots, Tensor k, Tensor v,
                      Tensor scales, Tensor table, Tensor lens, Tensor part_o, Tensor part_ml, c10::optional<Tensor> ctr, int64_t Hq, int64_t Hkv,
                      int64_t D, double scale, int64_t S) {
  Call c(slabs, "paged_decode_fused_kv8");
  const Heads h(c, Hq, Hkv, D);
  positive(c, scale);
  TORCH_CHECK(D == 128, c.what, ": head size 128, is ", D);
  c.whole(lens, torch::kInt32, "seq_lens");
  c.whole(positions, torch::kInt32, "positions");
  c.whole(cos_sin, torch::kFloat32, "cos_sin");
  c.whole(slabs, torch::kFloat32, "slabs");
  const int64_t B = lens.numel();
  TORCH_CHECK(nslabs >= 1 && nslabs < (1 << 20) && slabs.numel() >= nslabs * B * (Hq + 2 * Hkv) * D && (uintptr_t)slabs.data_ptr() % 16 == 0, c.what,
              ": slabs must hold nslabs x [B, (Hq + 2 Hkv) * D], from 16 bytes on");
  TORCH_CHECK(positions.numel() >= B && cos_sin.dim() == 2 && cos_sin.size(0) >= 1 && cos_sin.size(1) == D, c.what,
              ": positions [B] and cos_sin [positions, D]");
  const int* sl = nullptr;
  if (slots.has_value() && slots->numel() > 0) {
    c.whole(*slots, torch::kInt32, "slot_mapping");
    TORCH_CHECK(slots->numel() >= B, c.what, ": a slot for each row");
    sl = slots->data_ptr<int>();
  }
  const Cache cache(c, h, k, v, scales);
  const Table t(c, table, B);
  const DecodeOut o(c, h, out, B);
  int* counters = decode_parts(c, h, part_o, part_ml, ctr, B, S);
  c.done(k8sllm_kv8_decode(out.data_ptr(), o.stride, S > 1 ? part_o.data_ptr<float>() : nullptr, S > 1 ? part_ml.data_ptr<float>() : nullptr, nullptr,
                           0, cache.k, cache.v, cache.scales, cache.pages, t.p, t.stride, t.width, lens.data_ptr<int>(), (int)B, h.Hq, h.Hkv, h.D,
                           (int)S, (float)scale, counters, slabs.data_ptr<float>(), (int)nslabs, positions.data_ptr<int>(),
                           cos_sin.data_ptr<float>(), (int)cos_sin.size(0), sl, c.stream()));
}

void kv8_prefill(Tensor out, Tensor qkv, Tensor cu, Tensor ctx, Tensor qb_seq, Tensor qb_start, Tensor k, Tensor v, Tensor scales, Tensor table,
                 int64_t Hq, int64_t Hkv, int64_t D, double scale) {
  Call c(qkv, "flash_prefill_kv8");
  const Heads h(c, Hq, Hkv, D);
  positive(c, scale);
  c.rows(qkv, Hq * D, "qkv");
  for (const auto& t : {cu, ctx, qb_seq, qb_start}) c.whole(t, torch::kInt32, "cu_seqlens, ctx_start and qblocks");
  const int64_t seqs = cu.numel() - 1, T = qkv.size(0), nq = qb_seq.numel();
  TORCH_CHECK(seqs >= 0 && ctx.numel() >= seqs && qb_start.numel() == nq, c.what, ": cu_seqlens [S + 1], ctx_start [S], two equal lists of q-blocks");
  const Cache cache(c, h, k, v, scales);
  const Table t(c, table, seqs);
  c.typed(out, torch::kBFloat16, "out");
  TORCH_CHECK(out.dim() == 2 && out.size(0) >= T && out.size(1) == Hq * D && (T == 0 || out.stride(1) == 1) && ((out.stride(0) % 4 == 0 && out.stride(0) >= Hq * D) || T <= 1) &&
                  (uintptr_t)out.data_ptr() % 8 == 0, c.what, ": out must be [T, Hq * D], from 8 bytes on");
  TORCH_CHECK(nq * ((128 * (Hq / Hkv) + 255) / 256) <= 65535 && T < (1LL << 30), c.what, ": too many q-blocks");
  if (T == 0 || nq == 0) return;
  const int S = k8sllm_kv8_prefill_splits((int)nq, (int)T, h.Hq, h.Hkv, t.width);
  Tensor po, pml;
  if (S > 1) {  // the allocator's, on this stream: a later call on it may take them again when this one is done
    po = torch::empty({S, T, Hq, D}, qkv.options().dtype(torch::kFloat32));
    pml = torch::empty({S, T, Hq, 2}, qkv.options().dtype(torch::kFloat32));
  }
  c.done(k8sllm_kv8_prefill(out.data_ptr(), T > 1 ? out.stride(0) : Hq * D, qkv.data_ptr(), qkv.stride(0), cu.data_ptr<int>(), ctx.data_ptr<int>(),
                            qb_seq.data_ptr<int>(), qb_start.data_ptr<int>(), (int)nq, (int)seqs, (int)T, h.Hq, h.Hkv, h.D, (float)scale, cache.k,
                            cache.v, cache.scales, cache.pages, t.p, t.stride, t.width, S, S > 1 ? po.data_ptr<float>() : nullptr,
                            S > 1 ? pml.data_ptr<float>() : nullptr, c.stream()));
}

// Whether rows of `out` share memory with rows of `in` other than as one and the same view
bool half_shared(const Tensor& out, const Tensor& in) {
  const int64_t B = in.size(0), os = out.stride(0) * out.element_size(), is = in.stride(0) * in.element_size();
  const int64_t ow = out.size(1) * out.element_size(), iw = in.size(1) * in.element_size(), d = (char*)out.data_ptr() - (char*)in.data_ptr();
  if (d >= (B - 1) * is + iw || -d >= (B - 1) * os + ow) return false;
  if (B > 1 && os != is) return true;
  if (d == 0 && out.scalar_type() == in.scalar_type()) return false;
  // row i of out begins d + (i - j) * is behind row j of in
  for (int64_t k = -(B - 1); k < B; ++k)
    if (d + k * is < iw && -(d + k * is) < ow) return true;
  return false;
}

void logit_controls(Tensor out, Tensor logits, Tensor params, Tensor info, Tensor bias_ids, Tensor bias_vals, Tensor masks, Tensor rows, Tensor tokens,
                    Tensor table, Tensor lens) {
  Call c(logits, "control_logits");
  TORCH_CHECK(logits.dim() == 2 && out.dim() == 2 && out.sizes() == logits.sizes(), c.what, ": logits and out [B, V]");
  const int64_t B = logits.size(0), V = logits.size(1);
  const bool in32 = logits.scalar_type() == torch::kFloat32, out32 = out.scalar_type() == torch::kFloat32;
  TORCH_CHECK((in32 || logits.scalar_type() == torch::kBFloat16) && (out32 || (!in32 && out.scalar_type() == torch::kBFloat16)), c.what,
              ": logits bfloat16 or float32, out of the same type or float32");
  TORCH_CHECK(out.is_cuda() && out.get_device() == c.dev, c.what, ": out must be on the same GPU");
  TORCH_CHECK(B == 0 || V == 0 || (logits.stride(1) == 1 && out.stride(1) == 1 && V < (1LL << 30)), c.what, ": rows must be contiguous");
  TORCH_CHECK(B <= 1 || out.stride(0) >= V, c.what, ": rows of out must not overlap");
  TORCH_CHECK(B <= 65535, c.what, ": at most 65535 rows");
  if (B == 0 || V == 0) return;
  TORCH_CHECK(!half_shared(out, logits), c.what, ": out shares memory with the logits and is not the same rows");
  c.whole(params, torch::kFloat32, "controls.params");
  c.whole(info, torch::kInt32, "controls.info");
  c.whole(bias_ids, torch::kInt32, "controls.bias_ids");
  c.whole(bias_vals, torch::kFloat32, "controls.bias_vals");
  c.whole(masks, torch::kInt32, "controls.masks");
  const int64_t n = params.size(0), words = (V + 31) / 32;
  TORCH_CHECK(params.dim() == 2 && params.size(1) == 3 && info.dim() == 2 && info.size(0) == n && info.size(1) == 2 && bias_ids.dim() == 2 &&
                  bias_ids.size(0) == n && bias_vals.sizes() == bias_ids.sizes() && masks.dim() == 2 && masks.size(0) == n && masks.size(1) >= words,
              c.what, ": controls must be params [n, 3], info [n, 2], bias_ids and bias_vals [n, m], masks [n, ceil(V / 32)]");
  TORCH_CHECK(bias_ids.size(1) <= 2046, c.what, ": at most 2046 biased tokens a slot");
  c.whole(rows, torch::kInt32, "rows");
  c.whole(lens, torch::kInt32, "seq_lens");
  c.whole(tokens, torch::kInt32, "token_cache");
  TORCH_CHECK(rows.numel() >= B && lens.numel() >= B && tokens.dim() == 2 && tokens.size(1) == 16 && tokens.size(0) < (1 << 27) &&
                  (uintptr_t)tokens.data_ptr() % 16 == 0, c.what, ": rows [B], seq_lens [B], token_cache [pages, 16] from 16 bytes on");
  const Table t(c, table, B);
  TORCH_CHECK(t.width < (1 << 16), c.what, ": histories of less than 2^20 tokens");
  c.done(k8sllm_logit_controls(out.data_ptr(), out.stride(0), logits.data_ptr(), logits.stride(0), in32 ? 1 : out32 ? 2 : 0, (int)B, (int)V,
                               params.data_ptr<float>(), info.data_ptr<int>(), bias_ids.data_ptr<int>(), bias_vals.data_ptr<float>(),
                               masks.data_ptr<int>(), (int)n, (int)bias_ids.size(1), (int)masks.size(1), rows.data_ptr<int>(),
                               tokens.data_ptr<int>(), (int)tokens.size(0), t.p, t.stride, t.width, lens.data_ptr<int>(), c.stream()));
}

void cache_tokens(Tensor tokens, Tensor ids, Tensor slots, c10::optional<Tensor> src, c10::optional<Tensor> prev) {
  Call c(tokens, "cache_tokens");
  c.whole(tokens, torch::kInt32, "token_cache");
  c.whole(ids, torch::kInt32, "ids");
  c.whole(slots, torch::kInt32, "slot_mapping");
  TORCH_CHECK(tokens.dim() == 2 && tokens.size(1) == 16 && tokens.size(0) < (1 << 27), c.what, ": token_cache [pages, 16]");
  const int64_t n = ids.numel();
  TORCH_CHECK(slots.numel() >= n && n < (1LL << 30), c.what, ": a slot for each id");
  TORCH_CHECK(src.has_value() == prev.has_value(), c.what, ": src and prev go together");
  if (src.has_value()) {
    c.whole(*src, torch::kInt32, "src");
    c.whole(*prev, torch::kInt32, "prev");
    TORCH_CHECK(src->numel() >= n, c.what, ": a src for each id");
  }
  c.done(k8sllm_cache_tokens(tokens.data_ptr<int>(), (int)tokens.size(0), ids.data_ptr<int>(), slots.data_ptr<int>(),
                             src.has_value() ? src->data_ptr<int>() : nullptr, prev.has_value() ? prev->data_ptr<int>() : nullptr,
                             prev.has_value() ? (int)prev->numel() : 0, (int)n, c.stream()));
}

}  // namespace

void bind_serving(pybind11::module_& m) {
  m.def("kv8_write", &kv8_write);
  m.def("kv8_decode", &kv8_decode);
  m.def("kv8_decode_fused", &kv8_decode_fused);
  m.def("kv8_prefill", &kv8_prefill);
  m.def("logit_controls", &logit_controls);
  m.def("cache_tokens", &cache_tokens);
}
