// Host contract validation for the dense paged MLA launch, and the Philox4x32-10 test stream.
//
// Validation restates SmlaParams::new (crates/tq-core/src/contracts.rs:437-493) and its helpers
// check (:262-325), check_strides (:331-356), check_kv_strides (:359-371) and check_aliases
// (:407-421): same field names, same violation kinds, same checked 64-bit span arithmetic, same
// empty-launch rule (docs/HOST-CONTRACTS.md:96-102). The generalisations (576-wide rows, 16/128
// heads, runtime scale for the 576 format, no sparse index tensors, f32 partial outputs,
// unbounded prefill plans) are listed in tq_contracts.h.
//
// Philox restates crates/tq-testkit/src/philox.rs:57-111 (block, fill_words, uniform_f32).

#include "tq_contracts.h"

#include <cmath>
#include <cstring>

namespace tq {

namespace {

constexpr uint64_t kDimensionLimit = uint64_t(1) << 31;
constexpr uint64_t kPageRows = 64;
constexpr uint64_t kKvGranularity = 16;
constexpr uint32_t kGlmScaleBits = 0x3D800000u;  // 0.0625f
constexpr uint64_t kDigestSalt = 0x7C3A5E1B9D2F4861ull;

enum class Layout { Packed, PaddedOuter, Checked };

struct Extent {
  const char* field;
  uint64_t start, end;
  bool present;
};

struct Failure {
  const char* field;
  int32_t kind;
};

uint64_t element_bytes(int32_t dtype) {
  switch (dtype) {
    case TQ_DTYPE_U8: return 1;
    case TQ_DTYPE_BF16: return 2;
    case TQ_DTYPE_I32:
    case TQ_DTYPE_F32: return 4;
    default: return 0;
  }
}

bool mul_overflows(uint64_t a, uint64_t b, uint64_t* out) {
  return __builtin_mul_overflow(a, b, out);
}
bool add_overflows(uint64_t a, uint64_t b, uint64_t* out) {
  return __builtin_add_overflow(a, b, out);
}

// Innermost stride is the element size; each outer stride spans the axis inside it.
bool check_strides(const TqTensorSpec& t, int rank, Layout layout, uint64_t element,
                   int32_t* kind) {
  if (t.strides_bytes[rank - 1] != element) { *kind = TQ_STRIDE; return false; }
  for (int axis = rank - 2; axis >= 0; --axis) {
    uint64_t inner = t.strides_bytes[axis + 1];
    uint64_t extent = t.shape[axis + 1] > 1 ? t.shape[axis + 1] : 1;
    uint64_t needed;
    if (mul_overflows(inner, extent, &needed)) { *kind = TQ_OVERFLOW; return false; }
    uint64_t stride = t.strides_bytes[axis];
    bool fits = layout == Layout::Packed ? stride == needed
                                         : (stride >= needed && stride % element == 0);
    if (!fits) { *kind = TQ_STRIDE; return false; }
  }
  return true;
}

// Checks one tensor; on success fills `ext` (present only when launching and non-empty).
bool check(const char* field, const TqTensorSpec& t, const uint64_t* shape, int rank,
           int32_t dtype, Layout layout, bool launching, Extent* ext, Failure* f) {
  ext->present = false;
  ext->field = field;
  if (t.rank != rank) { *f = {field, TQ_SHAPE}; return false; }
  if (t.dtype != dtype) { *f = {field, TQ_DTYPE}; return false; }
  for (int i = 0; i < rank; ++i)
    if (t.shape[i] != shape[i]) { *f = {field, TQ_SHAPE}; return false; }
  for (int i = 0; i < rank; ++i)
    if (t.shape[i] >= kDimensionLimit) { *f = {field, TQ_DIMENSION}; return false; }
  const uint64_t element = element_bytes(dtype);
  int32_t kind = 0;
  if (layout != Layout::Checked && !check_strides(t, rank, layout, element, &kind)) {
    *f = {field, kind};
    return false;
  }
  bool empty = false;
  for (int i = 0; i < rank; ++i) empty |= t.shape[i] == 0;
  if (!launching || empty) return true;
  uint64_t span = element;
  for (int i = 0; i < rank; ++i) {
    uint64_t reach;
    if (mul_overflows(t.shape[i] - 1, t.strides_bytes[i], &reach) ||
        add_overflows(span, reach, &span)) {
      *f = {field, TQ_OVERFLOW};
      return false;
    }
  }
  if (t.device_address == 0) { *f = {field, TQ_ADDRESS}; return false; }
  const uint64_t granularity = layout == Layout::Checked ? kKvGranularity : element;
  if (t.device_address % granularity != 0) { *f = {field, TQ_ALIGNMENT}; return false; }
  if (t.buffer_bytes < span) { *f = {field, TQ_CAPACITY}; return false; }
  uint64_t end;
  if (add_overflows(t.device_address, t.buffer_bytes, &end)) {
    *f = {field, TQ_OVERFLOW};
    return false;
  }
  // The bytes the tensor covers, not the capacity behind it (contracts.rs:318-324).
  *ext = {field, t.device_address, t.device_address + span, true};
  return true;
}

// Paged KV rows are [64 r, r, 1] with r at least the payload and a multiple of 16.
bool check_kv_strides(const TqTensorSpec& t, uint64_t payload, Failure* f) {
  if (t.rank != 3) { *f = {"kv", TQ_SHAPE}; return false; }
  const uint64_t row = t.strides_bytes[1];
  if (t.strides_bytes[2] != 1 || row < payload || row % kKvGranularity != 0) {
    *f = {"kv", TQ_STRIDE};
    return false;
  }
  uint64_t page;
  if (mul_overflows(kPageRows, row, &page)) { *f = {"kv", TQ_OVERFLOW}; return false; }
  if (t.strides_bytes[0] != page) { *f = {"kv", TQ_STRIDE}; return false; }
  return true;
}

bool check_aliases(const Extent* inputs, int n_in, const Extent* outputs, int n_out, Failure* f) {
  for (int o = 0; o < n_out; ++o) {
    const Extent& out = outputs[o];
    if (!out.present) continue;
    for (int i = 0; i < n_in + o; ++i) {
      const Extent& other = i < n_in ? inputs[i] : outputs[i - n_in];
      if (!other.present) continue;
      if (out.start < other.end && other.start < out.end) {
        *f = {out.field, TQ_ALIAS};
        return false;
      }
    }
  }
  return true;
}

uint32_t f32_bits(float x) {
  uint32_t b;
  std::memcpy(&b, &x, 4);
  return b;
}

bool scale_ok(int32_t format, float scale) {
  if (format == TQ_KV_BF16 || format == TQ_KV_FP8_E4M3) return f32_bits(scale) == kGlmScaleBits;
  return std::isfinite(scale) && scale > 0.0f;
}

// FNV-1a over the bytes of the params (digest field excluded).
uint64_t digest_of(const TqMlaParams& p) {
  const unsigned char* b = reinterpret_cast<const unsigned char*>(&p);
  const size_t n = offsetof(TqMlaParams, digest);
  uint64_t h = 0xCBF29CE484222325ull ^ kDigestSalt;
  for (size_t i = 0; i < n; ++i) {
    h ^= b[i];
    h *= 0x100000001B3ull;
  }
  return h;
}

template <typename Count>
// `idx` / `k_len` non-null: a sparse top-k plan (contracts.rs:442-470 checks them in this order:
// the index width right after q, then idx padded and k_len packed after kv_len).
int32_t validate_impl(const TqMlaSpec* spec, const Count* counts, uint64_t n, int max_per_seq,
                      TqMlaParams* params, TqContractError* err,
                      const TqTensorSpec* idx = nullptr, const TqTensorSpec* k_len = nullptr) {
  Failure f{nullptr, TQ_OK};
  auto fail = [&](const char* field, int32_t kind) {
    if (err) { err->field = field; err->kind = kind; }
    return kind;
  };
  if (!spec || (!counts && n != 0)) return fail("spec", TQ_ERR_INVALID_ARGUMENT);
  const TqMlaSpec& s = *spec;
  if (s.q.rank != 3) return fail("q", TQ_SHAPE);
  const uint64_t tokens = s.q.shape[0], heads = s.q.shape[1], width = s.q.shape[2];
  uint64_t payload = 0, qk_width = 0;
  switch (s.kv_format) {
    case TQ_KV_BF16: payload = 1024; qk_width = 512; break;
    case TQ_KV_FP8_E4M3: payload = 528; qk_width = 512; break;
    case TQ_KV_BF16_ROPE576: payload = 1152; qk_width = 576; break;
    default: return fail("kv_format", TQ_SHAPE);
  }
  if ((heads != 16 && heads != 32 && heads != 64 && heads != 128) || width != qk_width)
    return fail("q", TQ_SHAPE);
  const bool sparse = idx != nullptr;
  if (sparse && (!k_len || s.kv_format == TQ_KV_BF16_ROPE576)) return fail("kv_format", TQ_SHAPE);
  if (sparse && (idx->rank != 2 || idx->shape[1] > TQ_MLA_MAX_TOPK)) return fail("idx", TQ_SHAPE);
  if (!scale_ok(s.kv_format, s.softmax_scale)) return fail("softmax_scale", TQ_SCALE);
  if (s.page_table.rank != 2) return fail("page_table", TQ_SHAPE);
  const uint64_t sequences = s.page_table.shape[0], slots = s.page_table.shape[1];
  const bool launching = tokens != 0;
  if (!check_kv_strides(s.kv, payload, &f)) return fail(f.field, f.kind);

  const uint64_t query[3] = {tokens, heads, width};
  const uint64_t pool[3] = {s.kv.shape[0], kPageRows, payload};
  const uint64_t table[2] = {sequences, slots};
  const uint64_t tok[1] = {tokens};
  const uint64_t seqs[1] = {sequences};
  const uint64_t outshape[3] = {tokens, heads, 512};
  const uint64_t lseshape[2] = {tokens, heads};
  Extent in[8], out[2];
  if (!check("q", s.q, query, 3, TQ_DTYPE_BF16, Layout::PaddedOuter, launching, &in[0], &f) ||
      !check("kv", s.kv, pool, 3, TQ_DTYPE_U8, Layout::Checked, launching, &in[1], &f) ||
      !check("page_table", s.page_table, table, 2, TQ_DTYPE_I32, Layout::Packed, launching,
             &in[2], &f) ||
      !check("seq_id", s.seq_id, tok, 1, TQ_DTYPE_I32, Layout::Packed, launching, &in[3], &f) ||
      !check("q_pos", s.q_pos, tok, 1, TQ_DTYPE_I32, Layout::Packed, launching, &in[4], &f) ||
      !check("kv_len", s.kv_len, seqs, 1, TQ_DTYPE_I32, Layout::Packed, launching, &in[5], &f))
    return fail(f.field, f.kind);
  const uint64_t topk = sparse ? idx->shape[1] : 0;
  if (sparse) {
    const uint64_t idx_shape[2] = {tokens, topk};
    if (!check("idx", *idx, idx_shape, 2, TQ_DTYPE_I32, Layout::PaddedOuter, launching, &in[6],
               &f) ||
        !check("k_len", *k_len, tok, 1, TQ_DTYPE_I32, Layout::Packed, launching, &in[7], &f))
      return fail(f.field, f.kind);
  }
  // The output may be bf16 (final) or f32 (a partial result to merge across devices).
  const int32_t out_dtype = s.out.dtype == TQ_DTYPE_F32 ? TQ_DTYPE_F32 : TQ_DTYPE_BF16;
  if (!check("out", s.out, outshape, 3, out_dtype, Layout::PaddedOuter, launching, &out[0], &f) ||
      !check("lse", s.lse, lseshape, 2, TQ_DTYPE_F32, Layout::Packed, launching, &out[1], &f))
    return fail(f.field, f.kind);

  if (n != sequences) return fail("query_counts", TQ_QUERY_COUNT);
  uint64_t planned = 0;
  for (uint64_t i = 0; i < n; ++i) {
    const uint64_t c = counts[i];
    if (max_per_seq > 0 && c > uint64_t(max_per_seq)) return fail("query_counts", TQ_QUERY_COUNT);
    planned += c;  // n < 2^31 and c < 2^32: cannot wrap
  }
  if (planned != tokens) return fail("query_counts", TQ_QUERY_COUNT);
  if (!check_aliases(in, sparse ? 8 : 6, out, 2, &f)) return fail(f.field, f.kind);

  if (params) {
    std::memset(params, 0, sizeof(*params));
    params->spec = s;
    params->tokens = tokens;
    params->heads = heads;
    params->sequences = sequences;
    params->slots = slots;
    params->pages = s.kv.shape[0];
    params->qk_width = qk_width;
    params->row_stride = s.kv.strides_bytes[1];
    params->max_queries_per_sequence = max_per_seq;
    params->should_launch = launching ? 1 : 0;
    if (sparse) {
      params->idx = *idx;
      params->k_len = *k_len;
      params->topk = topk;
      params->sparse = 1;
    }
    params->digest = digest_of(*params);
  }
  if (err) { err->field = nullptr; err->kind = TQ_OK; }
  return TQ_OK;
}

// The KV writer's declarations: the same per-tensor checks as the attention plan, the pool as
// the output that no input may overlap, and 16-byte vector access to the source rows.
int32_t kv_write_validate_impl(const TqKvWriteSpec* spec, TqContractError* err) {
  Failure f{nullptr, TQ_OK};
  auto fail = [&](const char* field, int32_t kind) {
    if (err) { err->field = field; err->kind = kind; }
    return kind;
  };
  if (!spec) return fail("spec", TQ_ERR_INVALID_ARGUMENT);
  const TqKvWriteSpec& s = *spec;
  uint64_t payload = 0, width = 0;
  switch (s.kv_format) {
    case TQ_KV_BF16: payload = 1024; width = 512; break;
    case TQ_KV_FP8_E4M3: payload = 528; width = 512; break;
    case TQ_KV_BF16_ROPE576: payload = 1152; width = 576; break;
    default: return fail("kv_format", TQ_SHAPE);
  }
  if (s.src.rank != 2) return fail("src", TQ_SHAPE);
  if (s.page_table.rank != 2) return fail("page_table", TQ_SHAPE);
  const uint64_t rows = s.src.shape[0];
  const uint64_t sequences = s.page_table.shape[0], slots = s.page_table.shape[1];
  const bool launching = rows != 0;
  if (!check_kv_strides(s.kv, payload, &f)) return fail(f.field, f.kind);
  const uint64_t src_shape[2] = {rows, width};
  const uint64_t pool[3] = {s.kv.shape[0], kPageRows, payload};
  const uint64_t table[2] = {sequences, slots};
  const uint64_t tok[1] = {rows};
  Extent in[5], out[1];
  if (!check("src", s.src, src_shape, 2, TQ_DTYPE_BF16, Layout::PaddedOuter, launching, &in[0],
             &f) ||
      !check("page_table", s.page_table, table, 2, TQ_DTYPE_I32, Layout::Packed, launching,
             &in[1], &f) ||
      !check("seq_id", s.seq_id, tok, 1, TQ_DTYPE_I32, Layout::Packed, launching, &in[2], &f) ||
      !check("pos", s.pos, tok, 1, TQ_DTYPE_I32, Layout::Packed, launching, &in[3], &f) ||
      !check("kv", s.kv, pool, 3, TQ_DTYPE_U8, Layout::Checked, launching, &out[0], &f))
    return fail(f.field, f.kind);
  if (launching) {
    if (s.src.strides_bytes[0] % 16) return fail("src", TQ_STRIDE);
    if (s.src.device_address % 16) return fail("src", TQ_ALIGNMENT);
  }
  int n_in = 4;
  if (s.norm_weight.rank != 0) {
    const uint64_t w_shape[1] = {512};
    if (!check("norm_weight", s.norm_weight, w_shape, 1, TQ_DTYPE_BF16, Layout::Packed,
               launching, &in[4], &f))
      return fail(f.field, f.kind);
    if (launching && s.norm_weight.device_address % 16) return fail("norm_weight", TQ_ALIGNMENT);
    if (!(std::isfinite(s.norm_eps) && s.norm_eps > 0.f)) return fail("norm_eps", TQ_SCALE);
    n_in = 5;
  }
  if (!check_aliases(in, n_in, out, 1, &f)) return fail(f.field, f.kind);
  if (err) { err->field = nullptr; err->kind = TQ_OK; }
  return TQ_OK;
}

// MLA prologue: the same tensor-declaration rules (shape, dtype, packed strides, spans, null,
// alignment, capacity; outputs never alias inputs), plus 16-byte aligned rows for the GEMMs.
int32_t prologue_validate_impl(const TqPrologueSpec* spec, TqContractError* err) {
  Failure f{nullptr, TQ_OK};
  auto fail = [&](const char* field, int32_t kind) {
    if (err) { err->field = field; err->kind = kind; }
    return kind;
  };
  if (!spec) return fail("spec", TQ_ERR_INVALID_ARGUMENT);
  const TqPrologueSpec& s = *spec;
  if (s.x.rank != 2) return fail("x", TQ_SHAPE);
  if (s.w_qa.rank != 2) return fail("w_qa", TQ_SHAPE);
  if (s.page_table.rank != 2) return fail("page_table", TQ_SHAPE);
  if (s.heads <= 0 || s.heads > 128) return fail("heads", TQ_SHAPE);
  if (s.nope_dim <= 0 || s.nope_dim > 512 || s.nope_dim % 8) return fail("nope_dim", TQ_SHAPE);
  if (s.rope_dim != 0 && s.rope_dim != 64) return fail("rope_dim", TQ_SHAPE);
  uint64_t payload = 0;
  switch (s.kv_format) {
    case TQ_KV_BF16: payload = 1024; break;
    case TQ_KV_FP8_E4M3: payload = 528; break;
    case TQ_KV_BF16_ROPE576: payload = 1152; break;
    default: return fail("kv_format", TQ_SHAPE);
  }
  if ((s.kv_format == TQ_KV_BF16_ROPE576) != (s.rope_dim == 64)) return fail("kv_format", TQ_SHAPE);
  const uint64_t T = s.x.shape[0], dm = s.x.shape[1], rq = s.w_qa.shape[0];
  const uint64_t H = uint64_t(s.heads), dn = uint64_t(s.nope_dim), dr = uint64_t(s.rope_dim);
  if (dm == 0 || dm % 8 || dm > (1u << 20)) return fail("x", TQ_SHAPE);
  if (rq == 0 || rq % 8 || rq > (1u << 16)) return fail("w_qa", TQ_SHAPE);
  if (T > (1u << 24)) return fail("x", TQ_SHAPE);
  const bool launching = T != 0;
  if (!check_kv_strides(s.kv, payload, &f)) return fail(f.field, f.kind);
  const uint64_t x_shape[2] = {T, dm}, wqa[2] = {rq, dm}, qn[1] = {rq};
  const uint64_t wqb[2] = {H * (dn + dr), rq}, wuk[3] = {H, dn, 512}, wkva[2] = {512 + dr, dm};
  const uint64_t kvn[1] = {512}, tok[1] = {T};
  const uint64_t table[2] = {s.page_table.shape[0], s.page_table.shape[1]};
  // Without w_uk the query is not absorbed: [Dn | Dr] per head.
  const bool absorb = s.w_uk.rank != 0;
  const uint64_t pool[3] = {s.kv.shape[0], kPageRows, payload};
  const uint64_t q_shape[3] = {T, H, (absorb ? 512 : dn) + dr};
  Extent in[10], out[2];
  in[4].present = false;
  if (!check("x", s.x, x_shape, 2, TQ_DTYPE_BF16, Layout::Packed, launching, &in[0], &f) ||
      !check("w_qa", s.w_qa, wqa, 2, TQ_DTYPE_BF16, Layout::Packed, launching, &in[1], &f) ||
      !check("q_norm", s.q_norm, qn, 1, TQ_DTYPE_BF16, Layout::Packed, launching, &in[2], &f) ||
      !check("w_qb", s.w_qb, wqb, 2, TQ_DTYPE_BF16, Layout::Packed, launching, &in[3], &f) ||
      (absorb &&
       !check("w_uk", s.w_uk, wuk, 3, TQ_DTYPE_BF16, Layout::Packed, launching, &in[4], &f)) ||
      !check("w_kva", s.w_kva, wkva, 2, TQ_DTYPE_BF16, Layout::Packed, launching, &in[5], &f) ||
      !check("kv_norm", s.kv_norm, kvn, 1, TQ_DTYPE_BF16, Layout::Packed, launching, &in[6], &f) ||
      !check("pos", s.pos, tok, 1, TQ_DTYPE_I32, Layout::Packed, launching, &in[7], &f) ||
      !check("seq_id", s.seq_id, tok, 1, TQ_DTYPE_I32, Layout::Packed, launching, &in[8], &f) ||
      !check("page_table", s.page_table, table, 2, TQ_DTYPE_I32, Layout::Packed, launching,
             &in[9], &f) ||
      !check("kv", s.kv, pool, 3, TQ_DTYPE_U8, Layout::Checked, launching, &out[0], &f) ||
      !check("q", s.q, q_shape, 3, TQ_DTYPE_BF16, Layout::Packed, launching, &out[1], &f))
    return fail(f.field, f.kind);
  if (launching) {
    const TqTensorSpec* mats[8] = {&s.x, &s.w_qa, &s.q_norm, &s.w_qb, &s.w_uk, &s.w_kva,
                                   &s.kv_norm, &s.q};
    const char* names[8] = {"x", "w_qa", "q_norm", "w_qb", "w_uk", "w_kva", "kv_norm", "q"};
    for (int i = 0; i < 8; ++i)
      if (mats[i]->rank != 0 && mats[i]->device_address % 16)
        return fail(names[i], TQ_ALIGNMENT);
  }
  if (!(std::isfinite(s.q_eps) && s.q_eps > 0.f)) return fail("q_eps", TQ_SCALE);
  if (!(std::isfinite(s.kv_eps) && s.kv_eps > 0.f)) return fail("kv_eps", TQ_SCALE);
  if (!(std::isfinite(s.rope_theta) && s.rope_theta > 1.f)) return fail("rope_theta", TQ_SCALE);
  if (!check_aliases(in, 10, out, 2, &f)) return fail(f.field, f.kind);
  if (err) { err->field = nullptr; err->kind = TQ_OK; }
  return TQ_OK;
}

// Step plan: whole-number tensors, packed; no output overlaps an input or another output.
int32_t step_plan_validate_impl(const TqStepPlanSpec* spec, TqContractError* err) {
  Failure f{nullptr, TQ_OK};
  auto fail = [&](const char* field, int32_t kind) {
    if (err) { err->field = field; err->kind = kind; }
    return kind;
  };
  if (!spec) return fail("spec", TQ_ERR_INVALID_ARGUMENT);
  const TqStepPlanSpec& s = *spec;
  if (s.cached_len.rank != 1) return fail("cached_len", TQ_SHAPE);
  if (s.page_table.rank != 2) return fail("page_table", TQ_SHAPE);
  if (s.free_pages.rank != 1) return fail("free_pages", TQ_SHAPE);
  if (s.seq_id.rank != 1) return fail("seq_id", TQ_SHAPE);
  const uint64_t reqs[1] = {s.cached_len.shape[0]}, starts[1] = {s.cached_len.shape[0] + 1};
  const uint64_t table[2] = {reqs[0], s.page_table.shape[1]}, one[1] = {1};
  const uint64_t pool[1] = {s.free_pages.shape[0]}, tok[1] = {s.seq_id.shape[0]};
  Extent in[4], out[7];
  int n_out = 6;
  const int32_t i32 = TQ_DTYPE_I32;
  const Layout packed = Layout::Packed;
  if (!check("cached_len", s.cached_len, reqs, 1, i32, packed, true, &in[0], &f) ||
      !check("new_len", s.new_len, reqs, 1, i32, packed, true, &in[1], &f) ||
      !check("page_table", s.page_table, table, 2, i32, packed, true, &out[0], &f) ||
      !check("free_pages", s.free_pages, pool, 1, i32, packed, true, &in[2], &f) ||
      !check("free_count", s.free_count, one, 1, i32, packed, true, &in[3], &f) ||
      !check("q_start", s.q_start, starts, 1, i32, packed, true, &out[1], &f) ||
      !check("kv_len", s.kv_len, reqs, 1, i32, packed, true, &out[2], &f) ||
      !check("seq_id", s.seq_id, tok, 1, i32, packed, true, &out[3], &f) ||
      !check("q_pos", s.q_pos, tok, 1, i32, packed, true, &out[4], &f) ||
      !check("free_left", s.free_left, one, 1, i32, packed, true, &out[5], &f))
    return fail(f.field, f.kind);
  if (s.slot.rank != 0) {
    if (!check("slot", s.slot, tok, 1, i32, packed, true, &out[6], &f))
      return fail(f.field, f.kind);
    n_out = 7;
  }
  if (!check_aliases(in, 4, out, n_out, &f)) return fail(f.field, f.kind);
  if (err) { err->field = nullptr; err->kind = TQ_OK; }
  return TQ_OK;
}

// Two declarations of the same elements: an output written in place over its input.
bool same_place(const TqTensorSpec& a, const TqTensorSpec& b) {
  return a.device_address == b.device_address && a.dtype == b.dtype &&
         a.strides_bytes[0] == b.strides_bytes[0] && a.strides_bytes[1] == b.strides_bytes[1];
}

int32_t block_norm_validate_impl(const TqBlockNormSpec* spec, TqContractError* err) {
  Failure f{nullptr, TQ_OK};
  auto fail = [&](const char* field, int32_t kind) {
    if (err) { err->field = field; err->kind = kind; }
    return kind;
  };
  if (!spec) return fail("spec", TQ_ERR_INVALID_ARGUMENT);
  const TqBlockNormSpec& s = *spec;
  if (s.y.rank != 2) return fail("y", TQ_SHAPE);
  const uint64_t rows = s.y.shape[0], width = s.y.shape[1];
  if (width == 0 || width % 8 || width > 32768) return fail("y", TQ_SHAPE);
  const uint64_t shape[2] = {rows, width}, w_shape[1] = {width};
  const bool launching = rows != 0;
  if (s.residual.dtype != TQ_DTYPE_BF16 && s.residual.dtype != TQ_DTYPE_F32)
    return fail("residual", TQ_DTYPE);
  const int32_t bf = TQ_DTYPE_BF16, kind = s.residual.dtype;
  Extent y, res, others[3], out, x;
  int n = 0;
  x.present = false;
  if (!check("y", s.y, shape, 2, bf, Layout::PaddedOuter, launching, &y, &f) ||
      !check("residual", s.residual, shape, 2, kind, Layout::PaddedOuter, launching, &res, &f))
    return fail(f.field, f.kind);
  if (s.gate.rank != 0) {
    if (s.gate.rank == 1 ? !check("gate", s.gate, w_shape, 1, bf, Layout::Packed, launching,
                                  &others[n++], &f)
                         : !check("gate", s.gate, shape, 2, bf, Layout::PaddedOuter, launching,
                                  &others[n++], &f))
      return fail(f.field, f.kind);
  }
  if (s.post_weight.rank != 0 &&
      !check("post_weight", s.post_weight, w_shape, 1, bf, Layout::Packed, launching,
             &others[n++], &f))
    return fail(f.field, f.kind);
  if ((s.pre_weight.rank != 0) != (s.x.rank != 0)) return fail("x", TQ_SHAPE);
  if (s.x.rank != 0 &&
      (!check("pre_weight", s.pre_weight, w_shape, 1, bf, Layout::Packed, launching,
              &others[n++], &f) ||
       !check("x", s.x, shape, 2, bf, Layout::PaddedOuter, launching, &x, &f)))
    return fail(f.field, f.kind);
  if (!check("out", s.out, shape, 2, kind, Layout::PaddedOuter, launching, &out, &f))
    return fail(f.field, f.kind);
  if (launching) {
    const TqTensorSpec* all[7] = {&s.y, &s.residual, &s.gate, &s.post_weight, &s.pre_weight,
                                  &s.out, &s.x};
    const char* names[7] = {"y", "residual", "gate", "post_weight", "pre_weight", "out", "x"};
    for (int i = 0; i < 7; ++i) {
      if (all[i]->rank == 0) continue;
      if (all[i]->device_address % 16) return fail(names[i], TQ_ALIGNMENT);
      if (all[i]->rank == 2 && all[i]->strides_bytes[0] % 16) return fail(names[i], TQ_STRIDE);
    }
  }
  if (!std::isfinite(s.scale)) return fail("scale", TQ_SCALE);
  if (s.post_weight.rank != 0 && !(std::isfinite(s.post_eps) && s.post_eps > 0.f))
    return fail("post_eps", TQ_SCALE);
  if (s.x.rank != 0 && !(std::isfinite(s.pre_eps) && s.pre_eps > 0.f))
    return fail("pre_eps", TQ_SCALE);
  // A row is read whole before any of it is written, so out over the residual and x over y are
  // fine row by row; any other overlap is not.
  Extent in[6];
  int m = 0;
  for (int i = 0; i < n; ++i) in[m++] = others[i];
  const int shared = m;
  in[m++] = y;
  if (!same_place(s.out, s.residual)) in[m++] = res;
  if (!check_aliases(in, m, &out, 1, &f)) return fail(f.field, f.kind);
  m = shared;
  in[m++] = res;
  in[m++] = out;
  if (s.x.rank != 0 && !same_place(s.x, s.y)) in[m++] = y;
  if (!check_aliases(in, m, &x, 1, &f)) return fail(f.field, f.kind);
  if (err) { err->field = nullptr; err->kind = TQ_OK; }
  return TQ_OK;
}

// Chunk attention: the attention plan's declarations with per-head widths and expansion weights.
int32_t chunk_validate_impl(const TqMlaChunkSpec* spec, TqContractError* err) {
  Failure f{nullptr, TQ_OK};
  auto fail = [&](const char* field, int32_t kind) {
    if (err) { err->field = field; err->kind = kind; }
    return kind;
  };
  if (!spec) return fail("spec", TQ_ERR_INVALID_ARGUMENT);
  const TqMlaChunkSpec& s = *spec;
  uint64_t payload = 0, dn = 256, dr = 0, dv = 256;
  switch (s.kv_format) {
    case TQ_KV_BF16: payload = 1024; break;
    case TQ_KV_FP8_E4M3: payload = 528; break;
    case TQ_KV_BF16_ROPE576: payload = 1152; dn = 128; dr = 64; dv = 128; break;
    default: return fail("kv_format", TQ_SHAPE);
  }
  if (s.q.rank != 3) return fail("q", TQ_SHAPE);
  const uint64_t T = s.q.shape[0], H = s.q.shape[1];
  if (H < 1 || H > 128 || T > (1u << 24)) return fail("q", TQ_SHAPE);
  if (!(std::isfinite(s.softmax_scale) && s.softmax_scale > 0.f))
    return fail("softmax_scale", TQ_SCALE);
  if (s.page_table.rank != 2) return fail("page_table", TQ_SHAPE);
  const uint64_t S = s.page_table.shape[0], L = s.page_table.shape[1];
  if (s.max_keys > (1u << 24) || s.max_keys + 127 * (S < T ? S : T) > (1u << 25))
    return fail("max_keys", TQ_CAPACITY);
  const bool launching = T != 0 && S != 0;
  if (!check_kv_strides(s.kv, payload, &f)) return fail(f.field, f.kind);
  const uint64_t q[3] = {T, H, dn + dr}, uk[3] = {H, dn, 512}, uv[3] = {H, dv, 512};
  const uint64_t pool[3] = {s.kv.shape[0], kPageRows, payload}, table[2] = {S, L};
  const uint64_t tok[1] = {T}, seqs[1] = {S}, starts[1] = {S + 1};
  const uint64_t o[3] = {T, H, dv}, l[2] = {T, H};
  if (s.kv.shape[0] >= kDimensionLimit / kPageRows) return fail("kv", TQ_DIMENSION);
  Extent in[8], out[2];
  const int32_t bf = TQ_DTYPE_BF16, i32 = TQ_DTYPE_I32;
  const Layout padded = Layout::PaddedOuter, packed = Layout::Packed;
  const int32_t out_dtype = s.out.dtype == TQ_DTYPE_F32 ? TQ_DTYPE_F32 : TQ_DTYPE_BF16;
  if (!check("q", s.q, q, 3, bf, padded, launching, &in[0], &f) ||
      !check("w_uk", s.w_uk, uk, 3, bf, padded, launching, &in[1], &f) ||
      !check("w_uv", s.w_uv, uv, 3, bf, padded, launching, &in[2], &f) ||
      !check("kv", s.kv, pool, 3, TQ_DTYPE_U8, Layout::Checked, launching, &in[3], &f) ||
      !check("page_table", s.page_table, table, 2, i32, packed, launching, &in[4], &f) ||
      !check("q_start", s.q_start, starts, 1, i32, packed, launching, &in[5], &f) ||
      !check("q_pos", s.q_pos, tok, 1, i32, packed, launching, &in[6], &f) ||
      !check("kv_len", s.kv_len, seqs, 1, i32, packed, launching, &in[7], &f) ||
      !check("out", s.out, o, 3, out_dtype, padded, launching, &out[0], &f))
    return fail(f.field, f.kind);
  out[1].present = false;
  if (s.lse.rank != 0 &&
      !check("lse", s.lse, l, 2, TQ_DTYPE_F32, packed, launching, &out[1], &f))
    return fail(f.field, f.kind);
  if (launching) {
    const TqTensorSpec* all[4] = {&s.q, &s.w_uk, &s.w_uv, &s.out};
    const char* names[4] = {"q", "w_uk", "w_uv", "out"};
    for (int i = 0; i < 4; ++i) {
      if (all[i]->device_address % 16) return fail(names[i], TQ_ALIGNMENT);
      if (all[i]->strides_bytes[0] % 16 || all[i]->strides_bytes[1] % 16)
        return fail(names[i], TQ_STRIDE);
    }
  }
  if (!check_aliases(in, 8, out, 2, &f)) return fail(f.field, f.kind);
  if (err) { err->field = nullptr; err->kind = TQ_OK; }
  return TQ_OK;
}

}  // namespace

int32_t chunk_validate(const TqMlaChunkSpec* spec, TqContractError* err) {
  return chunk_validate_impl(spec, err);
}

int32_t step_plan_validate(const TqStepPlanSpec* spec, TqContractError* err) {
  return step_plan_validate_impl(spec, err);
}

int32_t block_norm_validate(const TqBlockNormSpec* spec, TqContractError* err) {
  return block_norm_validate_impl(spec, err);
}

int32_t prologue_validate(const TqPrologueSpec* spec, TqContractError* err) {
  return prologue_validate_impl(spec, err);
}

bool params_intact(const TqMlaParams* p) { return p && p->digest == digest_of(*p); }

// ---------------------------------------------------------------------------------------------
// Philox4x32-10: ten rounds, key bumped by (W0, W1) per round (philox.rs:57-70).

void philox_block(const uint32_t counter[4], const uint32_t key[2], uint32_t out[4]) {
  uint32_t c0 = counter[0], c1 = counter[1], c2 = counter[2], c3 = counter[3];
  uint32_t k0 = key[0], k1 = key[1];
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = uint64_t(0xD2511F53u) * c0;
    const uint64_t p1 = uint64_t(0xCD9E8D57u) * c2;
    const uint32_t n0 = uint32_t(p1 >> 32) ^ c1 ^ k0;
    const uint32_t n2 = uint32_t(p0 >> 32) ^ c3 ^ k1;
    c1 = uint32_t(p1);
    c3 = uint32_t(p0);
    c0 = n0;
    c2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  out[0] = c0; out[1] = c1; out[2] = c2; out[3] = c3;
}

int32_t philox_words(uint64_t seed, uint64_t stream, uint64_t start, uint32_t* out,
                     uint64_t count) {
  if (count == 0) return TQ_OK;
  uint64_t last;
  if (add_overflows(start, count - 1, &last)) return TQ_ERR_RANGE;
  if (!out) return TQ_ERR_INVALID_ARGUMENT;
  const uint32_t key[2] = {uint32_t(seed), uint32_t(seed >> 32)};
  uint64_t i = start, written = 0;
  while (written < count) {
    const uint64_t group = i >> 2;
    const uint32_t counter[4] = {uint32_t(group), uint32_t(group >> 32), uint32_t(stream),
                                 uint32_t(stream >> 32)};
    uint32_t lanes[4];
    philox_block(counter, key, lanes);
    for (unsigned lane = unsigned(i & 3); lane < 4 && written < count; ++lane) {
      out[written++] = lanes[lane];
      ++i;
    }
  }
  return TQ_OK;
}

float philox_uniform_f32(uint32_t word) { return float(word >> 8) * (1.0f / 16777216.0f); }

}  // namespace tq

extern "C" {

int32_t tq_mla_validate(const TqMlaSpec* spec, const uint8_t* query_counts, uint64_t n,
                        TqMlaParams* params, TqContractError* err) {
  return tq::validate_impl(spec, query_counts, n, 4, params, err);
}

int32_t tq_mla_prefill_validate(const TqMlaSpec* spec, const uint32_t* query_counts, uint64_t n,
                                TqMlaParams* params, TqContractError* err) {
  return tq::validate_impl(spec, query_counts, n, 0, params, err);
}

int32_t tq_mla_sparse_validate(const TqMlaSpec* spec, const TqTensorSpec* idx,
                               const TqTensorSpec* k_len, const uint8_t* query_counts, uint64_t n,
                               TqMlaParams* params, TqContractError* err) {
  if (!idx || !k_len) {
    if (err) { err->field = "idx"; err->kind = TQ_ERR_INVALID_ARGUMENT; }
    return TQ_ERR_INVALID_ARGUMENT;
  }
  return tq::validate_impl(spec, query_counts, n, 4, params, err, idx, k_len);
}

int32_t tq_kv_write_validate(const TqKvWriteSpec* spec, TqContractError* err) {
  return tq::kv_write_validate_impl(spec, err);
}

int32_t tq_mla_prologue_validate(const TqPrologueSpec* spec, TqContractError* err) {
  return tq::prologue_validate(spec, err);
}

int32_t tq_step_plan_validate(const TqStepPlanSpec* spec, TqContractError* err) {
  return tq::step_plan_validate(spec, err);
}

int32_t tq_block_norm_validate(const TqBlockNormSpec* spec, TqContractError* err) {
  return tq::block_norm_validate(spec, err);
}

int32_t tq_mla_chunk_validate(const TqMlaChunkSpec* spec, TqContractError* err) {
  return tq::chunk_validate(spec, err);
}

int32_t tq_mla_should_launch(const TqMlaParams* params) {
  return tq::params_intact(params) ? params->should_launch : 0;
}

void tq_philox_block(const uint32_t counter[4], const uint32_t key[2], uint32_t out[4]) {
  tq::philox_block(counter, key, out);
}

int32_t tq_philox_words(uint64_t seed, uint64_t stream_id, uint64_t start, uint32_t* out,
                        uint64_t count) {
  return tq::philox_words(seed, stream_id, start, out, count);
}

float tq_philox_uniform_f32(uint32_t word) { return tq::philox_uniform_f32(word); }

const char* tq_mla_status_string(int32_t status) {
  switch (status) {
    case TQ_OK: return "ok";
    case TQ_SHAPE: return "Shape";
    case TQ_DTYPE: return "Dtype";
    case TQ_DIMENSION: return "Dimension";
    case TQ_STRIDE: return "Stride";
    case TQ_ALIGNMENT: return "Alignment";
    case TQ_ADDRESS: return "Address";
    case TQ_CAPACITY: return "Capacity";
    case TQ_OVERFLOW: return "Overflow";
    case TQ_QUERY_COUNT: return "QueryCount";
    case TQ_SCALE: return "Scale";
    case TQ_GROUP: return "Group";
    case TQ_ALIAS: return "Alias";
    case TQ_ERR_INVALID_ARGUMENT: return "invalid argument";
    case TQ_ERR_UNSUPPORTED: return "unsupported layout";
    case TQ_ERR_WORKSPACE: return "workspace missing, misaligned or too small";
    case TQ_ERR_CUDA: return "CUDA error";
    case TQ_ERR_PARAMS: return "params not produced by validation";
    case TQ_ERR_RANGE: return "word range exceeds u64";
    case TQ_ERR_COMM: return "NCCL unavailable or a collective failed";
    default: return "unknown status";
  }
}

}  // extern "C"
