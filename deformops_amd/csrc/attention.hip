// Cross attention: the checks of a call, its plan and its C entry points. The kernels are in
// attention.h.

#include "attention.h"

namespace {

using namespace attention;

constexpr int kWanted = 512;  // workgroups that fill 256 CUs twice

int element_size(int dtype) { return dtype == MSDA_F32 ? 4 : dtype == MSDA_F16 || dtype == MSDA_BF16 ? 2 : 0; }

struct Plan {
  bool few_rows;   // one row tile of 32: the waves share the rows
  int splits;      // of the keys
  int row_splits;  // of the rows, in the states' kernel
  int64_t forward_bytes, backward_bytes;
  int64_t delta_at, part_at, part_stats_at, part_k_at, part_v_at;
};

int64_t round_up(int64_t n) { return (n + 255) / 256 * 256; }

Plan plan_of(const deformops_attention& c) {
  Plan p = {};
  const int64_t G = c.heads / c.key_heads, R = c.queries * G, BK = c.batch * c.key_heads;
  const int DP = padded(c.channels), size = element_size(c.dtype);
  p.few_rows = R <= 64 && size * DP < 512;
  const int64_t rows = p.few_rows ? 32 : 128, keys = p.few_rows ? 128 : 64;
  const int64_t groups = BK * ceil_div(R, rows), tiles = ceil_div(c.keys, keys);
  p.splits = int(std::max<int64_t>(1, std::min<int64_t>(ceil_div(kWanted, std::max<int64_t>(1, groups)), tiles / 2)));
  const int64_t row_tile = DP * size <= 192 ? 64 : 32;
  const int64_t key_groups = BK * ceil_div(c.keys, 128), row_tiles = ceil_div(R, row_tile);
  p.row_splits = int(std::max<int64_t>(1, std::min<int64_t>(ceil_div(kWanted, std::max<int64_t>(1, key_groups)), row_tiles / 2)));

  const int64_t part = p.splits > 1 ? round_up(p.splits * BK * R * c.channels * 4) : 0;
  p.part_at = 0;
  p.part_stats_at = part;
  p.forward_bytes = part + (p.splits > 1 ? round_up(p.splits * BK * R * 8) : 0);
  p.delta_at = part;
  const int64_t states = p.row_splits > 1 ? round_up(p.row_splits * c.batch * c.keys * c.key_heads * c.channels * 4) : 0;
  p.part_k_at = part + round_up(BK * R * 4);
  p.part_v_at = p.part_k_at + states;
  p.backward_bytes = p.part_v_at + states;
  return p;
}

int check(const deformops_attention* c) {
  if (!c) return fail(MSDA_ERR_INVALID, "cross attention: null call");
  const int size = element_size(c->dtype);
  if (!size) return fail(MSDA_ERR_INVALID, "cross attention: dtype %d is not float32, float16 or bfloat16", c->dtype);
  if (c->batch < 0 || c->queries < 0 || c->keys < 0 || c->heads <= 0 || c->key_heads <= 0 || c->channels <= 0)
    return fail(MSDA_ERR_INVALID, "cross attention: a size is negative, or no heads or channels");
  if (c->heads % c->key_heads)
    return fail(MSDA_ERR_INVALID, "cross attention: %lld heads are not a multiple of %lld key heads",
                static_cast<long long>(c->heads), static_cast<long long>(c->key_heads));
  if (c->channels > 128)
    return fail(MSDA_ERR_UNSUPPORTED, "cross attention: %lld channels per head; the kernels take up to 128",
                static_cast<long long>(c->channels));
  constexpr int64_t kMost = (int64_t(1) << 31) - 256;
  if (c->keys > kMost || c->queries > kMost || c->heads > kMost || c->queries * (c->heads / c->key_heads) > kMost ||
      c->batch > kMost || c->batch * c->key_heads > kMost)
    return fail(MSDA_ERR_UNSUPPORTED, "cross attention: a size passes 2^31");
  if (!(c->scale > 0.0f) || !isfinite(c->scale))
    return fail(MSDA_ERR_INVALID, "cross attention: scale must be positive and finite");
  if (c->mask_kind < 0 || c->mask_kind > 2 || (c->mask_kind == kFloatMask && !element_size(c->mask_dtype)))
    return fail(MSDA_ERR_INVALID, "cross attention: unknown kind or dtype of mask");
  if (c->key_lengths && c->index_dtype != MSDA_I64 && c->index_dtype != MSDA_I32)
    return fail(MSDA_ERR_INVALID, "cross attention: key_lengths are int64 or int32");
  return MSDA_OK;
}

bool rows_aligned(const deformops_attention& c, const void* p, const int64_t (&strides)[3]) {
  const int n = 16 / element_size(c.dtype);
  return aligned(p, 16) && strides[0] % n == 0 && strides[1] % n == 0 && strides[2] % n == 0;
}

Args args_of(const deformops_attention& c, const Plan& p, void* workspace) {
  Args a = {};
  a.q = c.query; a.k = c.key; a.v = c.value;
  a.q_batch = c.query_strides[0]; a.q_row = c.query_strides[1]; a.q_head = c.query_strides[2];
  a.k_batch = c.key_strides[0]; a.k_row = c.key_strides[1]; a.k_head = c.key_strides[2];
  a.v_batch = c.value_strides[0]; a.v_row = c.value_strides[1]; a.v_head = c.value_strides[2];
  if (c.mask_kind != kNoMask) {
    const int size = c.mask_kind == kBoolMask ? 1 : element_size(c.mask_dtype);
    a.mask = c.mask;
    a.mask_batch = c.mask_strides[0]; a.mask_head = c.mask_strides[1];
    a.mask_row = c.mask_strides[2]; a.mask_key = c.mask_strides[3];
    a.mask_type = c.mask_dtype;
    a.mask_quads = c.mask_strides[3] == 1 && aligned(c.mask, 4 * size) && c.mask_strides[0] % 4 == 0 &&
                   c.mask_strides[1] % 4 == 0 && c.mask_strides[2] % 4 == 0;
    a.mask_of_keys = c.mask_kind == kBoolMask && (c.mask_strides[1] == 0 || c.heads == 1) &&
                     (c.mask_strides[2] == 0 || c.queries == 1);
  }
  a.lengths = c.key_lengths;
  a.lengths_i64 = c.index_dtype == MSDA_I64;
  a.out = c.output;
  a.B = int(c.batch); a.Q = int(c.queries); a.S = int(c.keys); a.K = int(c.key_heads);
  a.G = int(c.heads / c.key_heads); a.D = int(c.channels);
  a.R = uint32_t(c.queries * a.G);
  a.scale = c.scale;
  const int n = 16 / element_size(c.dtype);
  a.vector = a.D % n == 0 && rows_aligned(c, c.query, c.query_strides) && rows_aligned(c, c.key, c.key_strides) &&
             rows_aligned(c, c.value, c.value_strides);
  a.splits = p.splits;
  a.row_splits = p.row_splits;
  char* ws = static_cast<char*>(workspace);
  a.part = reinterpret_cast<float*>(ws + p.part_at);
  a.part_stats = reinterpret_cast<float2*>(ws + p.part_stats_at);
  a.delta = reinterpret_cast<float*>(ws + p.delta_at);
  a.part_k = reinterpret_cast<float*>(ws + p.part_k_at);
  a.part_v = reinterpret_cast<float*>(ws + p.part_v_at);
  return a;
}

template <typename F> void with_type(int dtype, F f) {
  if (dtype == MSDA_F32) f(float());
  else if (dtype == MSDA_F16) f(f16_t());
  else f(bf16_t());
}

int too_many(int64_t groups) {
  return groups > (int64_t(1) << 31) - 1
             ? fail(MSDA_ERR_UNSUPPORTED, "cross attention: %lld workgroups pass a grid", static_cast<long long>(groups))
             : MSDA_OK;
}

}  // namespace

extern "C" {

const char* deformops_last_error(void) { return g_error; }

int deformops_cross_attention_workspace_size(const deformops_attention* c, int64_t* forward, int64_t* backward) {
  if (const int e = check(c)) return e;
  if (!forward || !backward) return fail(MSDA_ERR_INVALID, "cross attention: null result");
  const Plan p = plan_of(*c);
  *forward = p.forward_bytes;
  *backward = p.backward_bytes;
  return MSDA_OK;
}

int deformops_cross_attention_forward(const deformops_attention* c, void* row_stats, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  if (const int e = check(c)) return e;
  if (c->batch == 0 || c->queries == 0) return MSDA_OK;
  if (!c->query || !c->output || (c->keys && (!c->key || !c->value)) || (c->keys && c->mask_kind && !c->mask))
    return fail(MSDA_ERR_INVALID, "cross attention: null tensor");
  const Plan p = plan_of(*c);
  if (p.forward_bytes && (!workspace || workspace_bytes < p.forward_bytes || !aligned(workspace, 256)))
    return fail(MSDA_ERR_INVALID, "cross attention: the workspace must hold %lld bytes, aligned to 256",
                static_cast<long long>(p.forward_bytes));
  Args a = args_of(*c, p, workspace);
  a.stats = static_cast<float2*>(row_stats);
  a.out_vector = a.D % 4 == 0 && aligned(c->output, 16);
  const int64_t rows = p.few_rows ? 32 : 128;
  const int64_t groups = int64_t(a.B) * a.K * ceil_div(a.R, rows) * a.splits;
  if (const int e = too_many(groups)) return e;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  with_type(c->dtype, [&](auto t) { launch_forward<decltype(t)>(a, c->mask_kind, p.few_rows, uint32_t(groups), s); });
  return launched("cross attention forward");
}

int deformops_cross_attention_backward(const deformops_attention* c, const void* row_stats, const void* grad_output,
                                       void* grad_query, void* grad_key, void* grad_value, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  if (const int e = check(c)) return e;
  if (c->batch == 0 || (c->queries == 0 && c->keys == 0)) return MSDA_OK;
  if ((c->queries && (!c->query || !c->output || !row_stats || !grad_output || !grad_query)) ||
      (c->keys && (!c->key || !c->value || !grad_key || !grad_value)) ||
      (c->keys && c->queries && c->mask_kind && !c->mask))
    return fail(MSDA_ERR_INVALID, "cross attention: null tensor");
  const Plan p = plan_of(*c);
  if (p.backward_bytes && (!workspace || workspace_bytes < p.backward_bytes || !aligned(workspace, 256)))
    return fail(MSDA_ERR_INVALID, "cross attention: the workspace must hold %lld bytes, aligned to 256",
                static_cast<long long>(p.backward_bytes));
  Args a = args_of(*c, p, workspace);
  a.row_stats = static_cast<const float2*>(row_stats);
  a.grad_out = grad_output;
  a.grad_q = grad_query;
  a.grad_k = grad_key;
  a.grad_v = grad_value;
  const int n = 16 / element_size(c->dtype);
  a.out_vector = a.D % n == 0 && aligned(c->output, 16) && aligned(grad_output, 16) && aligned(grad_query, 16) &&
                 aligned(grad_key, 16) && aligned(grad_value, 16);
  const int64_t rows = p.few_rows ? 32 : 128;
  const int64_t groups = int64_t(a.B) * a.K * ceil_div(a.R, rows) * a.splits;
  const int64_t key_groups = int64_t(a.B) * a.K * ceil_div(a.S, 128) * a.row_splits;
  if (const int e = too_many(std::max(groups, key_groups))) return e;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  with_type(c->dtype, [&](auto t) {
    launch_backward<decltype(t)>(a, c->mask_kind, p.few_rows, uint32_t(groups), uint32_t(key_groups), s);
  });
  return launched("cross attention backward");
}

}  // extern "C"
