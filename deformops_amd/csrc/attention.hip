// Cross attention: the checks of a call, its plan and its C entry points. The kernels are in
// attention.h.

#include "attention.h"

namespace {

using namespace attention;

constexpr int64_t kCus = 256;

int element_size(int dtype) { return dtype == MSDA_F32 ? 4 : dtype == MSDA_F16 || dtype == MSDA_BF16 ? 2 : 0; }

int64_t round_up(int64_t n) { return (n + 255) / 256 * 256; }

// Whether the kernels read these rows as they are: 16-byte pieces, and steps from row to row
// that a tile's 32-bit offsets hold and that tell the rows apart.
bool rows_as_they_are(const deformops_attention& c, const void* p, const int64_t (&strides)[3], int64_t rows) {
  const int size = element_size(c.dtype), n = 16 / size;
  return c.channels % n == 0 && aligned(p, 16) && strides[0] % n == 0 && strides[1] % n == 0 && strides[2] % n == 0 &&
         (rows <= 1 || (strides[1] >= c.channels && strides[1] * size <= (int64_t(1) << 23)));
}

// Words of a bool mask's row: of whole tiles of 128 keys.
int64_t mask_words(int64_t keys) { return ceil_div(keys, 128) * 4; }

// Where one operand's packed copy lies in the workspace, if it has one, and the threads that
// make it.
struct Packed {
  bool on;
  int64_t at, threads;
};

struct Plan {
  Variant variant;  // few_rows: tiles of 32 rows, which the waves share
  int splits;      // of an image's keys
  bool balanced;   // splits by the images' lengths
  int row_splits;  // of the rows, in the states' kernel
  int64_t forward_bytes, backward_bytes;
  int64_t delta_at, part_at, part_stats_at, part_k_at, part_v_at;
  Packed q, k, v, o, go, mask;
};

// `grad_output` and the output are dense: one packing rule for both by alignment (the size
// query assumes aligned ones, the launch checks).
Plan plan_of(const deformops_attention& c) {
  Plan p = {};
  const int64_t G = c.heads / c.key_heads, R = c.queries * G, BK = c.batch * c.key_heads;
  const int DP = padded(c.channels), size = element_size(c.dtype), n = 16 / size;
  p.variant.few_rows = R <= 64 && size * DP < 512;
  const int64_t rows = p.variant.few_rows ? 32 : 128, keys = p.variant.few_rows ? 128 : 64;
  const int64_t groups = BK * ceil_div(R, rows), tiles = ceil_div(c.keys, keys);
  // Pieces of the key axis (of the rows, in the states' kernel) where there is not a workgroup
  // for every CU, and then for as many as the card holds at once: one more would wait for a
  // whole turn. With a workgroup on every CU, the join costs more than fuller CUs give (7 x
  // 2,664 rows of 716 keys: 53 us in two pieces, 22 in one).
  auto pieces = [](int64_t groups, int waves, int64_t tiles) {
    if (groups >= kCus) return 1;
    return int(std::max<int64_t>(1, std::min<int64_t>(kCus * waves / std::max<int64_t>(1, groups), tiles / 2)));
  };
  // The LDS of a workgroup whose waves share the rows (ForwardShape), in KB of a CU's 160.
  const int tile = DP * (size == 4 ? 6 : 2) / 8, lds = 4 * tile <= 80 ? 4 * tile : std::max(2 * tile, DP / 2 + 1);
  const int lds_waves = p.variant.few_rows ? 160 / lds : 4;
  p.splits = pieces(groups, std::min(lds_waves, forward_waves(size, DP, c.mask_kind)), tiles);
  p.variant.fused = c.keys > 0 && c.keys <= 128 && fused_shape(c.dtype == MSDA_F16, size, DP);
  p.balanced = p.splits > 1 && c.key_lengths && c.batch > 1 && c.batch <= 64;
  const int64_t row_tile = DP * size <= 192 ? 64 : 32;
  const int64_t key_groups = BK * ceil_div(c.keys, 128), row_tiles = G * ceil_div(c.queries, row_tile);
  p.row_splits = pieces(key_groups, grad_states_waves(size, DP, c.mask_kind, p.variant.fused), row_tiles);

  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += round_up(bytes);
    return here;
  };
  const int64_t Dp = ceil_div(c.channels, n) * n;
  auto pack = [&](bool as_it_is, int64_t rows_of, int64_t heads) {
    const int64_t elements = c.batch * rows_of * heads * Dp;
    return as_it_is ? Packed{} : Packed{true, take(elements * size), elements / n};
  };
  p.q = pack(rows_as_they_are(c, c.query, c.query_strides, c.queries), c.queries, c.heads);
  p.k = pack(rows_as_they_are(c, c.key, c.key_strides, c.keys), c.keys, c.key_heads);
  p.v = pack(rows_as_they_are(c, c.value, c.value_strides, c.keys), c.keys, c.key_heads);
  const int64_t (&m)[4] = c.mask_strides;
  if (c.mask_kind != kNoMask && (c.mask_kind == kBoolMask || m[3] != 1 || c.keys < 4)) {
    const int64_t rows = (m[0] ? c.batch : 1) * (m[1] ? c.heads : 1) * (m[2] ? c.queries : 1);
    const bool bits = c.mask_kind == kBoolMask;
    const int64_t threads = rows * (bits ? mask_words(c.keys) : ceil_div(c.keys, 32) * 32);
    p.mask = Packed{true, take(threads * (bits ? 4 : element_size(c.mask_dtype))), threads};
  }
  // (The backward's sums of grad_q; none of them where that is fused.)
  p.part_at = take(p.splits > 1 ? p.splits * BK * R * c.channels * 4 : 0);
  const int64_t shared = at;
  p.part_stats_at = take(p.splits > 1 ? p.splits * BK * R * 8 : 0);
  p.forward_bytes = at;
  at = shared;
  const bool dense = c.channels % n == 0;
  p.o = pack(dense, c.queries, c.heads);
  p.go = pack(dense, c.queries, c.heads);
  p.delta_at = take(BK * R * 4);
  const int64_t states = p.row_splits > 1 ? p.row_splits * c.batch * c.keys * c.key_heads * c.channels * 4 : 0;
  p.part_k_at = take(states);
  p.part_v_at = take(states);
  p.backward_bytes = at;
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

template <typename F> void with_type(int dtype, F f);

// An operand's rows as the kernels read them, packed by a launch where they have to be.
Rows rows_of(const deformops_attention& c, const void* p, const int64_t (&strides)[3], Packed packed, int64_t rows,
             int64_t heads, char* workspace, hipStream_t s) {
  // The step past a single row may be anything; it bounds the tile's range of bytes.
  const Rows from = {p, strides[0], rows > 1 ? strides[1] : c.channels, strides[2]};
  if (!packed.on) return from;
  const int64_t n = 16 / element_size(c.dtype), Dp = ceil_div(c.channels, n) * n;
  void* to = workspace + packed.at;
  with_type(c.dtype, [&](auto t) {
    launch_pack<decltype(t)>(from, to, c.batch, rows, int(heads), int(c.channels), int(Dp), s);
  });
  return Rows{to, rows * heads * Dp, heads * Dp, Dp};
}

Args args_of(const deformops_attention& c, const Plan& p, void* workspace, hipStream_t s) {
  Args a = {};
  char* ws = static_cast<char*>(workspace);
  a.q = rows_of(c, c.query, c.query_strides, p.q, c.queries, c.heads, ws, s);
  a.k = rows_of(c, c.key, c.key_strides, p.k, c.keys, c.key_heads, ws, s);
  a.v = rows_of(c, c.value, c.value_strides, p.v, c.keys, c.key_heads, ws, s);
  if (c.mask_kind != kNoMask) {
    const int64_t (&m)[4] = c.mask_strides;
    a.mask = c.mask;
    a.mask_batch = m[0]; a.mask_head = m[1]; a.mask_row = m[2];
    a.mask_row_keys = int(c.keys);
    a.mask_type = c.mask_dtype;
    a.mask_of_keys = c.mask_kind == kBoolMask && (m[1] == 0 || c.heads == 1) && (m[2] == 0 || c.queries == 1);
    if (p.mask.on) {
      const int64_t images = m[0] ? c.batch : 1, heads = m[1] ? c.heads : 1, rows = m[2] ? c.queries : 1;
      const int64_t each = c.mask_kind == kBoolMask ? mask_words(c.keys) : ceil_div(c.keys, 32) * 32;
      const int64_t count = images * heads * rows * each;
      char* to = ws + p.mask.at;
      a.mask = to;
      a.mask_batch = m[0] ? heads * rows * each : 0;
      a.mask_head = m[1] ? rows * each : 0;
      a.mask_row = m[2] ? each : 0;
      a.mask_row_keys = int(each);
      const uint32_t groups = uint32_t(ceil_div(count, 256));
      auto pack = [&](auto v) {
        using V = decltype(v);
        attention_pack_mask_kernel<V><<<groups, 256, 0, s>>>(static_cast<const V*>(c.mask), reinterpret_cast<V*>(to), m[0],
                                                             m[1], m[2], m[3], int(heads), int(rows), int(c.keys),
                                                             int(each), count);
      };
      if (c.mask_kind == kBoolMask)
        attention_mask_bits_kernel<<<groups, 256, 0, s>>>(static_cast<const uint8_t*>(c.mask),
                                                          reinterpret_cast<uint32_t*>(to), m[0], m[1], m[2], m[3],
                                                          int(heads), int(rows), int(c.keys), int(each), count);
      else if (c.mask_dtype == MSDA_F32) pack(uint32_t());
      else pack(uint16_t());
    }
  }
  a.lengths = c.key_lengths;
  a.lengths_i64 = c.index_dtype == MSDA_I64;
  a.out = c.output;
  a.B = int(c.batch); a.Q = int(c.queries); a.S = int(c.keys); a.K = int(c.key_heads);
  a.G = int(c.heads / c.key_heads); a.D = int(c.channels);
  const int n = 16 / element_size(c.dtype);
  a.Dp = int(ceil_div(a.D, n) * n);
  a.R = uint32_t(c.queries * a.G);
  a.scale = c.scale;
  a.splits = p.splits;
  a.slots = p.splits * a.B;
  a.balanced = p.balanced;
  const int row_bytes = a.D * element_size(c.dtype);
  for (a.near = 1; a.near * row_bytes < 128 && a.K % (2 * a.near) == 0; a.near *= 2) {}
  a.row_splits = p.row_splits;
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

// A mask of no elements is not read, whatever its strides say: their zeros would look like axes
// that one element serves.
deformops_attention without_empty_mask(deformops_attention c) {
  if (c.queries == 0 || c.keys == 0) c.mask_kind = kNoMask;
  return c;
}

// Whether every launch of the call fits a grid: the walks' workgroups and the packed operands'.
int too_many(const Plan& p, int64_t groups) {
  for (const Packed* each : {&p.q, &p.k, &p.v, &p.o, &p.go, &p.mask})
    if (each->on) groups = std::max(groups, ceil_div(each->threads, 256));
  return groups > kMostGroups
             ? fail(MSDA_ERR_UNSUPPORTED, "cross attention: %lld workgroups pass a grid", static_cast<long long>(groups))
             : MSDA_OK;
}

int64_t row_groups(const deformops_attention& c, const Plan& p) {
  return c.batch * c.key_heads * ceil_div(c.queries * (c.heads / c.key_heads), p.variant.few_rows ? 32 : 128) * p.splits;
}

}  // namespace

extern "C" {

const char* deformops_last_error(void) { return g_error; }

int deformops_cross_attention_workspace_size(const deformops_attention* call, int64_t* forward, int64_t* backward) {
  if (const int e = check(call)) return e;
  const deformops_attention given = without_empty_mask(*call), *c = &given;
  if (!forward || !backward) return fail(MSDA_ERR_INVALID, "cross attention: null result");
  const Plan p = plan_of(*c);
  *forward = p.forward_bytes;
  *backward = p.backward_bytes;
  return MSDA_OK;
}

int deformops_cross_attention_forward(const deformops_attention* call, void* row_stats, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  if (const int e = check(call)) return e;
  const deformops_attention given = without_empty_mask(*call), *c = &given;
  if (c->batch == 0 || c->queries == 0) return MSDA_OK;
  if (!c->query || !c->output || (c->keys && (!c->key || !c->value)) || (c->mask_kind && !c->mask))
    return fail(MSDA_ERR_INVALID, "cross attention: null tensor");
  const Plan p = plan_of(*c);
  if (p.forward_bytes && (!workspace || workspace_bytes < p.forward_bytes || !aligned(workspace, 256)))
    return fail(MSDA_ERR_INVALID, "cross attention: the workspace must hold %lld bytes, aligned to 256",
                static_cast<long long>(p.forward_bytes));
  const int64_t groups = row_groups(*c, p);
  if (const int e = too_many(p, groups)) return e;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  Args a = args_of(*c, p, workspace, s);
  a.stats = static_cast<float2*>(row_stats);
  a.out_vector = a.D % 4 == 0 && aligned(c->output, 16);
  with_type(c->dtype, [&](auto t) { launch_forward<decltype(t)>(a, c->mask_kind, p.variant, uint32_t(groups), s); });
  return launched("cross attention forward");
}

int deformops_cross_attention_backward(const deformops_attention* call, const void* row_stats, const void* grad_output,
                                       void* grad_query, void* grad_key, void* grad_value, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  if (const int e = check(call)) return e;
  const deformops_attention given = without_empty_mask(*call), *c = &given;
  if (c->batch == 0 || (c->queries == 0 && c->keys == 0)) return MSDA_OK;
  if ((c->queries && (!c->query || !c->output || !row_stats || !grad_output || !grad_query)) ||
      (c->keys && (!c->key || !c->value || !grad_key || !grad_value)) ||
      (c->mask_kind && !c->mask))
    return fail(MSDA_ERR_INVALID, "cross attention: null tensor");
  const Plan p = plan_of(*c);
  if (p.backward_bytes && (!workspace || workspace_bytes < p.backward_bytes || !aligned(workspace, 256)))
    return fail(MSDA_ERR_INVALID, "cross attention: the workspace must hold %lld bytes, aligned to 256",
                static_cast<long long>(p.backward_bytes));
  const int n = 16 / element_size(c->dtype);
  if (!aligned(c->output, 16) || !aligned(grad_output, 16))
    return fail(MSDA_ERR_INVALID, "cross attention: output and grad_output must be aligned to 16 bytes");
  const int64_t groups = row_groups(*c, p);
  const int64_t key_groups = c->batch * c->key_heads * ceil_div(c->keys, 128) * p.row_splits;
  if (const int e = too_many(p, std::max(groups, key_groups))) return e;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  Args a = args_of(*c, p, workspace, s);
  const int64_t dense[3] = {c->queries * c->heads * c->channels, c->heads * c->channels, c->channels};
  a.o = rows_of(*c, c->output, dense, p.o, c->queries, c->heads, static_cast<char*>(workspace), s);
  a.go = rows_of(*c, grad_output, dense, p.go, c->queries, c->heads, static_cast<char*>(workspace), s);
  a.row_stats = static_cast<const float2*>(row_stats);
  a.grad_q = grad_query;
  a.grad_k = grad_key;
  a.grad_v = grad_value;
  a.out_vector = a.D % n == 0 && aligned(grad_query, 16) && aligned(grad_key, 16) && aligned(grad_value, 16);
  with_type(c->dtype, [&](auto t) {
    launch_backward<decltype(t)>(a, c->mask_kind, p.variant, uint32_t(groups), uint32_t(key_groups), s);
  });
  return launched("cross attention backward");
}

}  // extern "C"
