// Operator layer of the full-attention step: page plans, rotary positions with cache stores, attention.
#include "ops.hpp"

#include <algorithm>
#include <cmath>

namespace tk100 {

namespace {

#define TK100_TRY(expr)                  \
  do {                                   \
    Status _s = (expr);                  \
    if (_s != TK100_OK) return _s;       \
  } while (0)

constexpr int kMaxTokens = 1 << 24;          // rows of one launch
constexpr int kMaxSequences = 1 << 20;
constexpr long long kMaxKeys = 1ll << 30;    // keys of one sequence
constexpr int kAttentionRows = 128;          // rows of a tile (attention.cu)
constexpr size_t kTicketBytes = 4096;

// The caller's current device is the context's during a launch, whatever it was.
class DeviceScope {
 public:
  DeviceScope(Context& ctx) : ctx_(ctx) {
    status_ = cudaGetDevice(&before_);
    if (status_ == cudaSuccess && before_ != ctx.config().device) {
      status_ = cudaSetDevice(ctx.config().device);
      moved_ = status_ == cudaSuccess;
    }
  }
  ~DeviceScope() {
    if (moved_) cudaSetDevice(before_);
  }
  Status status() { return ctx_.check(status_, "making the context's device current"); }

 private:
  Context& ctx_;
  cudaError_t status_;
  int before_ = 0;
  bool moved_ = false;
};

Status refuse(Context& ctx, const char* what, const std::string& message) {
  return ctx.fail(TK100_ERR_LAUNCH, std::string("[gpu.launch] ") + what + ": " + message);
}

Status plane(Context& ctx, const char* what, const char* name, const void* p, size_t alignment) {
  if (p == nullptr) return refuse(ctx, what, std::string(name) + " plane is null");
  if ((reinterpret_cast<uintptr_t>(p) & (alignment - 1)) != 0)
    return refuse(ctx, what, std::string(name) + " plane is not " + std::to_string(alignment) + "-byte aligned");
  return TK100_OK;
}

Status range(Context& ctx, const char* what, const char* name, long long v, long long low, long long high) {
  if (v >= low && v <= high) return TK100_OK;
  return refuse(ctx, what, std::string(name) + " " + std::to_string(v) + " is outside the admitted range " +
                               std::to_string(low) + "..=" + std::to_string(high));
}

// Rows are read 16 bytes at a time: strides in whole groups of eight values.
Status stride(Context& ctx, const char* what, const char* name, int v, int least) {
  if (v >= least && v % 8 == 0) return TK100_OK;
  return refuse(ctx, what, std::string(name) + " stride " + std::to_string(v) + " is not a multiple of 8 of at least " +
                               std::to_string(least));
}

Status heads(Context& ctx, const char* what, int q_heads, int kv_heads, int head_dim) {
  if (head_dim != 128 && head_dim != 256)
    return refuse(ctx, what, "heads of " + std::to_string(head_dim) + " values are not admitted (128 or 256)");
  TK100_TRY(range(ctx, what, "key/value head count", kv_heads, 1, 1024));
  if (q_heads < kv_heads || q_heads % kv_heads != 0 || q_heads / kv_heads > kAttentionRows)
    return refuse(ctx, what, std::to_string(q_heads) + " query heads do not share " + std::to_string(kv_heads) +
                                 " key/value heads evenly, at most 128 each");
  return TK100_OK;
}

Status cache_geometry(Context& ctx, const char* what, const CacheGeometry& g, int head_dim) {
  TK100_TRY(range(ctx, what, "page count", g.pages, 1, 1 << 30));
  if (g.page_tokens < 16 || g.page_tokens > (1 << 20) || (g.page_tokens & (g.page_tokens - 1)) != 0)
    return refuse(ctx, what, "pages of " + std::to_string(g.page_tokens) + " tokens are not admitted (a power of two, 16 to 2^20)");
  TK100_TRY(stride(ctx, what, "cache page", g.page_stride, head_dim));
  TK100_TRY(stride(ctx, what, "cache token", g.token_stride, head_dim));
  return stride(ctx, what, "cache head", g.head_stride, head_dim);
}

int log2_of(int power) {
  int s = 0;
  while ((1 << s) < power) ++s;
  return s;
}

// [first, last) bytes that `tokens` rows of `heads` heads touch
struct Span {
  uintptr_t first, last;
  Span(const uint16_t* p, long long tokens, long long token_stride, long long heads, long long head_stride, int dim)
      : first(reinterpret_cast<uintptr_t>(p)),
        last(first + 2 * static_cast<uintptr_t>((tokens - 1) * token_stride + (heads - 1) * head_stride + dim)) {}
  // the same for a cache plane, from its first page to its last
  Span(const uint16_t* p, const CacheGeometry& g, int heads, int dim) : Span(p, g.page_tokens, g.token_stride, heads, g.head_stride, dim) {
    last += 2 * static_cast<uintptr_t>(static_cast<long long>(g.pages - 1) * g.page_stride);
  }
  bool meets(const Span& o) const { return first < o.last && o.first < last; }
};

// Whether two planes of the same extents and strides, the second `apart` values behind the first, have one in common:
// whether multiples of the strides, each below its extent either way, add up to less than `least` from `apart`.
// Strides fall; where they nest, as a plane's do whose own values lie apart, two multiples of each come near enough at
// most.  Where many do, the answer is yes.
struct Dimension {
  long long extent, stride;
};
bool planes_share(long long apart, const Dimension* dims, int count, long long least) {
  if (count == 0) return apart > -least && apart < least;
  const long long extent = dims[0].extent, stride = dims[0].stride;
  long long reach = least - 1;  // of what is left, either way
  for (int i = 1; i < count; ++i) reach += (dims[i].extent - 1) * dims[i].stride;
  auto below = [](long long a, long long b) { return a / b - (a % b < 0); };  // a / b rounded down, b > 0
  const long long from = std::max(-below(reach - apart, stride), 1 - extent), to = std::min(below(apart + reach, stride), extent - 1);
  if (to - from > 2) return true;
  for (long long m = from; m <= to; ++m)
    if (planes_share(apart - m * stride, dims + 1, count - 1, least)) return true;
  return false;
}

bool caches_share(const uint16_t* key, const uint16_t* value, const CacheGeometry& g, int heads, int dim) {
  Dimension dims[3] = {{g.pages, g.page_stride}, {g.page_tokens, g.token_stride}, {heads, g.head_stride}};
  std::sort(dims, dims + 3, [](const Dimension& a, const Dimension& b) { return a.stride > b.stride; });
  return planes_share((reinterpret_cast<intptr_t>(value) - reinterpret_cast<intptr_t>(key)) / 2, dims, 3, dim);
}

}  // namespace

// ---------------------------------------------------------------------- PagePlanOp

Status PagePlanOp::check(const char* what, const PageParams& p) {
  TK100_TRY(range(ctx_, what, "request count", p.requests, 1, kPageMaxRequests));
  TK100_TRY(range(ctx_, what, "block table row count", p.table_rows, 1, kPageMaxRows));
  TK100_TRY(range(ctx_, what, "pages per row", p.max_pages, 1, 1 << 30));
  if (p.page_tokens < 16 || p.page_tokens > (1 << 20) || (p.page_tokens & (p.page_tokens - 1)) != 0)
    return refuse(ctx_, what, "pages of " + std::to_string(p.page_tokens) + " tokens are not admitted (a power of two, 16 to 2^20)");
  // more pages than that hold more keys than a sequence may have
  if (static_cast<long long>(p.max_pages) * p.page_tokens > kMaxKeys)
    return refuse(ctx_, what, "a block table row of " + std::to_string(p.max_pages) + " pages exceeds 2^30 tokens");
  TK100_TRY(range(ctx_, what, "free page capacity", p.free_capacity, 1, 1 << 30));
  TK100_TRY(plane(ctx_, what, "length", p.lengths, 4));
  TK100_TRY(plane(ctx_, what, "length output", p.lengths_output, 4));
  TK100_TRY(plane(ctx_, what, "block table", p.block_table, 4));
  TK100_TRY(plane(ctx_, what, "free page", p.free_pages, 4));
  TK100_TRY(plane(ctx_, what, "free count", p.free_count, 4));
  return plane(ctx_, what, "free count output", p.free_count_output, 4);
}

Status PagePlanOp::launch(cudaStream_t stream, PageParams p) {
  const char* what = "page plan";
  TK100_TRY(check(what, p));
  TK100_TRY(range(ctx_, what, "token capacity", p.max_tokens, 1, kMaxTokens));
  TK100_TRY(plane(ctx_, what, "new token", p.new_tokens, 4));
  TK100_TRY(plane(ctx_, what, "start", p.starts, 4));
  TK100_TRY(plane(ctx_, what, "key length", p.kv_lengths, 4));
  TK100_TRY(plane(ctx_, what, "position", p.positions, 4));
  TK100_TRY(plane(ctx_, what, "slot", p.slots, 8));
  p.status = ctx_.status_word();
  DeviceScope device(ctx_);
  TK100_TRY(device.status());
  ctx_.count_launch();
  return ctx_.check(launch_page(stream, p, false), "launching the page plan");
}

Status PagePlanOp::release(cudaStream_t stream, PageParams p) {
  const char* what = "page release";
  TK100_TRY(check(what, p));
  p.status = ctx_.status_word();
  DeviceScope device(ctx_);
  TK100_TRY(device.status());
  ctx_.count_launch();
  return ctx_.check(launch_page(stream, p, true), "launching the page release");
}

// ------------------------------------------------------------------- RotaryCacheOp

Status RotaryCacheOp::launch(cudaStream_t stream, int head_dim, RotaryParams p, const CacheGeometry& cache) {
  const char* what = "rotary";
  TK100_TRY(heads(ctx_, what, p.q_heads, p.kv_heads, head_dim));
  TK100_TRY(range(ctx_, what, "token count", p.tokens, 1, kMaxTokens));
  if (p.half < 8 || p.half % 8 != 0 || 2 * p.half > head_dim)
    return refuse(ctx_, what, std::to_string(2 * p.half) + " rotated values are not admitted (a multiple of 16 up to the head's)");
  TK100_TRY(range(ctx_, what, "position axis count", p.axes, 1, 8));
  TK100_TRY(plane(ctx_, what, "frequency", p.frequencies, 8));
  TK100_TRY(plane(ctx_, what, "position", p.positions, 4));
  TK100_TRY(plane(ctx_, what, "query", p.query, 16));
  TK100_TRY(plane(ctx_, what, "key", p.key, 16));
  TK100_TRY(plane(ctx_, what, "query output", p.query_output, 16));
  TK100_TRY(stride(ctx_, what, "query token", p.query_token_stride, head_dim));
  TK100_TRY(stride(ctx_, what, "query head", p.query_head_stride, head_dim));
  TK100_TRY(stride(ctx_, what, "key/value token", p.kv_token_stride, head_dim));
  TK100_TRY(stride(ctx_, what, "key/value head", p.kv_head_stride, head_dim));
  if (p.query_norm) TK100_TRY(plane(ctx_, what, "query norm", p.query_norm, 16));
  if (p.key_norm) TK100_TRY(plane(ctx_, what, "key norm", p.key_norm, 16));
  if (p.key_output) TK100_TRY(plane(ctx_, what, "key output", p.key_output, 16));
  if (p.key_cache || p.value_cache) {
    TK100_TRY(cache_geometry(ctx_, what, cache, head_dim));
    TK100_TRY(plane(ctx_, what, "key cache", p.key_cache, 16));
    TK100_TRY(plane(ctx_, what, "value cache", p.value_cache, 16));
    TK100_TRY(plane(ctx_, what, "value", p.value, 16));
    TK100_TRY(plane(ctx_, what, "slot", p.slots, 8));
    p.pages = cache.pages;
    p.page_shift = log2_of(cache.page_tokens);
    p.page_stride = cache.page_stride;
    p.cache_token_stride = cache.token_stride;
    p.cache_head_stride = cache.head_stride;
  } else if (!p.key_output) {
    return refuse(ctx_, what, "rotated keys go nowhere: neither a key output nor a cache");
  }
  // An output may be the plane it is computed from, element for element; any other overlap would have one CTA write
  // what another still reads, or two CTAs write one place.
  const Span query(p.query, p.tokens, p.query_token_stride, p.q_heads, p.query_head_stride, head_dim);
  const Span key(p.key, p.tokens, p.kv_token_stride, p.kv_heads, p.kv_head_stride, head_dim);
  const Span q_out(p.query_output, p.tokens, static_cast<long long>(p.q_heads) * head_dim, p.q_heads, head_dim, head_dim);
  const bool q_same = p.query_output == p.query && p.query_head_stride == head_dim &&
                      p.query_token_stride == p.q_heads * head_dim;
  if (q_out.meets(query) && !q_same) return refuse(ctx_, what, "the query output overlaps the queries");
  if (q_out.meets(key)) return refuse(ctx_, what, "the query output overlaps the keys");
  if (p.key_output) {
    const Span k_out(p.key_output, p.tokens, static_cast<long long>(p.kv_heads) * head_dim, p.kv_heads, head_dim, head_dim);
    const bool k_same = p.key_output == p.key && p.kv_head_stride == head_dim && p.kv_token_stride == p.kv_heads * head_dim;
    if (k_out.meets(key) && !k_same) return refuse(ctx_, what, "the key output overlaps the keys");
    if (k_out.meets(query) || k_out.meets(q_out)) return refuse(ctx_, what, "the key output overlaps the queries or their output");
  }
  if (p.key_cache) {
    const Span value(p.value, p.tokens, p.kv_token_stride, p.kv_heads, p.kv_head_stride, head_dim);
    if (q_out.meets(value)) return refuse(ctx_, what, "the query output overlaps the values");
    const Span k_out = !p.key_output ? key
                                     : Span(p.key_output, p.tokens, static_cast<long long>(p.kv_heads) * head_dim, p.kv_heads,
                                            head_dim, head_dim);
    if (p.key_output && k_out.meets(value)) return refuse(ctx_, what, "the key output overlaps the values");
    const Span caches[2] = {{p.key_cache, cache, p.kv_heads, head_dim}, {p.value_cache, cache, p.kv_heads, head_dim}};
    for (const Span& c : caches) {
      const char* other = c.meets(query) ? "queries" : c.meets(key) ? "keys" : c.meets(value) ? "values"
                          : c.meets(q_out) ? "query output" : c.meets(k_out) ? "key output" : nullptr;
      if (other) return refuse(ctx_, what, std::string("a cache overlaps the ") + other);
    }
    if (caches_share(p.key_cache, p.value_cache, cache, p.kv_heads, head_dim))
      return refuse(ctx_, what, "the key cache overlaps the value cache");
  }
  p.epsilon = ctx_.config().rms_norm_epsilon;
  p.status = ctx_.status_word();
  DeviceScope device(ctx_);
  TK100_TRY(device.status());
  ctx_.count_launch();
  return ctx_.check(launch_rotary(stream, head_dim, p), "launching the rotary positions");
}

// --------------------------------------------------------------------- AttentionOp

size_t AttentionOp::workspace_bytes(int sms, int head_dim) {
  const size_t rows = 2 * static_cast<size_t>(sms) * kAttentionRows;
  return kTicketBytes + rows * sizeof(float2) + rows * head_dim * sizeof(float);
}

Status AttentionOp::prepare(const char* what, int head_dim, AttentionParams* p, const uint16_t* query, const uint16_t* key,
                            const uint16_t* value, float scale, void* workspace) {
  TK100_TRY(heads(ctx_, what, p->q_heads, p->kv_heads, head_dim));
  TK100_TRY(range(ctx_, what, "token count", p->tokens, 1, kMaxTokens));
  TK100_TRY(range(ctx_, what, "sequence count", p->sequences, 1, kMaxSequences));
  TK100_TRY(plane(ctx_, what, "start", p->starts, 4));
  TK100_TRY(plane(ctx_, what, "query", query, 16));
  TK100_TRY(plane(ctx_, what, "key", key, 16));
  TK100_TRY(plane(ctx_, what, "value", value, 16));
  TK100_TRY(plane(ctx_, what, "output", p->output, 32));
  TK100_TRY(plane(ctx_, what, "workspace", workspace, 16));
  TK100_TRY(stride(ctx_, what, "query token", p->query_token_stride, head_dim));
  TK100_TRY(stride(ctx_, what, "query head", p->query_head_stride, head_dim));
  if (p->gate) {
    TK100_TRY(plane(ctx_, what, "gate", p->gate, 16));
    TK100_TRY(stride(ctx_, what, "gate token", p->gate_token_stride, head_dim));
    TK100_TRY(stride(ctx_, what, "gate head", p->gate_head_stride, head_dim));
  }
  if (!(scale > 0.0f) || !std::isfinite(scale)) return refuse(ctx_, what, "the scale must be positive and finite");
  const Span out(p->output, p->tokens, static_cast<long long>(p->q_heads) * head_dim, p->q_heads, head_dim, head_dim);
  const Span in(query, p->tokens, p->query_token_stride, p->q_heads, p->query_head_stride, head_dim);
  if (out.meets(in)) return refuse(ctx_, what, "the output overlaps the queries");
  if (p->gate) {
    const Span gate(p->gate, p->tokens, p->gate_token_stride, p->q_heads, p->gate_head_stride, head_dim);
    if (out.meets(gate)) return refuse(ctx_, what, "the output overlaps the gate");
  }
  p->group = p->q_heads / p->kv_heads;
  p->half_tokens = kAttentionRows / p->group;
  p->tile_tokens = 2 * p->half_tokens;
  p->scale_log2 = scale * 1.4426950408889634f;
  // A tile's first scores and last rows, in keys of the line: too little gives pairs with many short tiles more than
  // their share, too much less.  480 / 608 / 768 at heads of 256, us: a prompt of 8192 tokens 753 / 732 / 741, seven packed
  // prompts 111 / 115 / 122, a decode batch of 32 203 / 193 / 190 (its tiles' ends cost more than this line says); 192 / 256 / 320 at
  // 128: seven packed prompts 90 / 89 / 91, nine mixed chunks 60 / 60 / 60.  256 at heads of 256 707 for the first.
  p->tile_keys = head_dim == 256 ? 608 : 256;
  uint8_t* w = static_cast<uint8_t*>(workspace);
  const size_t rows = 2 * static_cast<size_t>(ctx_.sm_count()) * kAttentionRows;
  p->tickets = reinterpret_cast<unsigned int*>(w);
  p->part_stats = reinterpret_cast<float2*>(w + kTicketBytes);
  p->parts = reinterpret_cast<float*>(w + kTicketBytes + rows * sizeof(float2));
  p->status = ctx_.status_word();
  return TK100_OK;
}

Status AttentionOp::launch(cudaStream_t stream, const char* what, int head_dim, const AttentionParams& p,
                           const uint16_t* query, const CUtensorMap& map_k, const CUtensorMap& map_v) {
  CUtensorMap map_q, map_q1;
  const uint64_t dims[4] = {static_cast<uint64_t>(head_dim), static_cast<uint64_t>(p.group),
                            static_cast<uint64_t>(p.kv_heads), static_cast<uint64_t>(p.tokens)};
  const uint64_t strides[3] = {static_cast<uint64_t>(p.query_head_stride),
                               static_cast<uint64_t>(p.query_head_stride) * p.group,
                               static_cast<uint64_t>(p.query_token_stride)};
  const uint32_t group = static_cast<uint32_t>(p.group);
  const uint32_t box[4] = {64u, group, 1u, static_cast<uint32_t>(p.half_tokens)}, box1[4] = {64u, group, 1u, 1u};
  TK100_TRY(ctx_.bf16_map(query, 4, dims, strides, box, &map_q));
  TK100_TRY(ctx_.bf16_map(query, 4, dims, strides, box1, &map_q1));
  DeviceScope device(ctx_);
  TK100_TRY(device.status());
  ctx_.count_launch();
  return ctx_.check(launch_attention(stream, head_dim, ctx_.sm_count() / 2, map_q, map_q1, map_k, map_v, p),
                    (std::string("launching the ") + what).c_str());
}

// Keys in boxes of up to 64 tokens x all chunks of 64 values, one chunk where a page ends inside the 64 (a chunk's
// 64 keys lie next to each other in shared memory); values in boxes of up to 128 tokens x half of a head.
Status AttentionOp::kv_map(const uint16_t* plane, int head_dim, int kv_heads, const CacheGeometry& g, int most_rows,
                           bool keys, CUtensorMap* out) {
  const bool eights = keys && most_rows == g.page_tokens && attention_eights(head_dim, log2_of(g.page_tokens));
  const int rows = eights ? 8 : std::min(most_rows, keys ? 64 : 128);
  const uint64_t dims[5] = {64u, static_cast<uint64_t>(g.page_tokens), static_cast<uint64_t>(head_dim / 64),
                            static_cast<uint64_t>(kv_heads), static_cast<uint64_t>(g.pages)};
  const uint64_t strides[4] = {static_cast<uint64_t>(g.token_stride), 64u, static_cast<uint64_t>(g.head_stride),
                               static_cast<uint64_t>(g.page_stride)};
  const uint32_t box[5] = {64u, static_cast<uint32_t>(rows),
                           static_cast<uint32_t>(!keys ? head_dim / 128 : rows < 64 && !eights ? 1 : head_dim / 64), 1u, 1u};
  return ctx_.bf16_map(plane, 5, dims, strides, box, out);
}

Status AttentionOp::paged(cudaStream_t stream, int head_dim, AttentionParams p, const uint16_t* query,
                          const uint16_t* key_cache, const uint16_t* value_cache, const CacheGeometry& cache, float scale,
                          void* workspace) {
  const char* what = "paged attention";
  TK100_TRY(prepare(what, head_dim, &p, query, key_cache, value_cache, scale, workspace));
  TK100_TRY(cache_geometry(ctx_, what, cache, head_dim));
  TK100_TRY(plane(ctx_, what, "key length", p.kv_lengths, 4));
  TK100_TRY(plane(ctx_, what, "block table", p.block_table, 4));
  TK100_TRY(range(ctx_, what, "block table row count", p.table_row_count, 1, 1 << 30));
  TK100_TRY(range(ctx_, what, "pages per row", p.max_pages, 1, 1 << 30));
  const Span out(p.output, p.tokens, static_cast<long long>(p.q_heads) * head_dim, p.q_heads, head_dim, head_dim);
  if (out.meets(Span(key_cache, cache, p.kv_heads, head_dim)) || out.meets(Span(value_cache, cache, p.kv_heads, head_dim)))
    return refuse(ctx_, what, "the output overlaps the key or value cache");
  if (!p.table_rows && p.sequences > p.table_row_count)
    return refuse(ctx_, what, "the block table has fewer rows than there are sequences");
  p.page_shift = log2_of(cache.page_tokens);
  p.pages = cache.pages;
  p.key_capacity = static_cast<int>(std::min(kMaxKeys, static_cast<long long>(p.max_pages) << p.page_shift));
  CUtensorMap map_k, map_v;
  TK100_TRY(kv_map(key_cache, head_dim, p.kv_heads, cache, cache.page_tokens, true, &map_k));
  TK100_TRY(kv_map(value_cache, head_dim, p.kv_heads, cache, cache.page_tokens, false, &map_v));
  return launch(stream, what, head_dim, p, query, map_k, map_v);
}

Status AttentionOp::prompt(cudaStream_t stream, int head_dim, AttentionParams p, const uint16_t* query, const uint16_t* key,
                           const uint16_t* value, int kv_token_stride, int kv_head_stride, float scale, void* workspace) {
  const char* what = "prompt attention";
  TK100_TRY(prepare(what, head_dim, &p, query, key, value, scale, workspace));
  TK100_TRY(stride(ctx_, what, "key/value token", kv_token_stride, head_dim));
  TK100_TRY(stride(ctx_, what, "key/value head", kv_head_stride, head_dim));
  const Span out(p.output, p.tokens, static_cast<long long>(p.q_heads) * head_dim, p.q_heads, head_dim, head_dim);
  if (out.meets(Span(key, p.tokens, kv_token_stride, p.kv_heads, kv_head_stride, head_dim)) ||
      out.meets(Span(value, p.tokens, kv_token_stride, p.kv_heads, kv_head_stride, head_dim)))
    return refuse(ctx_, what, "the output overlaps the keys or values");
  p.kv_lengths = nullptr;
  p.block_table = nullptr;
  const CacheGeometry rows = {1, p.tokens, kv_token_stride, kv_token_stride, kv_head_stride};
  CUtensorMap map_k, map_v;
  TK100_TRY(kv_map(key, head_dim, p.kv_heads, rows, 128, true, &map_k));
  TK100_TRY(kv_map(value, head_dim, p.kv_heads, rows, 128, false, &map_v));
  return launch(stream, what, head_dim, p, query, map_k, map_v);
}

}  // namespace tk100
