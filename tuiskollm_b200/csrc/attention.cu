// Causal attention with grouped heads over a paged key/value cache or over packed prompt rows.
//
// Sequence s has q new tokens and k keys (k = q for a prompt); its token i sees keys 0 .. k - q + i:
//     o_i = sum_j softmax_j(scale * q_i . k_j) v_j,   optionally times sigmoid(gate_i);
// a token that sees nothing (k - q + i < 0) gets zeros.
//
// Tiles.  Two CTAs of a cluster are one MMA unit of 256 rows (cta_group::2).  The G query heads that share a key/value
// head are rows of one tile: a CTA has floor(128 / G) whole tokens, row r = token r / G, head r % G, so a decoded
// token's heads read the cache once, and the keys that a prompt's diagonal tile computes in vain are 256 / G, not 256.
// A tile walks over its keys 128 at a time:
//     S = Q K^T (tcgen05, both from shared memory) -> TMEM, two buffers
//     P = exp2(scale log2e (S - m)) -> BF16 into the first half of S's columns
//     O += P V (tcgen05, P from TMEM, V from shared memory) -> TMEM
// m is the row's reference maximum: it follows the running maximum only when that has grown by more than 2^8,
// so O is rescaled in TMEM a few times per row, not per tile, and P stays below 2^8, where BF16 and the
// fp32 sum of P lose nothing.  P is rounded to BF16 (2^-8 of each, the tensor core's operand type); sums,
// maxima, O and the join of split rows are fp32.
// Each CTA brings half of the keys of K and half of the values of V, so a step costs its shared memory 64 KB written
// and 128 KB read by the MMAs at heads of 256; one CTA by itself moves 320 KB a step and took 3800 cycles where the
// MMAs take 2048 (prompt of 8192 tokens 1649 -> 1232 us with the pair).
//
// Roles, sixteen warps: TMA producer (each lane asks for a box: one elected lane needed 500 cycles a unit); MMA issuer
// in the even CTA, one step of scores ahead of the values so that the tensor pipe works during the softmax;
// two softmax warpgroups (thread = row) that take the steps in turn and hand on the rows' references, so that one
// step's exponentials run beside the other's loads and maxima; four epilogue warps, which normalise, gate and store
// while the others are on the next tile.  K and V share a ring of three (heads of 128: seven) units; a unit is
// read where the block table says, page by page.
//
// Work split.  All tiles of a launch in order (sequence, key/value head, tile) form one line of keys, and each pair
// takes an equal stretch of it, wherever tiles begin and end, but for cuts near a tile's end, which move there.  A
// tile that several pairs have is joined: each leaves its fp32 O, m and sum in the workspace, takes the tile's
// ticket, and the CTA that draws the last one adds the parts in order of their keys (the same bits whoever is last)
// and stores.  Pairs begin with such tiles, so that joins run beside whole ones.  The lengths stay on the device:
// every CTA sums the costs up for itself, in closed form, so a captured launch follows them.
//
// Measured (B200 at 1.65 to 1.9 GHz), us: prompt of 8192 tokens, 24 heads over 4 of 256, gated, 645 to 711 by the clock
// (1.16 to 1.28 PFLOP/s, 0.69 to 0.77 of cuBLAS' BF16 burst rate); seven packed prompts of up to 1777, 32 over 8 of
// 128, 110 to 117; decode batch of 32 over up to 16384 keys 190 to 214 (849 MB: 0.6 to 0.68 of the copy rate); 512
// tokens over 16000 keys 214 to 221; one token over 4096 keys 21.  A step takes 2400 cycles at heads of 256, where the
// MMAs take 2048, and 1600 at 128 (1024, of which the exponentials take 1024 too): the chain scores -> softmax -> values of
// a step, with one buffer of S per warpgroup, bounds both.
#include <cuda_fp16.h>

#include <new>

#include "common.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace tk100 {
namespace {

constexpr int kRows = 128;   // rows of a tile in each CTA of the pair
constexpr int kKeys = 128;   // keys of a step
constexpr int kThreads = 512;

template <int D>
struct Shape {
  static constexpr int CHUNKS = D / 64;      // 128-byte columns of a row
  static constexpr int K_KEYS = kKeys / 2;   // a K unit: half of the keys, all chunks
  static constexpr int V_CHUNKS = CHUNKS / 2;  // a V unit: all keys, half of the chunks
  static constexpr int UNIT = K_KEYS * 2 * D;  // bytes of a ring stage
  static constexpr int STAGES = D == 256 ? 3 : 7;
};

// ----------------------------------------------------------------- the line of keys

struct Sequence {
  int start, q, kv;  // first token row, new tokens, keys
};

__device__ __forceinline__ Sequence read_sequence(const AttentionParams& p, int s) {
  Sequence r;
  r.start = min(max(p.starts[s], 0), p.tokens);
  r.q = min(max(p.starts[s + 1], r.start), p.tokens) - r.start;
  r.kv = r.q;
  if (p.kv_lengths) r.kv = min(max(p.kv_lengths[s], 0), p.key_capacity);
  return r;
}

// Steps of tile i: at least one, so that a tile which sees nothing still stores its zeros.
__device__ __forceinline__ int tile_limit(const AttentionParams& p, const Sequence& s, int i) {
  return max(s.kv - s.q + min((i + 1) * p.tile_tokens, s.q), 0);  // keys its last token sees
}
__device__ __forceinline__ int tile_steps(const AttentionParams& p, const Sequence& s, int i) {
  return max((tile_limit(p, s, i) + kKeys - 1) / kKeys, 1);
}
__device__ __forceinline__ int tile_count(const AttentionParams& p, const Sequence& s) {
  return (s.q + p.tile_tokens - 1) / p.tile_tokens;
}

__device__ __forceinline__ int tile_cost(const AttentionParams& p, const Sequence& s, int i) {
  return p.tile_keys + tile_limit(p, s, i);
}
// Cost of the first i tiles of one key/value head, an arithmetic series but for tiles that see nothing and the last.
__device__ __forceinline__ long long cost_before(const AttentionParams& p, const Sequence& s, int i, int tiles) {
  long long sum = static_cast<long long>(i) * p.tile_keys;
  int full = i;  // tiles whose last token is their own
  if (i == tiles && i > 0) {
    sum += max(s.kv, 0);
    --full;
  }
  const int ahead = s.kv - s.q;  // keys in front of the first new token
  const int blind = ahead < 0 ? min(-ahead / p.tile_tokens, full) : 0;
  return sum + static_cast<long long>(full - blind) * ahead +
         static_cast<long long>(p.tile_tokens) * (static_cast<long long>(full) * (full + 1) - static_cast<long long>(blind) * (blind + 1)) / 2;
}

__device__ __forceinline__ long long divide(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// Step `step` of a tile that begins at `line`.
struct Place {
  int sequence, head, tile, step;
  long long line;
};

// This pair's stretch of the line, from one place up to another; `share` keys belong to each pair before cuts move.
struct Stretch {
  long long share;
  Place from, to;
};

// A cut closer than this to an end of the tile it falls into moves there: joining the parts of a tile of 128 rows
// costs as much as some four steps (their fp32 rows through L2 and back), of a decoded token's as one.
__device__ __forceinline__ int cut_margin(const AttentionParams& p, int tokens) {
  return 1 + min(tokens, p.half_tokens) * p.group / 32;
}

// One tile, or the part of it that this pair works on.
struct Item {
  Sequence seq;
  int sequence, head, tile;
  int first, last, steps;  // its steps [first, last) of `steps`
  int limit;               // keys its last token sees
  int tokens;              // tokens of the tile
  long long line;          // where it begins
};

__device__ __forceinline__ void describe(const AttentionParams& p, const Sequence& seq, int sequence, int head, int tile,
                                         long long line, Item* it) {
  it->seq = seq;
  it->sequence = sequence;
  it->head = head;
  it->tile = tile;
  it->line = line;
  it->limit = tile_limit(p, seq, tile);
  it->steps = max((it->limit + kKeys - 1) / kKeys, 1);
  it->tokens = min(p.tile_tokens, seq.q - tile * p.tile_tokens);
}

// The pair's items.  A tile that it begins and another pair goes on with comes first: with the tile that it goes on
// with itself, parts are there early and are joined while the whole tiles run.
struct Walk {
  const Stretch& ends;  // in shared memory: every role walks, and few of its registers are free
  int sequence, head, tile, step, tiles;
  long long line;
  Sequence seq;
  bool tail;

  __device__ __forceinline__ Walk(const AttentionParams& p, const Stretch& s)
      : ends(s), sequence(s.from.sequence), head(s.from.head), tile(s.from.tile), step(s.from.step), tiles(0),
        line(s.from.line), tail(s.to.step > 0) {
    seq = {0, 0, 0};
    if (line < s.to.line) {
      seq = read_sequence(p, sequence);
      tiles = tile_count(p, seq);
    }
  }
  __device__ __forceinline__ bool next(const AttentionParams& p, Item* it) {
    if (tail) {
      tail = false;
      const Place to = ends.to;
      describe(p, read_sequence(p, to.sequence), to.sequence, to.head, to.tile, to.line, it);
      it->first = to.line == line ? step : 0;  // both ends in one tile: its only item
      it->last = to.step;
      return true;
    }
    if (line >= ends.to.line) return false;
    while (tile >= tiles) {  // the next head, or the next sequence that has tokens
      tile = 0;
      if (tiles == 0 || ++head == p.kv_heads) {
        head = 0;
        if (++sequence >= p.sequences) return false;
        seq = read_sequence(p, sequence);
        tiles = tile_count(p, seq);
      }
    }
    describe(p, seq, sequence, head, tile, line, it);
    it->first = step;
    it->last = it->steps;
    line += p.tile_keys + it->limit;
    step = 0;
    ++tile;
    return true;
  }
};

// A warp's walk in shared memory, one lane's work: the softmax and epilogue warps have no registers to spare for it.
struct Stroll {
  alignas(16) unsigned char walk[sizeof(Walk)];
  Item it;
  int more;

  __device__ __forceinline__ void begin(const AttentionParams& p, const Stretch& s, int lane) {
    if (lane == 0) new (walk) Walk(p, s);
    __syncwarp();
  }
  __device__ __forceinline__ bool next(const AttentionParams& p, int lane) {
    __syncwarp();
    if (lane == 0) more = reinterpret_cast<Walk*>(walk)->next(p, &it);
    __syncwarp();
    return more != 0;
  }
};

// The items' steps one behind the other.
struct Steps {
  Walk walk;
  Item it;
  int j, item;

  __device__ __forceinline__ Steps(const AttentionParams& p, const Stretch& s) : walk(p, s), j(0), item(-1) {
    it.first = it.last = 0;
  }
  __device__ __forceinline__ bool next(const AttentionParams& p) {
    if (++j < it.last) return true;
    if (!walk.next(p, &it)) return false;
    j = it.first;
    ++item;
    return true;
  }
  __device__ __forceinline__ bool opens() const { return j == it.first; }
  __device__ __forceinline__ bool closes() const { return j + 1 == it.last; }
};

struct Scratch {
  long long warp_sums[kThreads / 32];
  int sequence[2];
  long long rest[2];
};

// Where cut u of the line falls, `rest` behind the first tile of sequence `sequence`, and where it moves to: by a warp,
// which bisects the sequence's tiles 32 at a time.
__device__ __forceinline__ Place locate(const AttentionParams& p, const Sequence& q, int sequence, long long rest, long long u,
                                        int lane) {
  Place at;
  at.sequence = sequence;
  const int tiles = tile_count(p, q);
  const long long per_head = cost_before(p, q, tiles, tiles);
  at.head = static_cast<int>(divide(rest, per_head));
  rest -= at.head * per_head;
  int low = 0, high = tiles;  // cost_before(low) <= rest < cost_before(high)
  while (high - low > 1) {
    const int width = (high - low + 31) / 32, probe = low + (lane + 1) * width;
    const bool behind = probe < high && cost_before(p, q, probe, tiles) <= rest;
    low += __popc(__ballot_sync(0xffffffffu, behind)) * width;
    high = min(high, low + width);
  }
  at.tile = low;
  rest -= cost_before(p, q, low, tiles);
  at.line = u - rest;
  at.step = static_cast<int>(static_cast<unsigned long long>(rest) / kKeys);
  const int steps = tile_steps(p, q, low);
  const int margin = cut_margin(p, min(p.tile_tokens, q.q - low * p.tile_tokens));
  if (at.step < margin) {
    at.step = 0;
  } else if (steps - at.step < margin) {
    at.step = 0;
    at.line += tile_cost(p, q, low);
    ++at.tile;
  }
  return at;
}

// The pair's even cuts; returns the keys of a pair.
__device__ __forceinline__ long long even_cuts(const AttentionParams& p, long long total, long long (&cuts)[2]) {
  const long long share = max(divide(total + gridDim.x / 2 - 1, gridDim.x / 2), static_cast<long long>(kKeys));
  cuts[0] = min(static_cast<long long>(blockIdx.x / 2) * share, total);
  cuts[1] = min(cuts[0] + share, total);
  return share;
}
__device__ __forceinline__ long long sequence_cost(const AttentionParams& p, const Sequence& q) {
  const int tiles = tile_count(p, q);
  return cost_before(p, q, tiles, tiles) * p.kv_heads;
}
// Lengths outside the planes are cut to them, and reported.
__device__ __forceinline__ void report_cut(const AttentionParams& p, const Sequence& q, int s) {
  if (blockIdx.x == 0 && (q.start != p.starts[s] || q.start + q.q != p.starts[s + 1] || (p.kv_lengths && q.kv != p.kv_lengths[s])))
    atomicOr(p.status, STATUS_BAD_ARGUMENT);
}
__device__ __forceinline__ long long warp_scan(long long sum, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += x;
  }
  return sum;
}

// Finds the pair's stretch; warp 0 has its beginning, warp 1 its end.  Up to 32 sequences a lane each, so that a warp
// needs no other; beyond, all threads sum up the sequences' costs and the thread that passes a cut names the sequence.
__device__ __forceinline__ void find_stretch(const AttentionParams& p, Scratch& sh, Stretch& found) {
  const int t = static_cast<int>(threadIdx.x), lane = t & 31, warp = t >> 5;
  long long cuts[2];
  if (p.sequences <= 32) {
    if (warp < 2) {
      Sequence q = {0, 0, 0};
      long long mine = 0;
      if (lane < p.sequences) {
        q = read_sequence(p, lane);
        mine = sequence_cost(p, q);
        if (warp == 0) report_cut(p, q, lane);
      }
      const long long sum = warp_scan(mine, lane), total = __shfl_sync(0xffffffffu, sum, 31);
      const long long share = even_cuts(p, total, cuts), u = warp == 0 ? cuts[0] : cuts[1];
      Place at = {};
      at.line = u;
      if (cuts[0] < cuts[1] && u < total) {
        const int s = __ffs(__ballot_sync(0xffffffffu, u < sum)) - 1;
        const long long rest = u - __shfl_sync(0xffffffffu, sum - mine, s);
        const Sequence its = {__shfl_sync(0xffffffffu, q.start, s), __shfl_sync(0xffffffffu, q.q, s),
                              __shfl_sync(0xffffffffu, q.kv, s)};
        at = locate(p, its, s, rest, u, lane);
      }
      if (lane == 0) (warp == 0 ? found.from : found.to) = at;
      if (t == 0) found.share = share;
    }
    __syncthreads();
    return;
  }
  const int run = (p.sequences + kThreads - 1) / kThreads;
  const int s0 = min(t * run, p.sequences), s1 = min(s0 + run, p.sequences);
  long long mine = 0;
  for (int s = s0; s < s1; ++s) {
    const Sequence q = read_sequence(p, s);
    mine += sequence_cost(p, q);
    report_cut(p, q, s);
  }
  const long long sum = warp_scan(mine, lane);
  if (lane == 31) sh.warp_sums[warp] = sum;
  __syncthreads();
  long long before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += sh.warp_sums[w];
    total += sh.warp_sums[w];
  }
  before += sum - mine;
  const long long share = even_cuts(p, total, cuts);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (cuts[0] < cuts[1] && before <= cuts[k] && cuts[k] < before + mine) {
      long long rest = cuts[k] - before;
      int s = s0;
      for (;; ++s) {
        const long long cost = sequence_cost(p, read_sequence(p, s));
        if (rest < cost) break;
        rest -= cost;
      }
      sh.sequence[k] = s;
      sh.rest[k] = rest;
    }
  }
  __syncthreads();
  if (warp < 2) {
    const long long u = warp == 0 ? cuts[0] : cuts[1];
    Place at = {};
    at.line = u;
    if (cuts[0] < cuts[1] && u < total)
      at = locate(p, read_sequence(p, sh.sequence[warp]), sh.sequence[warp], sh.rest[warp], u, lane);
    if (lane == 0) (warp == 0 ? found.from : found.to) = at;
    if (t == 0) found.share = share;
  }
  __syncthreads();
}

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Half a row of S; keys it does not see read as -infinity.
__device__ __forceinline__ void load_scores(uint32_t taddr, bool masked, int seen, uint32_t (&s)[kKeys / 2]) {
  tmem_ld32(taddr, s);
  tmem_ld32(taddr + 32, s + 32);
  tmem_ld_wait();
  if (masked) {
#pragma unroll
    for (int k = 0; k < kKeys / 2; ++k) s[k] = k < seen ? s[k] : 0xff800000u;
  }
}
__device__ __forceinline__ float top_of(const uint32_t (&s)[kKeys / 2]) {
  float tops[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) tops[k] = fmaxf(__uint_as_float(s[k]), __uint_as_float(s[k + 4]));
#pragma unroll
  for (int k = 8; k < kKeys / 2; k += 8) {
#pragma unroll
    for (int e = 0; e < 4; ++e) tops[e] = fmaxf(tops[e], fmaxf(__uint_as_float(s[k + e]), __uint_as_float(s[k + e + 4])));
  }
  return fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
}
// The scores' weights, packed into the first half of the array; returns their sum.
__device__ __forceinline__ float weights_of(uint32_t (&s)[kKeys / 2], float c, float shift) {
  const F32x2 scale2 = f32x2_splat(c), shift2 = f32x2_splat(-shift);
  F32x2 sums[2] = {f32x2_splat(0.0f), f32x2_splat(0.0f)};
#pragma unroll
  for (int k = 0; k < kKeys / 2; k += 2) {
    const float2 e = f32x2_parts(fma2(f32x2(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), scale2, shift2));
    const float a = exp2_approx(e.x), b = exp2_approx(e.y);
    sums[(k >> 1) & 1] = add2(sums[(k >> 1) & 1], f32x2(a, b));
    s[k / 2] = pack_bf16x2(a, b);
  }
  const float2 sum = f32x2_parts(add2(sums[0], sums[1]));
  return sum.x + sum.y;
}

// A bounded wait of a whole warp, with one verdict: mbar_wait written out, because a call, even one that is never
// made, would hold all warps to one register count.  CLUSTER: threads of the other CTA arrive on the barrier.
template <bool CLUSTER>
__device__ __forceinline__ bool bounded_wait(uint64_t* bar, uint32_t parity, uint32_t* status) {
  bool done = false;
  uint64_t start = 0;  // (reading the clock takes some 2000 cycles: not before the barrier has been looked at for a while)
#pragma unroll 1
  for (uint32_t i = 1; !done; ++i) {
    done = CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity);
    if (!done && (i & 1023u) == 0) {
      if (*reinterpret_cast<volatile uint32_t*>(status) & STATUS_WAIT_TIMEOUT) break;
      const uint64_t now = global_timer_ns();
      if (start == 0) start = now;
      if (now - start > 2000000000ull) {
        atomicOr(status, STATUS_WAIT_TIMEOUT);
        break;
      }
    }
  }
  return __all_sync(0xffffffffu, done);
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, uint32_t* status) {
  return bounded_wait<false>(bar, parity, status);
}
__device__ __forceinline__ bool warp_wait_cluster(uint64_t* bar, uint32_t parity, uint32_t* status) {
  return bounded_wait<true>(bar, parity, status);
}

// Keys of a step that count, of which the last 16 that are multiplied are not full: those behind them are zeroed.
__device__ __forceinline__ bool ragged(int keys) { return keys < kKeys && (keys <= 0 || keys % 16 != 0); }
template <int D>
__device__ __forceinline__ void zero_behind(uint8_t* unit, int keys, int v_box, int lane) {
  constexpr int PIECES = Shape<D>::V_CHUNKS * 8;  // of 16 bytes in a row
  const int first = max(keys, 0), rows = keys <= 0 ? 16 : 16 - keys % 16;
  for (int i = lane; i < rows * PIECES; i += 32) {
    const int r = first + i / PIECES, c = (i / 8) % Shape<D>::V_CHUNKS, piece = i % 8;
    *reinterpret_cast<uint4*>(unit + (r / v_box * Shape<D>::V_CHUNKS + c) * v_box * 128 + r % v_box * 128 + piece * 16) =
        make_uint4(0u, 0u, 0u, 0u);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

// 32 bytes of an output row: each thread has a row of its own, so a narrower store would touch every sector twice.
__device__ __forceinline__ void store_words8(uint16_t* to, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// Rows of a tile whose first token row is `token`.
__device__ __forceinline__ const uint16_t* gate_row(const AttentionParams& p, int token, int head, int row) {
  return p.gate + static_cast<size_t>(token + row / p.group) * p.gate_token_stride +
         static_cast<size_t>(head * p.group + row % p.group) * p.gate_head_stride;
}
template <int D>
__device__ __forceinline__ uint16_t* output_row(const AttentionParams& p, int token, int head, int row) {
  return p.output + (static_cast<size_t>(token + row / p.group) * p.q_heads + head * p.group + row % p.group) * D;
}
__device__ __forceinline__ uint32_t f32x2_to_f16x2(F32x2 v) {
  const float2 f = f32x2_parts(v);
  uint32_t w;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(f.y), "f"(f.x));
  return w;
}
__device__ __forceinline__ F32x2 f16x2_to_f32x2(uint32_t w) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return f32x2(f.x, f.y);
}
// Two values times the sigmoid of their packed gates.
__device__ __forceinline__ F32x2 gated(F32x2 v, uint32_t gate) {
  const float2 e = f32x2_parts(mul2(bf16x2_to_f32x2(gate), f32x2_splat(-1.4426950408889634f)));
  const float2 d = f32x2_parts(add2(f32x2(exp2_approx(e.x), exp2_approx(e.y)), f32x2_splat(1.0f)));
  float a, b;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(d.y));
  return mul2(v, f32x2(a, b));
}

// Parts of a tile's rows that this CTA and its likes in pairs c0 .. c1 left are joined in the order of their keys.
// A part is [four values][128 rows][4], so that threads next to each other have rows next to each other.
__device__ __forceinline__ size_t part_slot(int k, int c0, int rank) {
  return 2 * static_cast<size_t>(2 * k + rank) + (k == c0 ? 1 : 0);
}
__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Loads past L1 that stay where they are written: left to itself the compiler moves each of them into the branch
// that uses it, and a join of 18 parts waits for L2 60 times instead of 4.
__device__ __forceinline__ float4 load_part(const float4* p) {
  float4 v;
  asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ float2 load_part(const float2* p) {
  float2 v;
  asm volatile("ld.global.cg.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p));
  return v;
}

// The rows' common maximum, and 1 / the sum of their weights, with LANES lanes of the 128 threads to a row.
template <int LANES>
__device__ __forceinline__ void join_stats(const AttentionParams& p, int c0, int c1, int rank, int rows, int thread,
                                           float* row_top, float* row_scale) {
  const int lane = thread % LANES;
#pragma unroll 1
  for (int base = 0; base < rows; base += 128 / LANES) {
    const int row = base + thread / LANES, from = min(row, rows - 1);
    float top = -INFINITY, total = 0.0f;
#pragma unroll 1
    for (int k = c0 + lane; k <= c1; k += 4 * LANES) {
      float2 stats[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) stats[e] = load_part(p.part_stats + part_slot(min(k + e * LANES, c1), c0, rank) * kRows + from);
      float most = top;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (k + e * LANES > c1) stats[e] = make_float2(-INFINITY, 0.0f);
        most = fmaxf(most, stats[e].x);
      }
      const float shift = most == -INFINITY ? 0.0f : most;
      total *= exp2_approx(top - shift);
      top = most;
#pragma unroll
      for (int e = 0; e < 4; ++e) total = fmaf(stats[e].y, exp2_approx(stats[e].x - shift), total);
    }
    if (LANES > 1) {
      float most = top;
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      total *= exp2_approx(top - (most == -INFINITY ? 0.0f : most));
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
      top = most;
    }
    if (lane == 0 && row < rows) {
      row_top[row] = top == -INFINITY ? 0.0f : top;
      row_scale[row] = 1.0f / total;
    }
  }
  named_barrier(1, 128);
}

// The rows: a thread has four of a row's values at three places, and their loads of five parts under way together (four
// places and two parts are slower even where there are no more parts: six decoded tokens 41.6 us, not 41.1, twelve 65.3
// and 63.9).
template <int D>
__device__ __forceinline__ void join_rows(const AttentionParams& p, int c0, int c1, int rank, int rows, int thread, int ahead,
                                          int token, int head, const float* row_top, const float* row_scale) {
  constexpr int PLACES = 3, PARTS = 5;
  const int places = rows * (D / 4);
#pragma unroll 1
  for (int base = thread; base < places; base += 128 * PLACES) {
    float4 acc[PLACES];
    int row[PLACES], at[PLACES];
#pragma unroll
    for (int i = 0; i < PLACES; ++i) {
      const int place = min(base + 128 * i, places - 1), quad = place / rows;
      row[i] = place - quad * rows;
      at[i] = quad * kRows + row[i];
      acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    uint2 gate[PLACES];
    if (p.gate) {
#pragma unroll
      for (int i = 0; i < PLACES; ++i)
        gate[i] = __ldg(reinterpret_cast<const uint2*>(gate_row(p, token, head, row[i]) + 4 * (at[i] / kRows)));
    }
#pragma unroll 1
    for (int k = c0; k <= c1; k += PARTS) {
      float2 stats[PLACES][PARTS];
      float4 o[PLACES][PARTS];
#pragma unroll
      for (int e = 0; e < PARTS; ++e) {
        const size_t slot = part_slot(min(k + e, c1), c0, rank);
#pragma unroll
        for (int i = 0; i < PLACES; ++i) {
          stats[i][e] = load_part(p.part_stats + slot * kRows + row[i]);
          o[i][e] = load_part(reinterpret_cast<const float4*>(p.parts) + slot * kRows * (D / 4) + at[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < PLACES; ++i) {
        const float top = row_top[row[i]];
#pragma unroll
        for (int e = 0; e < PARTS; ++e) {
          // a part without a key of this row has nothing to add, whatever its O holds
          if (k + e <= c1 && !(stats[i][e].x == -INFINITY && stats[i][e].y == 0.0f)) {
            const float w = exp2_approx(stats[i][e].x - top);
            acc[i].x = fmaf(o[i][e].x, w, acc[i].x);
            acc[i].y = fmaf(o[i][e].y, w, acc[i].y);
            acc[i].z = fmaf(o[i][e].z, w, acc[i].z);
            acc[i].w = fmaf(o[i][e].w, w, acc[i].w);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < PLACES; ++i) {
      if (base + 128 * i < places) {
        const float scale = row_scale[row[i]];
        F32x2 v[2] = {mul2(f32x2(acc[i].x, acc[i].y), f32x2_splat(scale)), mul2(f32x2(acc[i].z, acc[i].w), f32x2_splat(scale))};
        if (p.gate) {
          v[0] = gated(v[0], gate[i].x);
          v[1] = gated(v[1], gate[i].y);
        }
        uint2 w = make_uint2(f32x2_to_bf16x2(v[0]), f32x2_to_bf16x2(v[1]));
        if (ahead + row[i] / p.group < 0) w = make_uint2(0u, 0u);  // sees no key
        *reinterpret_cast<uint2*>(output_row<D>(p, token, head, row[i]) + 4 * (at[i] / kRows)) = w;
      }
    }
  }
}

// The same where there are many rows: a thread has one, 16 of its values at a time, and the loads of two parts of them
// under way together.
template <int D>
__device__ __forceinline__ void join_tall(const AttentionParams& p, int c0, int c1, int rank, int rows, int thread, int ahead,
                                          int token, int head, const float* row_top, const float* row_scale) {
  constexpr int QUADS = 4;
  const int row = min(thread, rows - 1);
  const float top = row_top[row];
  const F32x2 scale = f32x2_splat(row_scale[row]);
  const bool blind = ahead + row / p.group < 0;  // sees no key
  uint16_t* out = output_row<D>(p, token, head, row);
  const uint4* gate = p.gate ? reinterpret_cast<const uint4*>(gate_row(p, token, head, row)) : nullptr;
#pragma unroll 1
  for (int quad = 0; quad < D / 4; quad += QUADS) {
    float4 acc[QUADS];
    uint4 g[QUADS / 2];
    if (gate) {
#pragma unroll
      for (int i = 0; i < QUADS / 2; ++i) g[i] = __ldg(gate + quad / 2 + i);
    }
#pragma unroll
    for (int i = 0; i < QUADS; ++i) acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
    for (int k = c0; k <= c1; k += 2) {
      float2 stats[2];
      float4 o[2][QUADS];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const size_t slot = part_slot(min(k + e, c1), c0, rank);
        stats[e] = load_part(p.part_stats + slot * kRows + row);
#pragma unroll
        for (int i = 0; i < QUADS; ++i)
          o[e][i] = load_part(reinterpret_cast<const float4*>(p.parts) + slot * kRows * (D / 4) + (quad + i) * kRows + row);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // a part without a key of this row has nothing to add, whatever its O holds
        if (k + e <= c1 && !(stats[e].x == -INFINITY && stats[e].y == 0.0f)) {
          const float w = exp2_approx(stats[e].x - top);
#pragma unroll
          for (int i = 0; i < QUADS; ++i) {
            acc[i].x = fmaf(o[e][i].x, w, acc[i].x);
            acc[i].y = fmaf(o[e][i].y, w, acc[i].y);
            acc[i].z = fmaf(o[e][i].z, w, acc[i].z);
            acc[i].w = fmaf(o[e][i].w, w, acc[i].w);
          }
        }
      }
    }
    uint32_t w[2 * QUADS];
#pragma unroll
    for (int i = 0; i < QUADS; ++i) {
      F32x2 a = mul2(f32x2(acc[i].x, acc[i].y), scale), b = mul2(f32x2(acc[i].z, acc[i].w), scale);
      if (gate) {
        const uint4 v = g[i / 2];
        a = gated(a, i % 2 == 0 ? v.x : v.z);
        b = gated(b, i % 2 == 0 ? v.y : v.w);
      }
      w[2 * i] = blind ? 0u : f32x2_to_bf16x2(a);
      w[2 * i + 1] = blind ? 0u : f32x2_to_bf16x2(b);
    }
    if (thread < rows) store_words8(out + 4 * quad, w);
  }
}

// ------------------------------------------------------------------------- the kernel

// Barriers that both CTAs' loads or threads arrive on are the even CTA's (full, q_full, p_full, o_free); those that
// the even CTA's MMA warp commits to are arrived on in both (empty, q_empty, s_full, pv_done, o_full).
template <int D>
struct Control {
  uint64_t full[Shape<D>::STAGES], empty[Shape<D>::STAGES], tail_full[Shape<D>::STAGES];
  uint64_t q_full, q_empty, s_full[2], p_full[2], pv_done, o_full, o_free, stats_full, stats_free, drained;
  uint64_t reference_set[2][4];
  uint32_t tmem_base;
  int last_part;
  Stretch stretch;
  uint4 rows[D == 256 ? 16 : 1][kRows];  // the second halves of rows of 256 between tensor memory and their gate
  Stroll strolls[12];      // of the softmax and epilogue warps
  float reference[kRows];  // the row's reference maximum, of the step before
  float row_sum[2][kRows];  // what either softmax warpgroup has of a row at a tile's end
  union {
    float row_max[2][kRows];
    Scratch scratch;  // in front of the roles
  };
};
template <int D>
constexpr int shared_bytes() {
  return kRows * 2 * D + Shape<D>::STAGES * Shape<D>::UNIT + static_cast<int>(sizeof(Control<D>));
}

static_assert(shared_bytes<256>() <= 232448 && shared_bytes<128>() <= 232448, "more shared memory than a CTA may have");

// Registers of the calling warpgroup from here on; the four shares make up the 4 x 128 that the block starts with.
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
// (Nothing spills at these; 8 fewer for the epilogue, or for the softmax, do.)
constexpr int kControlRegisters = 80, kSoftmaxRegisters = 120, kEpilogueRegisters = 192;
static_assert(kControlRegisters + 2 * kSoftmaxRegisters + kEpilogueRegisters <= 4 * 128, "the shares exceed the block's registers");

template <int D, bool PAGED>
__global__ void __launch_bounds__(kThreads, 1)
    attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_q1,
                     const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                     const __grid_constant__ AttentionParams p) {
  using S = Shape<D>;
  constexpr int STAGES = S::STAGES;
  extern __shared__ __align__(1024) uint8_t dynamic[];
  uint8_t* const smem_q = dynamic;
  uint8_t* const ring = smem_q + kRows * 2 * D;
  Control<D>& ctl = *reinterpret_cast<Control<D>*>(ring + STAGES * S::UNIT);

  const int warp = warp_index(), lane = static_cast<int>(threadIdx.x) & 31;
  const int rank = static_cast<int>(cluster_cta_rank());

  if (warp == 0 && elect_one()) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&ctl.full[i], 2);
      mbar_init(&ctl.empty[i], 1);
      mbar_init(&ctl.tail_full[i], 1);
    }
    mbar_init(&ctl.q_full, 1);
    mbar_init(&ctl.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl.s_full[i], 1);
      mbar_init(&ctl.p_full[i], 8);
    }
    mbar_init(&ctl.pv_done, 1);
    mbar_init(&ctl.o_full, 1);
    mbar_init(&ctl.o_free, 8);
    mbar_init(&ctl.stats_full, 8);
    mbar_init(&ctl.stats_free, 4);
    mbar_init(&ctl.drained, 1);
    for (int i = 0; i < 8; ++i) mbar_init(&ctl.reference_set[i / 4][i % 4], 1);
    fence_mbar_init();
    prefetch_tensormap(&map_q);
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  if (warp == 1) {
    tmem_alloc_pair(&ctl.tmem_base, 512);
    tmem_relinquish_pair();
  }
  pdl_wait();
  pdl_trigger();
  tc_fence_before_sync();
  __syncthreads();
  cluster_arrive();  // both CTAs' barriers exist before either touches the other's
  find_stretch(p, ctl.scratch, ctl.stretch);
  cluster_wait();
  tc_fence_after_sync();
  const uint32_t tmem = ctl.tmem_base;
  const Stretch& stretch = ctl.stretch;
  const uint32_t tmem_o = tmem + 2 * kKeys;
  const int v_box = PAGED ? min(kKeys, 1 << p.page_shift) : kKeys;  // keys of a box of V
  // A box of K that has all chunks of fewer than 64 keys leaves those keys' chunks behind one another: right for an
  // MMA when it has 8 keys, a swizzle's rows, whose distance the descriptor names.  Pages of 16 keys then take 8
  // boxes a unit, not one per page and chunk, 16, at which the loads of a step take twice its products (512 tokens over
  // 16000 keys).
  const bool eights = PAGED && attention_eights(D, p.page_shift);

  if (warp < 4) {
    fewer_registers<kControlRegisters>();
    if (warp == 0) {
      // ---------------------------------------------------------------- producer
      int stage = 0;
      uint32_t phase = 1;  // parity to wait for on `empty`: a fresh barrier's earlier phase
      bool ok = true;
      int items = 0;
      auto advance = [&]() {
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      };
      const uint32_t full_even = mapa_u32(smem_u32(&ctl.full[0]), 0), q_full_even = mapa_u32(smem_u32(&ctl.q_full), 0);
      const uint32_t tail_mine = mapa_u32(smem_u32(&ctl.tail_full[0]), static_cast<uint32_t>(rank));
      // Boxes of a unit, one per lane: K boxes of `k_box` keys and one chunk (all chunks where no page ends inside the
      // 64 keys), V boxes of `v_box` keys and half of the chunks.  What does not change from step to step:
      const int shift = p.page_shift;
      const int k_box = eights ? 8 : PAGED ? min(S::K_KEYS, 1 << shift) : S::K_KEYS;
      const bool all = eights || k_box == S::K_KEYS;
      const int k_key = (all ? lane : lane / S::CHUNKS) * k_box, k_chunk = all ? 0 : lane % S::CHUNKS, v_key = lane * v_box;
      uint8_t* const k_to = ring + k_chunk * (S::K_KEYS * 128) + k_key * (eights ? 2 * D : 128);
      uint8_t* const v_to = ring + v_key * S::V_CHUNKS * 128;
      const int within_page = PAGED ? (1 << shift) - 1 : -1;
      // page of key `key` of the sequence in table row `row`; outside the planes -1, where TMA fills zeros
      auto page_of = [&](int row, int key, bool needed) -> int {
        if (!PAGED) return 0;
        int id = -1;
        if (needed) {
          const int index = key >> shift;
          if (row >= 0 && index < p.max_pages) id = p.block_table[static_cast<size_t>(row) * p.max_pages + index];
          if (id < 0 || id >= p.pages) {
            id = -1;
            atomicOr(p.status, STATUS_BAD_ARGUMENT);
          }
        }
        return id;
      };
      struct Fetch {  // a step: its first key (as a coordinate for packed rows), how many of its keys count, pages
        int base, keys, head, k_page, v_page;
      };
      auto fetch_of = [&](const Steps& at, int row) -> Fetch {
        Fetch f;
        const int first = at.j * kKeys, k = rank * S::K_KEYS + k_key;
        f.keys = min(at.it.limit - first, kKeys);
        f.head = at.it.head;
        f.base = PAGED ? first : at.it.seq.start + first;
        f.k_page = page_of(row, first + k, k_key < S::K_KEYS && k < f.keys);
        f.v_page = page_of(row, first + v_key, v_key < f.keys);
        return f;
      };
      // keys of CTA r's half of K that boxes fetch
      auto k_fetched = [&](int keys, int r) { return (min(max(keys - r * S::K_KEYS, 0), S::K_KEYS) + k_box - 1) & ~(k_box - 1); };
      Steps now(p, stretch);
      int row = 0;
      Fetch fetch{}, earlier{};
      bool more = now.next(p), loaded = false;
      auto open = [&]() {
        if (PAGED) {
          row = p.table_rows ? p.table_rows[now.it.sequence] : now.it.sequence;
          if (row >= p.table_row_count) row = -1;
        }
      };
      if (more) {
        open();
        fetch = fetch_of(now, row);
      }
      // K of a step, then V of the step before it: the order in which the MMA warp asks for them
      while (ok && (more || loaded)) {
        if (more) {
          if (now.opens()) {
            const Item& it = now.it;
            if (now.item > 0) ok = warp_wait(&ctl.q_empty, (now.item - 1) & 1, p.status);
            if (!ok) break;
            const int mine = min(it.tokens - rank * p.half_tokens, p.half_tokens);  // tokens of this CTA's rows
            if (rank == 0 && lane == 0) {
              const int other = min(max(it.tokens - p.half_tokens, 0), p.half_tokens);
              const int tokens = (mine == 1 ? 1 : p.half_tokens) + (other <= 1 ? other : p.half_tokens);
              mbar_arrive_expect_tx(&ctl.q_full, static_cast<uint32_t>(p.group * tokens * 128 * S::CHUNKS));
            }
            if (lane < S::CHUNKS && mine > 0) {
              tma_load_4d_pair(smem_q + lane * kRows * 128, mine == 1 ? &map_q1 : &map_q, q_full_even, 64 * lane, 0, it.head,
                               it.seq.start + it.tile * p.tile_tokens + rank * p.half_tokens);
            }
            __syncwarp();
            ++items;
          }
          ok = warp_wait(&ctl.empty[stage], phase, p.status);
          if (!ok) break;
          if (lane == 0) {
            if (rank == 0) {
              mbar_arrive_expect_tx(&ctl.full[stage], static_cast<uint32_t>((k_fetched(fetch.keys, 0) + k_fetched(fetch.keys, 1)) * 2 * D));
            } else {
              mbar_arrive_remote_light(full_even + stage * 8);
            }
          }
          if (k_key < k_fetched(fetch.keys, rank))
            tma_load_5d_pair(k_to + stage * S::UNIT, &map_k, full_even + stage * 8, 0,
                             (fetch.base + rank * S::K_KEYS + k_key) & within_page, k_chunk, fetch.head, fetch.k_page);
          __syncwarp();
          advance();
        }
        if (loaded) {
          ok = warp_wait(&ctl.empty[stage], phase, p.status);
          if (!ok) break;
          const int fetched = (max(earlier.keys, 0) + v_box - 1) & ~(v_box - 1);
          const bool tail = ragged(earlier.keys);  // goes to this CTA's own barrier, `full` is arrived on behind the zeros
          if (lane == 0) {
            if (tail) {
              mbar_arrive_expect_tx(&ctl.tail_full[stage], static_cast<uint32_t>(fetched * D));
            } else if (rank == 0) {
              mbar_arrive_expect_tx(&ctl.full[stage], static_cast<uint32_t>(fetched * 2 * D));
            } else {
              mbar_arrive_remote_light(full_even + stage * 8);
            }
          }
          if (v_key < fetched)
            tma_load_5d_pair(v_to + stage * S::UNIT, &map_v, (tail ? tail_mine : full_even) + stage * 8, 0,
                             (earlier.base + v_key) & within_page, rank * S::V_CHUNKS, earlier.head, earlier.v_page);
          __syncwarp();
          advance();
        }
        loaded = more;
        if (more) {
          earlier = fetch;
          more = now.next(p);
          if (more) {
            if (now.opens()) open();
            fetch = fetch_of(now, row);
          }
        }
      }
      if (!ok) {
        // what was asked for lands before a CTA's shared memory is somebody else's; both leave together
        for (int n = 0; rank == 0 && items > 0 && n < 200000 && !mbar_try_wait(&ctl.q_full, (items - 1) & 1); ++n) {
        }
        for (int i = 0; i < STAGES; ++i) {
          for (int n = 0; rank == 0 && n < 200000 && !mbar_try_wait(&ctl.full[stage], phase); ++n) {
          }
          advance();
        }
        for (int i = 0; i < 64; ++i) __nanosleep(1000);  // what counts on other barriers
      }
    } else if (warp == 1 && rank == 0) {
      // ------------------------------------------------------------------- MMA
      constexpr uint32_t idesc_s = umma_idesc_bf16(2 * kRows, kKeys, false);
      constexpr uint32_t idesc_o = umma_idesc_bf16(2 * kRows, D, true);
      int stage = 0, n = 0;  // n: steps so far
      uint32_t phase = 0, tail_phase = 0;
      bool ok = true;
      auto advance = [&]() {
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      };
      const uint32_t q_addr = smem_u32(smem_q), ring_addr = smem_u32(ring);
      Steps next(p, stretch);
      // S[buffer] = Q K^T of step `next`
      auto scores = [&](int buffer) {
        if (next.opens()) ok = warp_wait(&ctl.q_full, next.item & 1, p.status);
        ok = ok && warp_wait_cluster(&ctl.full[stage], phase, p.status);
        if (!ok) return;
        if (elect_one()) {
          const uint64_t a = umma_desc_sw128(q_addr);
          const uint64_t b = umma_desc_sw128(ring_addr + stage * S::UNIT, eights ? 16 * D : 1024);
          const uint32_t chunk = (eights ? 1024 : S::K_KEYS * 128) >> 4;
#pragma unroll
          for (int k = 0; k < 4 * S::CHUNKS; ++k) {
            umma_bf16_pair(tmem + buffer * kKeys, a + (k >> 2) * (kRows * 128 >> 4) + 2 * (k & 3),
                           b + (k >> 2) * chunk + 2 * (k & 3), idesc_s, k > 0);
          }
          umma_commit_pair(&ctl.empty[stage]);
          umma_commit_pair(&ctl.s_full[buffer]);
          if (next.closes()) umma_commit_pair(&ctl.q_empty);
        }
        __syncwarp();
        advance();
      };
      bool more = next.next(p);
      if (more) scores(0);
      while (ok && more) {
        const int buffer = n & 1, keys = next.it.limit - next.j * kKeys, item = next.item;
        const bool opens = next.opens(), closes = next.closes();
        more = next.next(p);
        if (more) scores(buffer ^ 1);
        if (!ok) break;
        if (ragged(keys)) {
          // P is zero for the keys behind the last, but what lies there may be no number
          ok = warp_wait(&ctl.tail_full[stage], (tail_phase >> stage) & 1, p.status);
          if (!ok) break;
          tail_phase ^= 1u << stage;
          zero_behind<D>(ring + stage * S::UNIT, keys, v_box, lane);
          if (lane == 0) mbar_arrive(&ctl.full[stage]);
        }
        if (opens && item > 0) ok = warp_wait_cluster(&ctl.o_free, (item - 1) & 1, p.status);
        ok = ok && warp_wait_cluster(&ctl.full[stage], phase, p.status) && warp_wait_cluster(&ctl.p_full[buffer], (n >> 1) & 1, p.status);
        if (!ok) break;
        tc_fence_after_sync();
        if (elect_one()) {
          const uint64_t b = umma_desc_sw128_mn(ring_addr + stage * S::UNIT, v_box * 128);
          const int slices = keys <= 0 ? 1 : min((keys + 15) / 16, kKeys / 16);
          for (int k = 0; k < slices; ++k) {
            const uint32_t r = 16 * k;  // box r / v_box of [chunk][v_box keys][128 bytes]
            const uint32_t offset = (r & ~(v_box - 1u)) * S::V_CHUNKS * 128 + (r & (v_box - 1u)) * 128;
            umma_bf16_ta_pair(tmem_o, tmem + buffer * kKeys + 8 * k, b + (offset >> 4), idesc_o, !opens || k > 0);
          }
          umma_commit_pair(&ctl.empty[stage]);
          umma_commit_pair(&ctl.pv_done);
          if (closes) umma_commit_pair(&ctl.o_full);
        }
        __syncwarp();
        advance();
        ++n;
      }
      if (!ok) {
        if (elect_one()) umma_commit_pair(&ctl.drained);
        __syncwarp();
        for (int i = 0; i < 200000 && !mbar_try_wait(&ctl.drained, 0); ++i) {
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------- zeros behind the odd CTA's last keys
      const uint32_t full_even = mapa_u32(smem_u32(&ctl.full[0]), 0);
      uint32_t tail_phase = 0;
      int stage = 0;
      auto advance = [&]() { stage = stage + 1 == STAGES ? 0 : stage + 1; };
      Steps next(p, stretch);
      bool more = next.next(p);
      if (more) advance();
      while (more) {
        const int keys = next.it.limit - next.j * kKeys;
        more = next.next(p);
        if (more) advance();
        if (ragged(keys)) {
          if (!warp_wait(&ctl.tail_full[stage], (tail_phase >> stage) & 1, p.status)) break;
          tail_phase ^= 1u << stage;
          zero_behind<D>(ring + stage * S::UNIT, keys, v_box, lane);
          if (lane == 0) mbar_arrive_remote(full_even + stage * 8);
        }
        advance();
      }
    }
  } else if (warp < 12) {
    // ----------------------------------------------------------------- softmax
    fewer_registers<kSoftmaxRegisters>();
    const int group = (warp >> 2) - 1;  // has the steps of its parity, and S buffer `group`
    const int quadrant = warp & 3;      // the TMEM lanes this warp may touch
    const int r = quadrant * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quadrant * 32) << 16;
    const uint32_t at = tmem + group * kKeys + lanes;
    const float c = p.scale_log2;
    const uint32_t p_full_even = mapa_u32(smem_u32(&ctl.p_full[group]), 0);
    int n = 0, item = 0;
    bool ok = true;
    Stroll& stroll = ctl.strolls[warp - 4];
    stroll.begin(p, stretch, lane);
    const Item& it = stroll.it;
    while (ok && stroll.next(p, lane)) {
      const int rows = min(it.tokens - rank * p.half_tokens, p.half_tokens) * p.group;
      const bool active = quadrant * 32 < rows;
      const int ahead = it.seq.kv - it.seq.q + it.tile * p.tile_tokens + rank * p.half_tokens;
      const int limit = ahead + r / p.group + 1;  // keys this row sees
      const int first = it.first, last = it.last;
      float mine = -INFINITY, sum = 0.0f;  // the reference that `sum` is relative to
      for (int j = first; j < last; ++j, ++n) {
        if ((n & 1) != group) continue;
        ok = warp_wait(&ctl.s_full[group], (n >> 1) & 1, p.status);
        if (!ok) break;
        tc_fence_after_sync();
        // the second half of the keys first: the first half stays in registers, and what P overwrites of S is of it
        uint32_t s[kKeys / 2];
        const int seen = limit - j * kKeys;
        const bool masked = active && __any_sync(0xffffffffu, seen < kKeys);
        float top = -INFINITY;
        if (active) {
          load_scores(at + kKeys / 2, masked, seen - kKeys / 2, s);
          top = top_of(s);
          load_scores(at, masked, seen, s);
          top = fmaxf(top, top_of(s));
        }
        if (n > 0) ok = warp_wait(&ctl.reference_set[group ^ 1][quadrant], ((n - 1) >> 1) & 1, p.status);
        if (!ok) break;
        const float before = j == first ? top : ctl.reference[r];
        const bool grown = (top - before) * c > 8.0f;
        const float now = grown ? top : before;
        ctl.reference[r] = now;
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.reference_set[group][quadrant]);
        if (active) {
          if (__any_sync(0xffffffffu, grown)) {
            // O of the steps before this one is complete, and none is added until P of this one is
            ok = warp_wait(&ctl.pv_done, (n - 1) & 1, p.status);
            if (!ok) break;
            tc_fence_after_sync();
            const float alpha = grown ? exp2_approx((before - now) * c) : 1.0f;
#pragma unroll 1
            for (int k = 0; k < D; k += 32) {
              uint32_t o[32];
              tmem_ld32(tmem_o + lanes + k, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st32(tmem_o + lanes + k, o);
            }
            tmem_st_wait();
            load_scores(at, masked, seen, s);  // rather than 64 registers kept over the wait
          }
          if (mine != now) sum *= exp2_approx((mine - now) * c);
          mine = now;
          const float shift = now == -INFINITY ? 0.0f : now * c;
          sum += weights_of(s, c, shift);
          tmem_st32(at, s);
          load_scores(at + kKeys / 2, masked, seen - kKeys / 2, s);
          sum += weights_of(s, c, shift);
          tmem_st32(at + kKeys / 4, s);
          tmem_st_wait();
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote_light(p_full_even);
      }
      if (!ok) break;
      if (item > 0) ok = warp_wait(&ctl.stats_free, (item - 1) & 1, p.status);  // the epilogue has read the last tile's
      if (!ok) break;
      ctl.row_max[group][r] = mine == -INFINITY ? -INFINITY : mine * c;
      ctl.row_sum[group][r] = sum;
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.stats_full);
      ++item;
    }
  } else {
    // ---------------------------------------------------------------- epilogue
    more_registers<kEpilogueRegisters>();
    const int quadrant = warp & 3, thread = static_cast<int>(threadIdx.x) - 384;
    const int r = quadrant * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quadrant * 32) << 16;
    const uint32_t o_free_even = mapa_u32(smem_u32(&ctl.o_free), 0);
    int item = 0;
    Stroll& stroll = ctl.strolls[warp - 4];
    stroll.begin(p, stretch, lane);
    const Item& it = stroll.it;
    bool ok = true;  // a warp whose wait ran out still takes part in the barriers of the four
    while (stroll.next(p, lane)) {
      const int rows = min(it.tokens - rank * p.half_tokens, p.half_tokens) * p.group;  // of this CTA, below 1: none
      const int tile_token = it.seq.start + it.tile * p.tile_tokens + rank * p.half_tokens;  // first token row
      const int ahead = it.seq.kv - it.seq.q + it.tile * p.tile_tokens + rank * p.half_tokens;
      const bool whole = it.first == 0 && it.last == it.steps;
      const bool mine = quadrant * 32 < rows;
      const uint4* gate = nullptr;
      if (p.gate && whole && mine) {
        gate = reinterpret_cast<const uint4*>(gate_row(p, tile_token, it.head, min(r, rows - 1)));
#pragma unroll
        for (int k = 0; k < D / 64; ++k) prefetch_l2(gate + 8 * k);
      }
      ok = ok && warp_wait(&ctl.stats_full, item & 1, p.status) && warp_wait(&ctl.o_full, item & 1, p.status);
      tc_fence_after_sync();
      const float m0 = ctl.row_max[0][r], m1 = ctl.row_max[1][r], m = fmaxf(m0, m1), base = m == -INFINITY ? 0.0f : m;
      const float sum = ctl.row_sum[0][r] * exp2_approx(m0 - base) + ctl.row_sum[1][r] * exp2_approx(m1 - base);
      if (whole) {
        const bool blind = ahead + r / p.group < 0;  // sees no key
        const F32x2 scale2 = f32x2_splat(blind ? 0.0f : 1.0f / sum);
        // The row leaves tensor memory in 16 bits a value, so that O is free for the next tile before gate and stores: as
        // the BF16 that is stored, or in front of a gate as FP16 times a power of two that puts the row's largest value
        // in [2^14, 2^15).  All values that are not zero then have to be normal there, 2^-28 of the largest or more, so that
        // each is rounded by 2^-11 of itself, where BF16 would take 2^-8.  A warp that has another row (with smaller
        // values, one that is infinite, or a largest one whose factor fp32 does not hold) gates its rows in fp32 as they leave.
        float up = 1.0f, down = 1.0f;
        bool direct = false;
        if (ok && mine && gate) {
          float most = 0.0f;
          uint32_t lowest = 0xffffffffu;  // of 2 |bits| - 1, which puts zeros behind all others
#pragma unroll
          for (int k = 0; k < D / 64; ++k) {
            uint32_t o[64];
            tmem_ld32(tmem_o + lanes + 64 * k, o);
            tmem_ld32(tmem_o + lanes + 64 * k + 32, o + 32);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 64; i += 2) {
              most = fmaxf(most, fmaxf(fabsf(__uint_as_float(o[i])), fabsf(__uint_as_float(o[i + 1]))));
              lowest = min(lowest, min(2 * o[i] - 1, 2 * o[i + 1] - 1));
            }
          }
          const float scale = fabsf(f32x2_parts(scale2).x);
          const float least = __uint_as_float((lowest + 1) >> 1) * scale;  // (with zeros alone, of no use)
          most *= scale;
          if (most >= 0x1p-90f && most <= 0x1p100f) {
            const int e = 141 - static_cast<int>(__float_as_uint(most) >> 23);  // 14 - exponent
            up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
            down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
            direct = least < most * 0x1p-28f;
          } else {
            direct = most != 0.0f;  // a row of zeros, or of zeros and NaN, waits as it is
          }
          direct = __any_sync(0xffffffffu, direct && !blind && r < rows);
        }
        const F32x2 factor = mul2(scale2, f32x2_splat(up));
        constexpr int HELD = D == 256 ? 64 : D / 2;  // words of a row in registers, the rest in shared memory
        uint32_t held[HELD];
        uint16_t* out = output_row<D>(p, tile_token, it.head, min(r, max(rows, 1) - 1));
        if (direct) {
#pragma unroll 1
          for (int k = 0; k < D / 16; ++k) {
            uint32_t o[16];
            tmem_ld16(tmem_o + lanes + 16 * k, o);
            const uint4 g[2] = {__ldg(gate + 2 * k), __ldg(gate + 2 * k + 1)};
            const uint32_t pairs[8] = {g[0].x, g[0].y, g[0].z, g[0].w, g[1].x, g[1].y, g[1].z, g[1].w};
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const F32x2 v = mul2(f32x2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])), scale2);
              o[i] = blind ? 0u : f32x2_to_bf16x2(gated(v, pairs[i]));  // (values 0 .. 2 i + 1 have been used)
            }
            if (r < rows) store_words8(out + 16 * k, o);
          }
        } else if (ok && mine) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            uint32_t o[16];
            tmem_ld16(tmem_o + lanes + 16 * k, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const F32x2 v = mul2(f32x2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1])), factor);
              const uint32_t w = gate ? f32x2_to_f16x2(v) : f32x2_to_bf16x2(v);
              if (8 * k < HELD) {
                held[(8 * k + i) % HELD] = blind ? 0u : w;
              } else {
                o[i] = blind ? 0u : w;  // (values 0 .. 2 i + 1 have been used)
              }
            }
            if (8 * k >= HELD) {
              ctl.rows[(8 * k - HELD) / 4][r] = make_uint4(o[0], o[1], o[2], o[3]);
              ctl.rows[(8 * k - HELD) / 4 + 1][r] = make_uint4(o[4], o[5], o[6], o[7]);
            }
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_remote_light(o_free_even);
          mbar_arrive(&ctl.stats_free);
        }
        if (ok && mine && !direct) {
          const F32x2 down2 = f32x2_splat(down);
#pragma unroll
          for (int k = 0; k < D / 32; ++k) {
            uint32_t w[16];
            if (16 * k < HELD) {
#pragma unroll
              for (int i = 0; i < 16; ++i) w[i] = held[(16 * k + i) % HELD];
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint4 v = ctl.rows[(16 * k - HELD) / 4 + e][r];
                w[4 * e] = v.x;
                w[4 * e + 1] = v.y;
                w[4 * e + 2] = v.z;
                w[4 * e + 3] = v.w;
              }
            }
            if (gate) {
              uint4 g[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) g[e] = __ldg(gate + 4 * k + e);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const uint32_t pair = i % 4 == 0 ? g[i / 4].x : i % 4 == 1 ? g[i / 4].y : i % 4 == 2 ? g[i / 4].z : g[i / 4].w;
                w[i] = f32x2_to_bf16x2(gated(mul2(f16x2_to_f32x2(w[i]), down2), pair));
              }
            }
            if (r < rows) {
              store_words8(out + 32 * k, w);
              store_words8(out + 32 * k + 16, w + 8);
            }
          }
        }
      } else {
        // the pair that the tile begins in, and the last one that it reaches, with the cuts where they moved to
        const int margin = cut_margin(p, it.tokens);
        const long long inner = static_cast<long long>(margin) * kKeys, cost = p.tile_keys + it.limit;
        const long long outer = max(inner, static_cast<long long>(it.steps - margin + 1) * kKeys);
        const int c0 = static_cast<int>(divide(it.line + min(inner, cost) - 1, stretch.share));
        const int c1 = static_cast<int>(divide(it.line + min(outer, cost) - 1, stretch.share));
        // the part that begins a tile goes to the CTA's slot 1, one that goes on with a tile to slot 0
        const size_t slot = 2 * static_cast<size_t>(blockIdx.x) + (it.first == 0 ? 1 : 0);
        float* part = p.parts + slot * kRows * D;
        if (ok && quadrant * 32 < rows) {
#pragma unroll 1
          for (int k = 0; k < D; k += 32) {
            uint32_t o[32];
            tmem_ld32(tmem_o + lanes + k, o);
            tmem_ld_wait();
            if (r < rows) {
              uint4* to = reinterpret_cast<uint4*>(part) + (k / 4) * kRows + r;
#pragma unroll
              for (int e = 0; e < 32; e += 4) to[e / 4 * kRows] = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
          }
          if (r < rows) p.part_stats[slot * kRows + r] = make_float2(m, sum);
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote_light(o_free_even);
        __threadfence();
        named_barrier(1, 128);
        unsigned int* ticket = p.tickets + 2 * c0 + rank;
        if (thread == 0) ctl.last_part = rows > 0 && atomicAdd(ticket, 1u) == static_cast<unsigned>(c1 - c0);
        named_barrier(1, 128);
        if (ctl.last_part) {
          __threadfence();
          // row_max and row_sum have been read by their rows' threads: here they hold what the parts have in common
          // What is faster, us of a launch at 24 over 4 heads of 256.  Eight lanes a row / one: 6 rows in 72 parts 33.5 / 40.1,
          // in 18 parts 20.9 / 22.6, 48 rows 61.7 / 63.0, 72 81.8 / 82.5, 90 100.4 / 99.9, 126 121.3 / 117.1; in 4 parts 54
          // rows 60.5 / 58.7, 90 69.8 / 65.6.  Rows by all threads / a thread each: 18 parts of 54 rows 69 / 111, of 96 97 /
          // 107, of 108 114 / 117, of 126 127 / 118; 12 parts of 90 66.9 / 69.8, of 108 64.2 / 62.6; 6 parts of 72 57.9 / 60.9,
          // of 90 68.8 / 64.4; 4 parts of 72 62.7 / 63.5, of 90 70.6 / 66.0; 2 parts of 54 84.8 / 90.1, of 72 90.6 / 89.8.
          const bool many = c1 - c0 >= 8;
          if (many && rows <= 72) {
            join_stats<8>(p, c0, c1, rank, rows, thread, ctl.row_max[0], ctl.row_sum[0]);
          } else {
            join_stats<1>(p, c0, c1, rank, rows, thread, ctl.row_max[0], ctl.row_sum[0]);
          }
          if (rows > (many ? 96 : 72)) {
            join_tall<D>(p, c0, c1, rank, rows, thread, ahead, tile_token, it.head, ctl.row_max[0], ctl.row_sum[0]);
          } else {
            join_rows<D>(p, c0, c1, rank, rows, thread, ahead, tile_token, it.head, ctl.row_max[0], ctl.row_sum[0]);
          }
          if (thread == 0) *ticket = 0u;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.stats_free);
        named_barrier(1, 128);  // `last_part` is written again
      }
      ++item;
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  cluster_arrive_relaxed();  // nothing of the other CTA's works on this one's memory any more
  cluster_wait_relaxed();
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

}  // namespace

template <int D, bool PAGED>
static cudaError_t prepare_one() {
  return cudaFuncSetAttribute(attention_kernel<D, PAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize, shared_bytes<D>());
}

cudaError_t attention_prepare() {
  cudaError_t e = prepare_one<256, true>();
  if (e == cudaSuccess) e = prepare_one<256, false>();
  if (e == cudaSuccess) e = prepare_one<128, true>();
  if (e == cudaSuccess) e = prepare_one<128, false>();
  return e;
}


cudaError_t launch_attention(cudaStream_t stream, int dim, int pairs, const CUtensorMap& map_q, const CUtensorMap& map_q1,
                             const CUtensorMap& map_k, const CUtensorMap& map_v, const AttentionParams& p) {
  auto kernel = p.block_table ? (dim == 256 ? attention_kernel<256, true> : attention_kernel<128, true>)
                              : (dim == 256 ? attention_kernel<256, false> : attention_kernel<128, false>);
  return launch_kernel_cluster(kernel, dim3(2 * pairs), dim3(kThreads), dim == 256 ? shared_bytes<256>() : shared_bytes<128>(),
                               stream, dim3(2, 1, 1), map_q, map_q1, map_k, map_v, p);
}

}  // namespace tk100
