// Rotary positions with several axes, fused with the head norms in front of them and the key/value cache
// behind them.
//
// A head x of D values, optionally normalised to y = x / sqrt(mean(x^2) + eps) * (1 + w), turns in the planes
// (y_i, y_{i + R/2}), i < R/2, by the angle a_i = position[axis_i] * frequency_i:
//     z_i = y_i cos a_i - y_{i + R/2} sin a_i,   z_{i + R/2} = y_{i + R/2} cos a_i + y_i sin a_i,
// and values from R on pass.  One rounding to BF16 at the end; sums, norm and products are fp32.
// The angle needs 64 bits: at position 10^6 one unit in the last place of an fp32 product is 0.06 rad.  It is
// formed in turns, position * (frequency / 2 pi), in double, its whole turns dropped there, and only the
// remainder in [-1/2, 1/2] is rounded to fp32 (3e-8 of a turn) for sincospif.
//
// Each query, key and value is read once and written once, 31 us at 8192 tokens of 32 + 8 heads of 128 where the kernel
// takes 48.5: bound by shared memory (partners by shuffle, sines with bank conflicts) at few warps, with norms by
// instruction issue; by latency for few tokens.
// A CTA has TOKENS tokens: its threads form their sines and cosines once for all heads while every thread already
// holds DEPTH heads' values; a head is DIM / 8 lanes of 16 bytes, so the partner of a lane in a rotation is R / 16
// lanes away and comes by shuffle.  One token a CTA leaves most threads idle in the first half and has its chain of
// loads, angles and stores to itself; four share it, at half of the CTAs an SM, which pays where the loop over heads is
// short: without norms and within one round of heads, or with norms within half of one.  us with one / with four, all with
// cache stores:
//                                 tokens      1024       1536       2048       4096       8192
//   32 + 8 + 8 heads of 128             9.0/ 7.9  12.6/13.8  16.0/14.4  28.6/27.2  53.8/47.7
//   the same with norms                10.8/10.5  15.3/18.6  19.6/19.4  35.1/36.5  66.5/63.9
//   24 + 4 + 4 of 256, 64 turned        8.9/ 8.6  12.3/14.2  15.7/15.5  28.1/28.6  52.5/51.5
//   the same with norms                11.5/12.1  16.1/21.4  20.2/22.5  35.9/41.6  67.1/73.3
//   64 + 8 + 8 of 128 (two rounds)     11.8/11.7  16.1/19.9  20.3/21.4  36.4/40.4  68.6/72.6
//   8 + 2 + 2 of 128 with norms         7.5/ 6.6  10.4/11.8  13.4/12.1  23.4/22.7  44.7/39.6
//   8 + 1 + 1 of 256 with norms         8.8/ 8.7  12.2/15.3  15.7/15.9  27.9/29.5  53.8/51.9
#include "common.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace tk100 {
namespace {

constexpr int kThreads = 256;
constexpr int kDepth = 4;  // heads of a thread in one round
constexpr int kRotaryManyTokens = 2048;

template <int DIM, int TOKENS>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
  constexpr int LANES = DIM / 8;             // lanes of a head
  constexpr int AT_ONCE = kThreads / LANES;  // heads of a CTA side by side
  constexpr int DEPTH = kDepth;              // and one behind the other, all of them requested at once
  __shared__ float2 turn[TOKENS][DIM / 2];
  __shared__ long long places[TOKENS];  // of the tokens in the cache, -1: nowhere
  pdl_wait();
  pdl_trigger();

  const int first_token = static_cast<int>(blockIdx.x) * TOKENS, tokens = min(TOKENS, p.tokens - first_token);
  const int lane = static_cast<int>(threadIdx.x) % LANES, group = static_cast<int>(threadIdx.x) / LANES;
  const int heads = p.q_heads + p.kv_heads + (p.key_cache ? p.kv_heads : 0);  // queries, keys, values for the cache

  // The thread's heads are the same ones for every token: where they are read, by how much a token moves that, and
  // what becomes of them are found once.
  const uint16_t* from[DEPTH];
  int token_stride[DEPTH];
  auto find = [&](int base) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      int h = min(base + d * AT_ONCE + group, heads - 1);
      const bool query = h < p.q_heads;
      if (!query) h -= p.q_heads;
      const uint16_t* plane = query ? p.query : h < p.kv_heads ? p.key : p.value;
      if (!query && h >= p.kv_heads) h -= p.kv_heads;
      token_stride[d] = query ? p.query_token_stride : p.kv_token_stride;
      from[d] = plane + static_cast<size_t>(first_token) * token_stride[d] +
                static_cast<size_t>(h) * (query ? p.query_head_stride : p.kv_head_stride) + 8 * lane;
    }
  };
  uint4 raw[DEPTH];
  auto request = [&](int t) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
      raw[d] = *reinterpret_cast<const uint4*>(from[d] + static_cast<size_t>(t) * token_stride[d]);
  };
  find(0);
  request(0);

  for (int i = threadIdx.x; i < tokens * p.half; i += kThreads) {
    const int t = TOKENS == 1 ? 0 : i / p.half, pair = i - t * p.half;
    int axis = p.pair_axes ? p.pair_axes[pair] : 0;
    if (axis >= p.axes) {
      axis = 0;
      if (blockIdx.x == 0) atomicOr(p.status, STATUS_BAD_ARGUMENT);
    }
    const double turns = static_cast<double>(p.positions[static_cast<size_t>(axis) * p.tokens + first_token + t]) *
                         (p.frequencies[pair] * 0.15915494309189533577);  // 1 / (2 pi)
    const float rest = static_cast<float>(turns - rint(turns));
    float s, c;
    sincospif(2.0f * rest, &s, &c);
    turn[t][pair] = make_float2(c, s);
  }
  // where the tokens' keys and values go; a negative slot (a padded row) goes nowhere
  if (p.key_cache && static_cast<int>(threadIdx.x) < tokens) {
    const long long slot = p.slots[first_token + threadIdx.x];
    const long long page = slot >> p.page_shift;
    long long place = -1;
    if (slot >= 0 && page < p.pages) {
      place = page * p.page_stride + (slot & ((1ll << p.page_shift) - 1)) * p.cache_token_stride;
    } else if (slot >= 0) {
      atomicOr(p.status, STATUS_BAD_ARGUMENT);
    }
    places[threadIdx.x] = place;
  }
  __syncthreads();

  const int rotary_lanes = p.half / 8;  // lanes of the first half of the rotated values
  const bool first_half = lane < rotary_lanes, second_half = !first_half && lane < 2 * rotary_lanes;
  const int partner = first_half ? lane + rotary_lanes : second_half ? lane - rotary_lanes : lane;
  const int pair0 = first_half ? 8 * lane : second_half ? 8 * (lane - rotary_lanes) : 0;
  const bool normed = p.query_norm || p.key_norm;

  for (int base = 0; base < heads; base += DEPTH * AT_ONCE) {
    if (base > 0) {
      find(base);
      request(0);
    }
#pragma unroll 1
    for (int t = 0; t < tokens; ++t) {
      uint4 now[DEPTH];
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) now[d] = raw[d];
      if (t + 1 < tokens) request(t + 1);
      const size_t token = static_cast<size_t>(first_token + t);
      const long long place = p.key_cache ? places[t] : -1;
      float2 cs[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cs[j] = turn[t][pair0 + j];
        if (first_half) cs[j].y = -cs[j].y;
      }
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        if (base + d * AT_ONCE >= heads) break;
        const int h = base + d * AT_ONCE + group;
        const bool query = h < p.q_heads, key = !query && h < p.q_heads + p.kv_heads;
        const uint16_t* norm = query ? p.query_norm : key ? p.key_norm : nullptr;
        const uint32_t w[4] = {now[d].x, now[d].y, now[d].z, now[d].w};
        float y[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          y[2 * j] = bf16x2_lo(w[j]);
          y[2 * j + 1] = bf16x2_hi(w[j]);
        }
        if (normed) {  // (all lanes: a warp may have heads of two kinds)
          float sum = 0.0f;
#pragma unroll
          for (int j = 0; j < 8; ++j) sum = fmaf(y[j], y[j], sum);
#pragma unroll
          for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          if (norm) {
            const float scale = __frsqrt_rn(sum * (1.0f / DIM) + p.epsilon);
            const uint4 n = __ldg(reinterpret_cast<const uint4*>(norm + 8 * lane));
            const uint32_t v[4] = {n.x, n.y, n.z, n.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              y[2 * j] = y[2 * j] * scale * (1.0f + bf16x2_lo(v[j]));
              y[2 * j + 1] = y[2 * j + 1] * scale * (1.0f + bf16x2_hi(v[j]));
            }
          }
        }
        uint32_t r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a = __shfl_sync(0xffffffffu, y[2 * j], partner, LANES), b = __shfl_sync(0xffffffffu, y[2 * j + 1], partner, LANES);
          // a lane behind the rotated values passes its own on, whatever their sign or kind
          const bool turns = first_half || second_half;
          r[j] = pack_bf16x2(turns ? fmaf(y[2 * j], cs[2 * j].x, a * cs[2 * j].y) : y[2 * j],
                             turns ? fmaf(y[2 * j + 1], cs[2 * j + 1].x, b * cs[2 * j + 1].y) : y[2 * j + 1]);
        }
        if (h >= heads) continue;
        const uint4 result = query || key ? make_uint4(r[0], r[1], r[2], r[3]) : now[d];
        if (query) {
          *reinterpret_cast<uint4*>(p.query_output + (token * p.q_heads + h) * DIM + 8 * lane) = result;
        } else {
          const int k = h - p.q_heads - (key ? 0 : p.kv_heads);
          if (place >= 0)
            *reinterpret_cast<uint4*>((key ? p.key_cache : p.value_cache) + place + static_cast<size_t>(k) * p.cache_head_stride + 8 * lane) = result;
          if (key && p.key_output)
            *reinterpret_cast<uint4*>(p.key_output + (token * p.kv_heads + k) * DIM + 8 * lane) = result;
        }
      }
    }
  }
}

template <int TOKENS>
cudaError_t launch(cudaStream_t stream, int dim, const RotaryParams& p) {
  return launch_kernel(dim == 256 ? rotary_kernel<256, TOKENS> : rotary_kernel<128, TOKENS>,
                       dim3((p.tokens + TOKENS - 1) / TOKENS), dim3(kThreads), 0, stream, p);
}

}  // namespace

cudaError_t launch_rotary(cudaStream_t stream, int dim, const RotaryParams& p) {
  const int heads = p.q_heads + p.kv_heads + (p.key_cache ? p.kv_heads : 0), round = kDepth * (kThreads * 8 / dim);
  const bool four = p.tokens >= kRotaryManyTokens && heads <= (p.query_norm || p.key_norm ? round / 2 : round);
  return four ? launch<4>(stream, dim, p) : launch<1>(stream, dim, p);
}

}  // namespace tk100
