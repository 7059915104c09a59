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
// HBM-bound for many tokens (each query, key and value read once and written once), latency-bound for few.
// One CTA per token: R/2 threads form the token's sines and cosines once for all heads while every warp
// already holds its first head; a head is DIM / 8 lanes of 16 bytes, so the partner of a lane in a rotation is
// R / 16 lanes away and comes by shuffle.
#include "common.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace tk100 {
namespace {

constexpr int kThreads = 256;

template <int DIM>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p) {
  constexpr int LANES = DIM / 8;             // lanes of a head
  constexpr int AT_ONCE = kThreads / LANES;  // heads of a CTA side by side
  __shared__ float2 turn[DIM / 2];
  pdl_wait();
  pdl_trigger();

  const int token = static_cast<int>(blockIdx.x);
  const int lane = static_cast<int>(threadIdx.x) % LANES, group = static_cast<int>(threadIdx.x) / LANES;
  const int cached = p.key_cache ? p.kv_heads : 0;
  const int heads = p.q_heads + p.kv_heads + cached;  // queries, keys, values that go to the cache

  auto load = [&](int h) -> uint4 {
    const uint16_t* src;
    if (h < p.q_heads) {
      src = p.query + static_cast<size_t>(token) * p.query_token_stride + static_cast<size_t>(h) * p.query_head_stride;
    } else {
      h -= p.q_heads;
      src = p.key;
      if (h >= p.kv_heads) {
        h -= p.kv_heads;
        src = p.value;
      }
      src += static_cast<size_t>(token) * p.kv_token_stride + static_cast<size_t>(h) * p.kv_head_stride;
    }
    return *reinterpret_cast<const uint4*>(src + 8 * lane);
  };

  uint4 raw = make_uint4(0u, 0u, 0u, 0u);
  if (group < heads) raw = load(group);

  for (int i = threadIdx.x; i < p.half; i += kThreads) {
    int axis = p.pair_axes ? p.pair_axes[i] : 0;
    if (axis >= p.axes) {
      axis = 0;
      if (token == 0) atomicOr(p.status, STATUS_BAD_ARGUMENT);
    }
    const double turns = static_cast<double>(p.positions[static_cast<size_t>(axis) * p.tokens + token]) *
                         (p.frequencies[i] * 0.15915494309189533577);  // 1 / (2 pi)
    const float rest = static_cast<float>(turns - rint(turns));
    float s, c;
    sincospif(2.0f * rest, &s, &c);
    turn[i] = make_float2(c, s);
  }

  // where the token's keys and values go; a negative slot (a padded row) goes nowhere
  bool stored = false;
  size_t place = 0;
  if (p.key_cache) {
    const long long slot = p.slots[token];
    const long long page = slot >> p.page_shift;
    stored = slot >= 0 && page < p.pages;
    if (stored) {
      place = static_cast<size_t>(page) * p.page_stride +
              static_cast<size_t>(slot & ((1ll << p.page_shift) - 1)) * p.cache_token_stride;
    } else if (slot >= 0 && threadIdx.x == 0) {
      atomicOr(p.status, STATUS_BAD_ARGUMENT);
    }
  }
  __syncthreads();

  const int rotary_lanes = p.half / 8;  // lanes of the first half of the rotated values
  const bool first_half = lane < rotary_lanes, second_half = !first_half && lane < 2 * rotary_lanes;
  const int partner = first_half ? lane + rotary_lanes : second_half ? lane - rotary_lanes : lane;
  float2 mine[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = (first_half ? lane : lane - rotary_lanes) * 8 + j;
    mine[j] = first_half || second_half ? turn[i] : make_float2(1.0f, 0.0f);
    if (first_half) mine[j].y = -mine[j].y;
  }

  for (int base = 0; base < heads; base += AT_ONCE) {
    const int h = base + group;
    const uint4 now = raw;
    if (h + AT_ONCE < heads) raw = load(h + AT_ONCE);
    uint16_t* out = nullptr;
    uint16_t* second = nullptr;
    const uint16_t* norm = nullptr;
    bool turns = true;
    if (h < p.q_heads) {
      out = p.query_output + (static_cast<size_t>(token) * p.q_heads + h) * DIM;
      norm = p.query_norm;
    } else if (h < p.q_heads + p.kv_heads) {
      const int k = h - p.q_heads;
      if (stored) out = p.key_cache + place + static_cast<size_t>(k) * p.cache_head_stride;
      if (p.key_output) second = p.key_output + (static_cast<size_t>(token) * p.kv_heads + k) * DIM;
      norm = p.key_norm;
    } else if (h < heads) {
      if (stored) out = p.value_cache + place + static_cast<size_t>(h - p.q_heads - p.kv_heads) * p.cache_head_stride;
      turns = false;
    }
    uint4 result = now;
    const uint32_t w[4] = {now.x, now.y, now.z, now.w};
    float y[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      y[2 * j] = bf16x2_lo(w[j]);
      y[2 * j + 1] = bf16x2_hi(w[j]);
    }
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(y[j], y[j], sum);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (norm) {
      const float scale = __frsqrt_rn(sum * (1.0f / DIM) + p.epsilon);
      const uint4 n = *reinterpret_cast<const uint4*>(norm + 8 * lane);
      const uint32_t v[4] = {n.x, n.y, n.z, n.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[2 * j] = y[2 * j] * scale * (1.0f + bf16x2_lo(v[j]));
        y[2 * j + 1] = y[2 * j + 1] * scale * (1.0f + bf16x2_hi(v[j]));
      }
    }
    float other[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) other[j] = __shfl_sync(0xffffffffu, y[j], partner, LANES);
    if (turns) {
      uint32_t r[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float z[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = 2 * j + e;
          // a lane behind the rotated values passes its own on, whatever its sign or kind
          z[e] = first_half || second_half ? fmaf(y[i], mine[i].x, other[i] * mine[i].y) : y[i];
        }
        r[j] = pack_bf16x2(z[0], z[1]);
      }
      result = make_uint4(r[0], r[1], r[2], r[3]);
    }
    if (out) *reinterpret_cast<uint4*>(out + 8 * lane) = result;
    if (second) *reinterpret_cast<uint4*>(second + 8 * lane) = result;
  }
}

}  // namespace

cudaError_t launch_rotary(cudaStream_t stream, int dim, const RotaryParams& p) {
  return launch_kernel(dim == 256 ? rotary_kernel<256> : rotary_kernel<128>, dim3(p.tokens), dim3(kThreads), 0, stream, p);
}

}  // namespace tk100
