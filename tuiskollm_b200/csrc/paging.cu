// Pages of the key/value cache handed out and taken back on the device.
//
// Requests own rows of a block table; pages come off the top of a stack of free ids in request order and
// go back onto it in request order.  With n_r new tokens behind l_r cached ones, request r needs
//     d_r = ceil((l_r + n_r) / P) - ceil(l_r / P)
// pages, the k-th page handed out (k counted over all requests: exclusive sum of d) is
// free_pages[free_count - 1 - k], and token i of request r lies at position l_r + i in slot
// page(position / P) * P + position % P.  All whole numbers, so the result is one result.
//
// One cluster of 1 to 8 CTAs.  Every CTA computes both exclusive sums over all requests for itself (they
// fit its shared memory), then the cluster meets once -- from there nobody reads the lengths, the counter
// or the pages' old owners again, so outputs may be the planes they were read from -- and the CTAs share the
// writing: a token or a new page finds its request by bisection of the sums.  Latency-bound: 8 requests of
// one token 3.8 us, 301 requests with 24000 tokens 12.
#include "common.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace tk100 {
namespace {

constexpr int kThreads = 1024;

struct Request {
  int token, page;  // tokens and pages of the requests in front
  int length, row;  // cached tokens before this call; row of the table
};

// Exclusive sum over the CTA of two counts; `carry` holds the sums of earlier rounds and is advanced.
__device__ __forceinline__ void scan_pair(long long& a, long long& b, long long (&carry)[2], long long (*warps)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long a0 = a, b0 = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) {
      a += x;
      b += y;
    }
  }
  if (lane == 31) {
    warps[warp][0] = a;
    warps[warp][1] = b;
  }
  __syncthreads();
  long long before[2] = {carry[0], carry[1]};
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) {
      before[0] += warps[w][0];
      before[1] += warps[w][1];
    }
    carry[0] += warps[w][0];
    carry[1] += warps[w][1];
  }
  a += before[0] - a0;
  b += before[1] - b0;
  __syncthreads();
}

// Last request whose first token (BY_PAGE: page) is at or before `at`; requests without any are passed over
// because the next one starts at the same place.
template <bool BY_PAGE>
__device__ __forceinline__ int request_of(const Request* r, int n, int at) {
  int low = 0, high = n;  // r[low] <= at < r[high]
  while (high - low > 1) {
    const int middle = (low + high) >> 1;
    if ((BY_PAGE ? r[middle].page : r[middle].token) <= at) {
      low = middle;
    } else {
      high = middle;
    }
  }
  return low;
}

template <bool RELEASE>
__global__ void __launch_bounds__(kThreads) page_kernel(const PageParams p) {
  extern __shared__ __align__(16) unsigned char shared[];
  Request* requests = reinterpret_cast<Request*>(shared);
  uint32_t* taken = reinterpret_cast<uint32_t*>(requests + p.requests);
  __shared__ long long warps[kThreads / 32][2];
  __shared__ int bad;

  const int words = (p.table_rows + 31) / 32;
  for (int i = threadIdx.x; i < words; i += kThreads) taken[i] = 0u;
  if (threadIdx.x == 0) bad = 0;
  pdl_wait();
  pdl_trigger();
  __syncthreads();

  const int page = p.page_tokens, shift = __ffs(page) - 1;
  const long long capacity = static_cast<long long>(p.max_pages) * page;
  const int free_count = *p.free_count;
  long long carry[2] = {0, 0};
  for (int first = 0; first < p.requests; first += kThreads) {
    const int i = first + static_cast<int>(threadIdx.x);
    long long tokens = 0, pages = 0;
    int length = 0, row = 0;
    if (i < p.requests) {
      row = p.request_rows ? p.request_rows[i] : i;
      const int fresh = RELEASE ? 0 : p.new_tokens[i];
      bool ok = row >= 0 && row < p.table_rows && fresh >= 0;
      // a row twice in one call would be handed, or give back, the same pages twice
      if (ok && ((atomicOr(&taken[row >> 5], 1u << (row & 31)) >> (row & 31)) & 1u)) ok = false;
      if (ok) length = p.lengths[row];
      ok = ok && length >= 0 && static_cast<long long>(length) + fresh <= capacity;
      if (!ok) {
        bad = 1;
      } else {
        tokens = fresh;
        const long long held = (static_cast<long long>(length) + page - 1) >> shift;
        pages = RELEASE ? held : ((static_cast<long long>(length) + fresh + page - 1) >> shift) - held;
      }
    }
    scan_pair(tokens, pages, carry, warps);
    if (i < p.requests) {
      requests[i] = {static_cast<int>(tokens), static_cast<int>(pages), length, row};
    }
  }
  __syncthreads();
  const long long tokens = carry[0], pages = carry[1];
  const bool fits = !bad && free_count >= 0 && free_count <= p.free_capacity &&
                    (RELEASE ? free_count + pages <= p.free_capacity : pages <= free_count && tokens <= p.max_tokens);
  cluster_arrive();
  cluster_wait();

  const int stride = static_cast<int>(gridDim.x) * kThreads;
  const int me = static_cast<int>(blockIdx.x) * kThreads + static_cast<int>(threadIdx.x);
  if (me == 0) {
    if (!fits) atomicOr(p.status, STATUS_BAD_ARGUMENT);
    *p.free_count_output = fits ? static_cast<int>(free_count + (RELEASE ? pages : -pages)) : free_count;
    if (!RELEASE) p.starts[p.requests] = fits ? static_cast<int>(tokens) : 0;
  }
  for (int i = me; i < p.requests; i += stride) {
    const Request r = requests[i];
    const int length = RELEASE ? 0 : r.length + p.new_tokens[i];
    if (!RELEASE) {
      p.starts[i] = fits ? r.token : 0;
      p.kv_lengths[i] = fits ? length : 0;
    }
    if (fits) {
      p.lengths_output[r.row] = length;
    } else if (p.lengths_output != p.lengths && r.row >= 0 && r.row < p.table_rows) {
      p.lengths_output[r.row] = p.lengths[r.row];
    }
  }
  if (fits) {
#pragma unroll 4
    for (int k = me; k < static_cast<int>(pages); k += stride) {
      const Request r = requests[request_of<true>(requests, p.requests, k)];
      int* line = p.block_table + static_cast<size_t>(r.row) * p.max_pages;
      if (RELEASE) {
        const int id = line[k - r.page];
        if (id < 0) atomicOr(p.status, STATUS_BAD_ARGUMENT);
        p.free_pages[free_count + k] = id;
      } else {
        line[((r.length + page - 1) >> shift) + (k - r.page)] = p.free_pages[free_count - 1 - k];
      }
    }
  }
  if constexpr (!RELEASE) {
#pragma unroll 4
    for (int t = me; t < p.max_tokens; t += stride) {
      int position = 0;
      long long slot = -1;
      if (fits && t < static_cast<int>(tokens)) {
        const Request r = requests[request_of<false>(requests, p.requests, t)];
        position = r.length + (t - r.token);
        // a page that this call hands out is read where it comes from, not where it is being written
        const int index = position >> shift, fresh = index - ((r.length + page - 1) >> shift);
        const int id = fresh < 0 ? p.block_table[static_cast<size_t>(r.row) * p.max_pages + index]
                                 : p.free_pages[free_count - 1 - (r.page + fresh)];
        if (id >= 0) {
          slot = (static_cast<long long>(id) << shift) + (position & (page - 1));
        } else {  // no page; a negative slot alone would pass for padding
          atomicOr(p.status, STATUS_BAD_ARGUMENT);
        }
      }
      p.positions[t] = position;
      p.slots[t] = slot;
    }
  }
}

size_t shared_bytes(const PageParams& p) {
  return static_cast<size_t>(p.requests) * sizeof(Request) + static_cast<size_t>((p.table_rows + 31) / 32) * 4;
}

}  // namespace

cudaError_t page_prepare() {
  const int most = kPageMaxRequests * static_cast<int>(sizeof(Request)) + kPageMaxRows / 8;
  cudaError_t e = cudaFuncSetAttribute(page_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e != cudaSuccess) return e;
  return cudaFuncSetAttribute(page_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
}

cudaError_t launch_page(cudaStream_t stream, const PageParams& p, bool release) {
  // CTAs by what there may be to write, two a thread: 24000 tokens of 301 requests 8 CTAs, 20000 pages of 37 the
  // same (a single one took 33 us).
  const long long work = release ? static_cast<long long>(p.requests) * p.max_pages : p.max_tokens;
  unsigned ctas = 1;
  while (ctas < 8 && static_cast<long long>(ctas) * 2 * kThreads < work) ctas *= 2;
  return launch_kernel_cluster(release ? page_kernel<true> : page_kernel<false>, dim3(ctas), dim3(kThreads),
                               shared_bytes(p), stream, dim3(ctas), p);
}

}  // namespace tk100
