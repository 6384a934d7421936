// Blocks of a paged pool copied to other blocks, in many tensors at once (gfx950).
//
//   t[dst[i]] = t[src[i]]  for every tensor t (K and V of all layers, scales) and pair i
//
// The copies behind a fork of a sequence (its last, partly filled block), beams that take
// over others' blocks and contexts that are moved together. One launch for all tensors:
// their addresses travel in the launch's arguments. Bound by memory, a block read and
// written once; for a few blocks by the chain launch -> ids -> block. Each wavefront takes
// one piece of a block, U loads per lane on their way at once; blocks smaller than a
// piece share wavefronts by lane. On MI355X, 24 layers of 4 KB blocks: 700 pairs in 53.6 us (275
// MB read and written, 5.1 TB/s; a large copy runs at 5.4), 7 pairs in 2.8 us, 6.6 with the host.
#include <algorithm>

#include "../../include/paged_attention.h"
#include "pa_common.h"
#include "pa_tiles.h"

namespace pa {
namespace blocks {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxTensors = 96;  // of a launch
constexpr int kU = 4;            // loads of a lane on their way

struct Entry {
  char* base;
  int64_t stride;  // bytes from block to block
  int bytes;       // of a block
  int width;       // bytes of a lane's load: 16, 4 or 1
};

struct Args {
  const int32_t* src;
  int64_t src_s;
  const int32_t* dst;
  int64_t dst_s;
  int pairs, num_blocks;
  Entry t[kMaxTensors];
};

// Wavefronts that the pairs of a tensor take.
__host__ __device__ inline int64_t waves_of(int bytes, int width, int pairs) {
  const int lane_words = bytes / width;  // words of a block
  if (lane_words >= 64 * kU)
    return (int64_t)pairs * ((lane_words + 64 * kU - 1) / (64 * kU));
  return ((int64_t)pairs * lane_words + 64 * kU - 1) / (64 * kU);
}

template <typename W>
__device__ inline void copy_piece(const Args& a, const Entry& t, int64_t item, int lane) {
  const int words = t.bytes / (int)sizeof(W);
  auto word = [&](int32_t id, int w) { return reinterpret_cast<W*>(t.base + id * t.stride) + w; };
  auto inside = [&](int id) { return (unsigned)id < (unsigned)a.num_blocks; };
  W x[kU];
  if (words >= 64 * kU) {  // a piece of one block
    const int pieces = (words + 64 * kU - 1) / (64 * kU);
    const int pair = (int)(item / pieces);
    const int w0 = (int)(item - (int64_t)pair * pieces) * 64 * kU + lane;
    const int from = tiles::load_uniform(a.src + pair * a.src_s);
    const int to = tiles::load_uniform(a.dst + pair * a.dst_s);
    if (!inside(from) || !inside(to)) return;
    const W* in = word(from, w0);
    W* out = word(to, w0);
    if (w0 - lane + 64 * kU <= words) {
#pragma unroll
      for (int u = 0; u < kU; ++u) x[u] = __builtin_nontemporal_load(in + u * 64);
#pragma unroll
      for (int u = 0; u < kU; ++u) __builtin_nontemporal_store(x[u], out + u * 64);
    } else {
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (w0 + u * 64 < words) x[u] = in[u * 64];
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (w0 + u * 64 < words) out[u * 64] = x[u];
    }
    return;
  }
  // Words of small blocks, pair after pair.
  W* out[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const int64_t i = (item * kU + u) * 64 + lane;
    out[u] = nullptr;
    if (i < (int64_t)a.pairs * words) {
      const int pair = (int)(i / words), w = (int)(i - (int64_t)pair * words);
      const int from = a.src[pair * a.src_s], to = a.dst[pair * a.dst_s];
      if (inside(from) && inside(to)) {
        x[u] = *word(from, w);
        out[u] = word(to, w);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kU; ++u)
    if (out[u]) *out[u] = x[u];
}

// blockIdx.y: the tensor.
__global__ __launch_bounds__(kThreads) void copy_blocks_kernel(Args a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = (int64_t)blockIdx.x * kWaves + wave;
  const Entry t = a.t[blockIdx.y];
  if (item >= waves_of(t.bytes, t.width, a.pairs)) return;
  if (t.width == 16)
    copy_piece<tiles::u32x4>(a, t, item, lane);
  else if (t.width == 4)
    copy_piece<unsigned>(a, t, item, lane);
  else
    copy_piece<unsigned char>(a, t, item, lane);
}

}  // namespace blocks
}  // namespace pa

using namespace pa;
using namespace pa::blocks;

extern "C" int pa_copy_blocks(void* const* tensors, const int64_t* block_strides,
                              const int64_t* block_bytes, int num_tensors,
                              const int32_t* src_blocks, int64_t src_stride,
                              const int32_t* dst_blocks, int64_t dst_stride, int num_pairs,
                              int num_blocks, void* stream) {
  clear_error();
  if (num_tensors < 0 || num_pairs < 0 || num_blocks < 0) {
    set_error("num_tensors (%d), num_pairs (%d) and num_blocks (%d) must be >= 0", num_tensors,
              num_pairs, num_blocks);
    return PA_ERR_ARG;
  }
  if (num_tensors == 0 || num_pairs == 0 || num_blocks == 0) return PA_OK;
  if (!tensors || !block_strides || !block_bytes || !src_blocks || !dst_blocks) {
    set_error("null pointer argument");
    return PA_ERR_ARG;
  }
  // All of them are looked at before the first launch.
  for (int i = 0; i < num_tensors; ++i) {
    if (!tensors[i] && block_bytes[i] != 0) {
      set_error("null pointer argument (tensor %d)", i);
      return PA_ERR_ARG;
    }
    if (block_bytes[i] < 0 || block_strides[i] < block_bytes[i]) {
      set_error("tensor %d: blocks of %lld bytes must not overlap (%lld bytes apart)", i,
                (long long)block_bytes[i], (long long)block_strides[i]);
      return PA_ERR_ARG;
    }
    if (block_bytes[i] > 0x7fffffff - 4096) {
      set_error("tensor %d: a block of %lld bytes is not built", i, (long long)block_bytes[i]);
      return PA_ERR_UNSUPPORTED;
    }
  }
  Args a;
  a.src = src_blocks;
  a.src_s = src_stride;
  a.dst = dst_blocks;
  a.dst_s = dst_stride;
  a.pairs = num_pairs;
  a.num_blocks = num_blocks;
  for (int pass = 0; pass < 2; ++pass) {  // the sizes of all launches, then the launches
    for (int first = 0; first < num_tensors; first += kMaxTensors) {
      int n = 0;
      int64_t most = 0;
      for (int i = first; i < std::min(num_tensors, first + kMaxTensors); ++i) {
        if (block_bytes[i] == 0) continue;
        const uintptr_t bits = (uintptr_t)tensors[i] | (uintptr_t)block_bytes[i] |
                               (num_blocks > 1 ? (uintptr_t)block_strides[i] : 0);
        Entry& t = a.t[n++];
        t.base = (char*)tensors[i];
        t.stride = block_strides[i];
        t.bytes = (int)block_bytes[i];
        t.width = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
        most = std::max(most, waves_of(t.bytes, t.width, num_pairs));
      }
      const int64_t grid = (most + kWaves - 1) / kWaves;
      if (grid > 0x7fffff) {
        set_error("%d pairs of these blocks exceed one launch", num_pairs);
        return PA_ERR_UNSUPPORTED;
      }
      if (pass == 0 || n == 0) continue;
      copy_blocks_kernel<<<dim3((unsigned)grid, n), kThreads, 0, (hipStream_t)stream>>>(a);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) {
        set_error("HIP launch failed: %s", hipGetErrorString(e));
        return PA_ERR_HIP;
      }
    }
  }
  return PA_OK;
}
