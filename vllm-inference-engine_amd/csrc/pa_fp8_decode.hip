// Decode attention over the 8-bit paged pool: launch plan, argument checks and the C entry
// points. The kernel is in pa_fp8_attend.h.
#include "../../include/paged_attention.h"
#include "pa_fp8_attend.h"

namespace pa {
namespace fp8 {

DecodePlan decode_plan(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                       int block_size, int max_blocks, int new_tokens) {
  DecodePlan p{};
  const int n = device_cus();
  const bool multi = new_tokens > 0;
  const int64_t cap = (int64_t)max_blocks * block_size;
  // Two kv heads per pair read rows of twice the bytes and halve the merges. Measured on
  // MI355X at 14 / 2 heads of 64, one head against two, (sequence, head) pairs more than
  // compute units: 256 x ~4.6k tokens 103.7 against 62.2 us, 140 x 4k 34.0 against 25.0 (300 x
  // 1k 17.7 against 18.1); fewer, in ranges: 128 x 4k 28.8 against 23.6, 64 x 4k 18.7 against
  // 18.2, 8 x 4k 12.0 against 14.4, and 12 x 4k at 16 heads 35.8 against 22.7; fewer, as whole
  // pairs: 100 x 2k 14.4 against 17.8.
  const int64_t total = (int64_t)num_seqs * num_kv_heads;
  p.head_group = !multi && head_dim <= 64 && num_kv_heads % 2 == 0 &&
                         (total > n || (2 * total > n && cap > kWholePairsBusy)) ? 2 : 1;
  const int64_t pairs = total / p.head_group;
  // Few pairs: one workgroup of eight wavefronts per compute unit, which halves the parts of
  // a merge, instead of two of four. Measured on MI355X: one sequence of 24001 tokens 13.5
  // against 15.2 us, of 300 6.5 against 6.9; 4 x 5 drafts of 8k 25.1 against 29.4. One range
  // per compute unit also at head_dim 256, of four wavefronts there, against two: at 16 / 2
  // heads 8 x 8k 19.8 for either, 32 x 8k 38.9 against 41.6, 4 x 32k 35.2 against 40.9, 100 x 4k
  // 55.2 against 58.9.
  const bool few = p.head_group == 1 && pairs <= n;
  p.waves = few && head_dim <= 128 ? 8 : 4;
  const int64_t whole = 2 * pairs >= n ? kWholePairsBusy : kWholePairs;
  p.ranged = cap > whole && pairs <= kMaxCounters &&
             pairs * ((cap + kChunk - 1) / kChunk + kPairCost) < 0x7fffffff;
  p.grid = pairs > 0x7fffffff ? -1 : (int)pairs;
  if (p.ranged) {
    // No more ranges than the longest lengths fill.
    const int64_t most = pairs * ((cap + kChunk - 1) / kChunk + kPairCost) / kMinRange;
    const int want = (few ? 1 : 2) * n;
    p.grid = (int)(most < want ? (most < 1 ? 1 : most) : want);
    const int heads = num_q_heads / num_kv_heads * p.head_group * (multi ? new_tokens : 1);
    p.rec_floats = record_size(heads, head_dim);
    p.ws_bytes =
        kCounterBytes + (size_t)2 * p.grid * p.rec_floats * sizeof(float);
  }
  return p;
}

static bool decode_sizes_ok(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                            int block_size, int max_blocks) {
  return num_seqs > 0 && num_q_heads > 0 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0 &&
         num_q_heads / num_kv_heads <= 16 && block_size > 0 && max_blocks > 0 &&
         (int64_t)max_blocks * block_size <= 0x7fffffff - 4096 &&
         (head_dim == 32 || head_dim == 64 || head_dim == 128 || head_dim == 256);
}

template <int D, int HG, int NW>
static void launch_decode_bs(const DecodeFp8Args& a, unsigned grid, hipStream_t s) {
  const bool near = near_strides(a);
  if (a.bs == 16 && near)
    attend_fp8_kernel<D, HG, 16, NW, 1, false><<<grid, 64 * NW, 0, s>>>(a);
  else if (a.bs == 32 && near)
    attend_fp8_kernel<D, HG, 32, NW, 1, false><<<grid, 64 * NW, 0, s>>>(a);
  else
    attend_fp8_kernel<D, HG, 0, NW, 1, false><<<grid, 64 * NW, 0, s>>>(a);
}

static hipError_t launch_decode(const DecodeFp8Args& a, int D, const DecodePlan& p, hipStream_t s) {
  const unsigned grid = (unsigned)p.grid;
  switch (D * 16 + p.head_group + p.waves) {
    case 32 * 16 + 1 + 4: launch_decode_bs<32, 1, 4>(a, grid, s); break;
    case 32 * 16 + 1 + 8: launch_decode_bs<32, 1, 8>(a, grid, s); break;
    case 32 * 16 + 2 + 4: launch_decode_bs<32, 2, 4>(a, grid, s); break;
    case 64 * 16 + 1 + 4: launch_decode_bs<64, 1, 4>(a, grid, s); break;
    case 64 * 16 + 1 + 8: launch_decode_bs<64, 1, 8>(a, grid, s); break;
    case 64 * 16 + 2 + 4: launch_decode_bs<64, 2, 4>(a, grid, s); break;
    case 128 * 16 + 1 + 4: launch_decode_bs<128, 1, 4>(a, grid, s); break;
    case 128 * 16 + 1 + 8: launch_decode_bs<128, 1, 8>(a, grid, s); break;
    case 256 * 16 + 1 + 4: launch_decode_bs<256, 1, 4>(a, grid, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace fp8
}  // namespace pa

using namespace pa;
using namespace pa::fp8;

extern "C" {

size_t pa_decode_fp8_workspace_bytes(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                                     int block_size, int max_blocks_per_seq) {
  if (!decode_sizes_ok(num_seqs, num_q_heads, num_kv_heads, head_dim, block_size,
                       max_blocks_per_seq))
    return 0;
  return decode_plan(num_seqs, num_q_heads, num_kv_heads, head_dim, block_size,
                     max_blocks_per_seq, 0).ws_bytes;
}

int pa_decode_fp8(const void* q, const int64_t q_strides[3], const void* k_cache,
                  const int64_t k_strides[4], const void* v_cache, const int64_t v_strides[4],
                  const float* k_scale, const int64_t k_scale_strides[2], const float* v_scale,
                  const int64_t v_scale_strides[2], const int32_t* block_tables,
                  const int64_t bt_strides[2], const int32_t* seq_lens, void* out,
                  const int64_t out_strides[3], int num_seqs, int num_q_heads, int num_kv_heads,
                  int head_dim, int block_size, int num_blocks, int max_blocks_per_seq, float scale,
                  void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (num_seqs < 0) {
    set_error("num_seqs must be >= 0");
    return PA_ERR_ARG;
  }
  if (num_seqs == 0) return PA_OK;
  if (num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0) {
    set_error("num_q_heads (%d) must be divisible by num_kv_heads (%d)", num_q_heads, num_kv_heads);
    return PA_ERR_ARG;
  }
  if (block_size <= 0 || num_blocks <= 0 || max_blocks_per_seq <= 0) {
    set_error("block_size (%d), num_blocks (%d) and the table width (%d) must be positive",
              block_size, num_blocks, max_blocks_per_seq);
    return PA_ERR_ARG;
  }
  if (!decode_sizes_ok(num_seqs, num_q_heads, num_kv_heads, head_dim, block_size,
                       max_blocks_per_seq)) {
    set_error("not built: head_dim %d (32, 64, 128, 256), query group size %d (at most 16), or "
              "tables of 2^31 tokens", head_dim, num_q_heads / num_kv_heads);
    return PA_ERR_UNSUPPORTED;
  }
  if (!q || !q_strides || !k_cache || !k_strides || !v_cache || !v_strides || !k_scale ||
      !k_scale_strides || !v_scale || !v_scale_strides || !block_tables || !bt_strides ||
      !seq_lens || !out || !out_strides) {
    set_error("null pointer argument");
    return PA_ERR_ARG;
  }
  for (int i = 0; i < 3; ++i) {
    if (k_strides[i] % 16 || v_strides[i] % 16 || k_strides[i] < 0 || v_strides[i] < 0) {
      set_error("cache strides must be non-negative multiples of 16 bytes");
      return PA_ERR_ARG;
    }
  }
  if (k_strides[3] != 1 || v_strides[3] != 1 || q_strides[2] != 1 || out_strides[2] != 1 ||
      q_strides[0] % 8 || q_strides[1] % 8 || out_strides[0] % 4 || out_strides[1] % 4) {
    set_error("q, out and the caches need unit head_dim stride, q 8-element and out 4-element "
              "aligned strides");
    return PA_ERR_ARG;
  }
  if ((uintptr_t)q % 16 || (uintptr_t)k_cache % 16 || (uintptr_t)v_cache % 16 || (uintptr_t)out % 8) {
    set_error("q and the caches must be 16-byte aligned and out 8-byte aligned");
    return PA_ERR_ARG;
  }
  const DecodePlan p = decode_plan(num_seqs, num_q_heads, num_kv_heads, head_dim, block_size,
                                   max_blocks_per_seq, 0);
  if (p.ws_bytes && (!workspace || workspace_bytes < p.ws_bytes)) {
    set_error("workspace of %zu bytes needed, %zu given", p.ws_bytes, workspace_bytes);
    return PA_ERR_WORKSPACE;
  }
  if (p.grid < 0) {
    set_error("%d sequences of %d kv heads exceed one launch", num_seqs, num_kv_heads);
    return PA_ERR_UNSUPPORTED;
  }
  DecodeFp8Args a{};
  a.q = (const f16*)q;
  a.q_sb = q_strides[0];
  a.q_sh = q_strides[1];
  a.k = (const uint8_t*)k_cache;
  a.k_sb = k_strides[0];
  a.k_st = k_strides[1];
  a.k_sh = k_strides[2];
  a.v = (const uint8_t*)v_cache;
  a.v_sb = v_strides[0];
  a.v_st = v_strides[1];
  a.v_sh = v_strides[2];
  a.ks = k_scale;
  a.ks_sb = k_scale_strides[0];
  a.ks_sh = k_scale_strides[1];
  a.vs = v_scale;
  a.vs_sb = v_scale_strides[0];
  a.vs_sh = v_scale_strides[1];
  a.bt = block_tables;
  a.bt_sb = bt_strides[0];
  a.bt_sk = bt_strides[1];
  a.lens = seq_lens;
  a.out = (f16*)out;
  a.o_sb = out_strides[0];
  a.o_sh = out_strides[1];
  a.num_seqs = num_seqs;
  a.hkv = num_kv_heads;
  a.g = num_q_heads / num_kv_heads;
  a.bs = block_size;
  a.num_blocks = num_blocks;
  a.max_blocks = max_blocks_per_seq;
  p.fill(a, workspace);
  a.scale_log2 = scale * kLog2e;
  const hipError_t e = launch_decode(a, head_dim, p, (hipStream_t)stream);
  if (e == hipSuccess) return PA_OK;
  set_error("HIP launch failed: %s", hipGetErrorString(e));
  return PA_ERR_HIP;
}

}  // extern "C"
