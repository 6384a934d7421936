// The few-tokens form of the 8-bit attention (pa_fp8_attend.h): drafted tokens, short chunks.
//
// The prefill kernel stages K and V once per 64 or 128 columns of tokens x query heads; with
// a few columns it spends its time on the ones that are not there, and on key ranges too
// few to fill the GPU: 16 sequences of 0.3k to 4k tokens and 5 drafts at 32 / 8 heads of 128
// take 59 us there and 31 here (MI355X).
#include "../../include/paged_attention.h"
#include "pa_fp8_attend.h"

namespace pa {
namespace fp8 {

// (Calls take the same workspaces as the prefill kernel's.)
static_assert(kCounterBytes == kPfCounterBytes, "counters, and nothing else, where it has its own");

// Columns of a sequence and kv head that the registers hold: four blocks of 16, or two at
// head_dim 128 (four would spill 91 registers there). At the full number the prefill kernel
// against this one on MI355X: 100 x 9 tokens on up to 4k at 14 / 2 heads of 64 53.2 against 36.4
// us, 16 x 9 18.2 for either, 16 x 8 at 32 / 8 heads of 128 59.8 against 32.9. What it costs to
// be past it: 16 sequences of 0.3k to 4k tokens at 28 / 4 heads of 128 take 21.7 us with 4 tokens
// each (28 columns) and 40.7 with 5 (35).
static int most_columns(int D) { return D <= 64 ? 64 : 32; }

bool takes_drafts(int head_dim, int g, int max_query_len) {
  return (head_dim == 32 || head_dim == 64 || head_dim == 128) && g <= 16 &&
         (int64_t)max_query_len * g <= most_columns(head_dim);
}

size_t drafts_workspace_bytes(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                              int block_size, int max_blocks, int max_query_len) {
  return decode_plan(num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks,
                     max_query_len).ws_bytes;
}

// (Blocks of 32 tokens take the general form: 16 x 5 drafts at 32 / 8 heads of 128 34.0 us where
// blocks of 16 take 30.9 and the prefill kernel 64.4, 64 x 4 at 14 / 2 heads of 64 23.8 for 20.2
// and 38.0.)
template <int D, int CB, int NW>
static hipError_t launch_drafts_nw(const DecodeFp8Args& a, unsigned grid, hipStream_t s) {
  if (a.bs == 16 && near_strides(a))
    attend_fp8_kernel<D, 1, 16, NW, CB, true><<<grid, 64 * NW, 0, s>>>(a);
  else
    attend_fp8_kernel<D, 1, 0, NW, CB, true><<<grid, 64 * NW, 0, s>>>(a);
  return hipGetLastError();
}

template <int D, int CB>
static hipError_t launch_drafts_cb(const DecodeFp8Args& a, const DecodePlan& p, hipStream_t s) {
  const unsigned grid = (unsigned)p.grid;
  return p.waves == 8 ? launch_drafts_nw<D, CB, 8>(a, grid, s)
                      : launch_drafts_nw<D, CB, 4>(a, grid, s);
}

static hipError_t launch_drafts(const DecodeFp8Args& a, int D, const DecodePlan& p, hipStream_t s) {
  const bool two = a.max_new * a.g <= 32;
  switch (D) {
    case 32: return two ? launch_drafts_cb<32, 2>(a, p, s) : launch_drafts_cb<32, 4>(a, p, s);
    case 64: return two ? launch_drafts_cb<64, 2>(a, p, s) : launch_drafts_cb<64, 4>(a, p, s);
    case 128: return launch_drafts_cb<128, 2>(a, p, s);
    default: return hipErrorInvalidValue;
  }
}

int prefill_drafts(const PrefillAttnArgs& p, int D, int max_query_len, void* workspace,
                   size_t workspace_bytes, hipStream_t s) {
  if ((int64_t)p.max_blocks * p.bs > 0x7fffffff - 4096) {
    set_error("tables of 2^31 tokens are not built");
    return PA_ERR_UNSUPPORTED;
  }
  const DecodePlan plan =
      decode_plan(p.num_seqs, p.hkv * p.g, p.hkv, D, p.bs, p.max_blocks, max_query_len);
  if (plan.grid < 0) {
    set_error("%d sequences of %d kv heads exceed one launch", p.num_seqs, p.hkv);
    return PA_ERR_UNSUPPORTED;
  }
  if (plan.ws_bytes && (!workspace || workspace_bytes < plan.ws_bytes)) {
    set_error("workspace of %zu bytes needed, %zu given", plan.ws_bytes, workspace_bytes);
    return PA_ERR_WORKSPACE;
  }
  DecodeFp8Args a{};
  a.q = p.q;
  a.q_sb = p.q_st;
  a.q_sh = p.q_sh;
  a.k = reinterpret_cast<const uint8_t*>(p.k);
  a.k_sb = p.k_sb;
  a.k_st = p.k_st;
  a.k_sh = p.k_sh;
  a.v = reinterpret_cast<const uint8_t*>(p.v);
  a.v_sb = p.v_sb;
  a.v_st = p.v_st;
  a.v_sh = p.v_sh;
  a.ks = p.ks;
  a.ks_sb = p.ks_sb;
  a.ks_sh = p.ks_sh;
  a.vs = p.vs;
  a.vs_sb = p.vs_sb;
  a.vs_sh = p.vs_sh;
  a.bt = p.bt;
  a.bt_sb = p.bt_sb;
  a.bt_sk = p.bt_sk;
  a.lens = p.lens;
  a.out = p.out;
  a.o_sb = p.o_st;
  a.o_sh = p.o_sh;
  a.num_seqs = p.num_seqs;
  a.hkv = p.hkv;
  a.g = p.g;
  a.bs = p.bs;
  a.num_blocks = p.num_blocks;
  a.max_blocks = p.max_blocks;
  a.qstart = p.qstart;
  a.num_tokens = p.num_tokens;
  a.max_new = max_query_len;
  a.scale_log2 = p.scale_log2;
  plan.fill(a, workspace);
  const hipError_t e = launch_drafts(a, D, plan, s);
  if (e == hipSuccess) return PA_OK;
  set_error("HIP launch failed: %s", hipGetErrorString(e));
  return PA_ERR_HIP;
}

}  // namespace fp8
}  // namespace pa
