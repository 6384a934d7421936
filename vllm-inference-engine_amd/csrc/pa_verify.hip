// Verification of drafted tokens against the target's probabilities (gfx950).
//
// Sequence b drafted ids x_0 .. x_{k-1} from distributions q_0 .. q_{k-1}; p_0 ..
// p_k are the target's. With n the number of leading i with u_i q_i(x_i) < p_i(x_i)
// -- draft i survives with probability min(1, p/q) -- the next token is drawn from
//   w = max(p_n - q_n, 0)   after a rejection (n < k),
//   w = p_n                 when all drafts survived, or when the difference is 0
//                           everywhere,
// by the inverse of its cumulative sums at u': the first index whose sum exceeds
// u' * (sum of all). The tokens so made follow the target's distribution.
//
// All sums and products are in 64 bits: the products of two fp32 numbers are then
// exact, and sums in any order agree to 2^-40 or better, so the chosen index does
// not depend on how the row is split.
//
// A row of the vocabulary is split over workgroups of kChunk entries. Each finds n
// for itself (the drafts' entries are a few loads), sums its chunk of w and of p, and
// leaves the sums in the workspace; the last of a sequence's workgroups finds the
// chunk in which the cumulative sum crosses u' * total and looks for the index there.
// Bound by memory: two fp32 rows per sequence, read once (and one chunk twice).
#include "../../include/paged_attention.h"
#include "pa_common.h"

namespace pa {
namespace verify {

constexpr int kThreads = 256;
constexpr int kPer = 16;  // entries per thread in a chunk
constexpr int kChunk = kThreads * kPer;
constexpr int kMaxDrafts = 64;  // one per lane of a wavefront
// The workspace starts with one arrival counter per sequence, at the same place for
// every call.
constexpr int kMaxSeqs = 16384;
constexpr size_t kCounterBytes = (size_t)kMaxSeqs * sizeof(int);

struct Args {
  const float* p;
  int64_t p_sb, p_si;
  const float* q;  // null: the drafts were certain, q_i(x_i) = 1
  int64_t q_sb, q_si;
  const int64_t* ids;
  int64_t i_sb, i_si;
  const float* u;
  int64_t u_sb, u_si;
  const float* u_next;
  const int32_t* counts;  // drafts of each sequence, or null: k
  int64_t* tokens;        // [seqs, k + 1]
  int32_t* accepted;
  int* cnt;
  double* sums;  // [seqs][chunks][2]: max(p - q, 0), p
  int seqs, k, vocab, chunks;
};

struct Weights {
  const float* p;
  const float* q;      // null: nothing is taken off
  int64_t certain;     // with q null: the index whose weight is 0, or -1
};

// Weight of entry v. Negative numbers and NaN count as 0.
__device__ inline double weight(float p, float q) {
  const double d = (double)p - (double)q;
  return d > 0.0 ? d : 0.0;
}

__device__ inline double wave_sum(double x) {
#pragma unroll
  for (int off = 32; off; off >>= 1) x += __shfl_xor(x, off);
  return x;
}

// One thread's entries [v0, v0 + 4) of the chunk: p and q, zeros past the vocabulary.
template <bool VEC>
__device__ inline void load4(const Args& a, const Weights& w, int64_t v0, float (&p)[4],
                             float (&q)[4]) {
  if (VEC && v0 + 4 <= a.vocab) {
    const float4 x = *reinterpret_cast<const float4*>(w.p + v0);
    p[0] = x.x, p[1] = x.y, p[2] = x.z, p[3] = x.w;
    if (w.q) {
      const float4 y = *reinterpret_cast<const float4*>(w.q + v0);
      q[0] = y.x, q[1] = y.y, q[2] = y.z, q[3] = y.w;
    } else {
      q[0] = q[1] = q[2] = q[3] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = v0 + i < a.vocab;
      p[i] = in ? w.p[v0 + i] : 0.f;
      q[i] = in && w.q ? w.q[v0 + i] : 0.f;
    }
  }
  if (!w.q) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (v0 + i == w.certain) q[i] = __builtin_huge_valf();
  }
}

template <bool VEC>
__global__ __launch_bounds__(kThreads) void verify_kernel(Args a) {
  __shared__ double s_sum[2][kThreads / 64];
  __shared__ double s_before[kThreads / 64];
  __shared__ int s_flag;
  __shared__ int s_best, s_last;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x / a.chunks;
  const int chunk = blockIdx.x - b * a.chunks;

  // Every wavefront decides the drafts for itself, one per lane.
  int k = a.counts ? a.counts[b] : a.k;
  k = k < 0 ? 0 : (k > a.k ? a.k : k);
  bool ok = false;
  int64_t id = -1;
  if (lane < k) {
    id = a.ids[b * a.i_sb + lane * a.i_si];
    if (id >= 0 && id < a.vocab) {
      const float p = a.p[b * a.p_sb + lane * a.p_si + id];
      const float q = a.q ? a.q[b * a.q_sb + lane * a.q_si + id] : 1.f;
      ok = (double)a.u[b * a.u_sb + lane * a.u_si] * (double)q < (double)p;
    }
  }
  const uint64_t rejected = ~__ballot(ok);  // lanes from k on among them
  const int n = k < 64 || rejected ? min(k, (int)__builtin_ctzll(rejected)) : k;
  Weights w;
  w.p = a.p + b * a.p_sb + n * a.p_si;
  w.q = n < k && a.q ? a.q + b * a.q_sb + n * a.q_si : nullptr;
  w.certain = n < k && !a.q ? __shfl(id, n) : -1;

  const int64_t c0 = (int64_t)chunk * kChunk;
  double sd = 0.0, sp = 0.0;
#pragma unroll
  for (int j = 0; j < kPer / 4; ++j) {
    float p[4], q[4];
    load4<VEC>(a, w, c0 + ((int64_t)j * kThreads + tid) * 4, p, q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sd += weight(p[i], q[i]);
      sp += weight(p[i], 0.f);
    }
  }
  sd = wave_sum(sd);
  sp = wave_sum(sp);
  if (lane == 0) {
    s_sum[0][wave] = sd;
    s_sum[1][wave] = sp;
  }
  __syncthreads();
  double* sums = a.sums + (int64_t)b * a.chunks * 2;
  if (tid == 0) {
    double x = 0.0, y = 0.0;
    for (int i = 0; i < kThreads / 64; ++i) {
      x += s_sum[0][i];
      y += s_sum[1][i];
    }
    // Device-coherent: the sequence's last workgroup may run on another XCD.
    __hip_atomic_store(sums + 2 * chunk, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(sums + 2 * chunk + 1, y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);  // the sums have landed before the arrival counts
    s_flag = __hip_atomic_fetch_add(a.cnt + b, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
             a.chunks - 1;
  }
  __syncthreads();
  if (!s_flag) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");

  // The chunk of the crossing, by every wavefront: lanes take chunks lane, lane + 64, ...
  auto chunk_sum = [&](int c, int which) {
    return c < a.chunks ? __hip_atomic_load(sums + 2 * c + which, __ATOMIC_RELAXED,
                                            __HIP_MEMORY_SCOPE_AGENT)
                        : 0.0;
  };
  double total = 0.0;
  for (int c = lane; c < a.chunks; c += 64) total += chunk_sum(c, 0);
  total = wave_sum(total);
  const bool whole = !(total > 0.0);  // p <= q everywhere: the target's own row
  if (whole) {
    w.q = nullptr;
    w.certain = -1;
    total = 0.0;
    for (int c = lane; c < a.chunks; c += 64) total += chunk_sum(c, 1);
    total = wave_sum(total);
  }
  const double aim = (double)a.u_next[b] * total;
  // First chunk whose inclusive sum exceeds aim, and the last with any weight.
  int at = -1, last = 0;
  double before = 0.0, last_before = 0.0, run = 0.0;
  for (int c = 0; c < a.chunks && at < 0; c += 64) {
    const double x = chunk_sum(c + lane, whole);
    double incl = x;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const double y = __shfl_up(incl, off);
      if (lane >= off) incl += y;
    }
    incl += run;
    const uint64_t over = __ballot(x > 0.0 && incl > aim);
    const uint64_t some = __ballot(x > 0.0);
    if (over) {
      const int l = (int)__builtin_ctzll(over);
      at = c + l;
      before = __shfl(incl - x, l);
    }
    if (some) {
      const int l = 63 - (int)__builtin_clzll(some);
      last = c + l;
      last_before = __shfl(incl - x, l);
    }
    run = __shfl(incl, 63);
  }
  if (at < 0) {  // u' * total not below the sum of all, by rounding or u' >= 1
    at = last;
    before = last_before;
  }

  // The index within the chunk: thread t now holds kPer consecutive entries.
  if (tid == 0) {
    s_best = 0x7fffffff;
    s_last = -1;
  }
  const int64_t v0 = (int64_t)at * kChunk + (int64_t)tid * kPer;
  double x[kPer], mine = 0.0;
  int mine_last = -1;
#pragma unroll
  for (int j = 0; j < kPer / 4; ++j) {
    float p[4], q[4];
    load4<VEC>(a, w, v0 + 4 * j, p, q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[4 * j + i] = weight(p[i], q[i]);
      mine += x[4 * j + i];
      if (x[4 * j + i] > 0.0) mine_last = 4 * j + i;
    }
  }
  double incl = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double y = __shfl_up(incl, off);
    if (lane >= off) incl += y;
  }
  if (lane == 63) s_before[wave] = incl;
  __syncthreads();
  double sum = before + (incl - mine);
  for (int i = 0; i < wave; ++i) sum += s_before[i];
  int found = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    sum += x[i];
    if (x[i] > 0.0 && sum > aim && found == 0x7fffffff) found = tid * kPer + i;
  }
  if (found != 0x7fffffff) atomicMin(&s_best, found);
  if (mine_last >= 0) atomicMax(&s_last, tid * kPer + mine_last);
  __syncthreads();
  int64_t* out = a.tokens + (int64_t)b * (a.k + 1);
  if (tid <= a.k) {
    // With no weight anywhere: index 0.
    const int64_t next = s_best != 0x7fffffff ? (int64_t)at * kChunk + s_best
                                              : (s_last >= 0 ? (int64_t)at * kChunk + s_last : 0);
    out[tid] = tid < n ? a.ids[b * a.i_sb + tid * a.i_si] : (tid == n ? next : -1);
  }
  if (tid == 0) {
    a.accepted[b] = n;
    __hip_atomic_store(a.cnt + b, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

static int chunks_of(int vocab) { return (int)(((int64_t)vocab + kChunk - 1) / kChunk); }

}  // namespace verify
}  // namespace pa

using namespace pa;
using namespace pa::verify;

extern "C" {

size_t pa_verify_drafts_workspace_bytes(int num_seqs, int vocab) {
  if (num_seqs <= 0 || num_seqs > kMaxSeqs || vocab <= 0) return 0;
  return kCounterBytes + (size_t)num_seqs * chunks_of(vocab) * 2 * sizeof(double);
}

int pa_verify_drafts_f32(const float* target, const int64_t target_strides[3], const float* draft,
                         const int64_t draft_strides[3], const int64_t* draft_ids,
                         const int64_t id_strides[2], const float* accept_u,
                         const int64_t u_strides[2], const float* next_u,
                         const int32_t* num_drafts, int64_t* tokens, int32_t* accepted,
                         int num_seqs, int max_drafts, int vocab, void* workspace,
                         size_t workspace_bytes, void* stream) {
  clear_error();
  if (num_seqs < 0 || max_drafts < 0 || vocab <= 0) {
    set_error("num_seqs (%d) and max_drafts (%d) must be >= 0, vocab (%d) positive", num_seqs,
              max_drafts, vocab);
    return PA_ERR_ARG;
  }
  if (num_seqs == 0) return PA_OK;
  if (num_seqs > kMaxSeqs || max_drafts > kMaxDrafts) {
    set_error("at most %d sequences of %d drafts, %d of %d given", kMaxSeqs, kMaxDrafts, num_seqs,
              max_drafts);
    return PA_ERR_UNSUPPORTED;
  }
  if (!target || !target_strides || !next_u || !tokens || !accepted ||
      (max_drafts > 0 && (!draft_ids || !id_strides || !accept_u || !u_strides)) ||
      (draft && !draft_strides)) {
    set_error("null pointer argument");
    return PA_ERR_ARG;
  }
  if (target_strides[2] != 1 || (draft && draft_strides[2] != 1)) {
    set_error("the rows of probabilities need unit vocabulary stride");
    return PA_ERR_ARG;
  }
  const size_t need = pa_verify_drafts_workspace_bytes(num_seqs, vocab);
  if (!workspace || workspace_bytes < need) {
    set_error("workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    return PA_ERR_WORKSPACE;
  }
  const int chunks = chunks_of(vocab);
  const int64_t grid = (int64_t)num_seqs * chunks;
  if (grid > 0x7fffffff) {
    set_error("%d sequences of a vocabulary of %d exceed one launch", num_seqs, vocab);
    return PA_ERR_UNSUPPORTED;
  }
  auto by4 = [](const float* p, const int64_t* st) {
    return (uintptr_t)p % 16 == 0 && st[0] % 4 == 0 && st[1] % 4 == 0;
  };
  Args a{};
  a.p = target;
  a.p_sb = target_strides[0];
  a.p_si = target_strides[1];
  bool vec = by4(target, target_strides);
  if (draft && max_drafts > 0) {
    a.q = draft;
    a.q_sb = draft_strides[0];
    a.q_si = draft_strides[1];
    vec = vec && by4(draft, draft_strides);
  }
  if (max_drafts > 0) {
    a.ids = draft_ids;
    a.i_sb = id_strides[0];
    a.i_si = id_strides[1];
    a.u = accept_u;
    a.u_sb = u_strides[0];
    a.u_si = u_strides[1];
  }
  a.u_next = next_u;
  a.counts = num_drafts;
  a.tokens = tokens;
  a.accepted = accepted;
  a.cnt = (int*)workspace;
  a.sums = (double*)((char*)workspace + kCounterBytes);
  a.seqs = num_seqs;
  a.k = max_drafts;
  a.vocab = vocab;
  a.chunks = chunks;
  if (vec)
    verify_kernel<true><<<(unsigned)grid, kThreads, 0, (hipStream_t)stream>>>(a);
  else
    verify_kernel<false><<<(unsigned)grid, kThreads, 0, (hipStream_t)stream>>>(a);
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return PA_OK;
  set_error("HIP launch failed: %s", hipGetErrorString(e));
  return PA_ERR_HIP;
}

}  // extern "C"
