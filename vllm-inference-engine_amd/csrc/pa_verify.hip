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
// exact, and sums in any order agree to 2^-40 of the whole or better. The chosen index is
// that of the definition except where u' * (sum of all) lies that near to a cumulative
// sum: there the neighbour with a weight may be taken.
//
// A row of the vocabulary is cut into pieces of 1024 entries, one wavefront's work at a
// time: the sums of w and of p over each piece go to the workspace. The wavefronts of a few
// workgroups per sequence take the pieces in turn (each decides n for itself: the drafts'
// entries are a few loads), two pieces in flight; the last of the sequence's workgroups
// finds the piece in which the cumulative sum crosses u' * total and looks for the index
// there. Bound by memory: two fp32 rows per sequence, read once (and one piece twice), and
// for a few sequences by the chain drafts -> their entries -> pieces -> arrival -> sums ->
// piece. On MI355X with 4 drafts and a vocabulary of 151936: 64 sequences (78 MB) 16.7 us, 4.7
// TB/s; one 6.1 us.
#include "../../include/paged_attention.h"
#include "pa_tiles.h"

namespace pa {
namespace verify {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kPiece = 1024;  // entries; 16 per lane
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
  double* sums;  // [seqs][pieces][2]: max(p - q, 0), p
  int k, vocab, pieces;
  int groups;  // workgroups per sequence
};

struct Weights {
  const float* p;
  const float* q;      // null: nothing is taken off
  int certain;     // with q null: the index whose weight is 0, or -1
};

// Weight of entry v. Negative numbers and NaN count as 0.
__device__ inline double weight(float p, float q) {
  const double d = (double)p - (double)q;
  return d > 0.0 ? d : 0.0;
}

// x of another lane of the row of 16 (a data-parallel-primitive control word), 0 where there
// is none.
template <int CTRL>
__device__ inline double row_lane(double x) {
  const uint2 v = __builtin_bit_cast(uint2, x);
  return __builtin_bit_cast(
      double, make_uint2((unsigned)__builtin_amdgcn_update_dpp(0, (int)v.x, CTRL, 0xf, 0xf, false),
                         (unsigned)__builtin_amdgcn_update_dpp(0, (int)v.y, CTRL, 0xf, 0xf, false)));
}

// Lane l's x, l uniform.
__device__ inline double lane_of(double x, int l) {
  const uint2 v = __builtin_bit_cast(uint2, x);
  return __builtin_bit_cast(double, make_uint2((unsigned)__builtin_amdgcn_readlane((int)v.x, l),
                                               (unsigned)__builtin_amdgcn_readlane((int)v.y, l)));
}

// Sum over a wavefront, in every lane: rotations within rows of 16, then the rows.
__device__ inline double wave_sum(double x) {
  x += row_lane<0x128>(x);
  x += row_lane<0x124>(x);
  x += row_lane<0x122>(x);
  x += row_lane<0x121>(x);
  return (lane_of(x, 0) + lane_of(x, 16)) + (lane_of(x, 32) + lane_of(x, 48));
}

// Sums over the lanes up to each: shifts within rows of 16, then the rows before.
__device__ inline double wave_scan(double x, int lane) {
  x += row_lane<0x111>(x);
  x += row_lane<0x112>(x);
  x += row_lane<0x114>(x);
  x += row_lane<0x118>(x);
  const double r0 = lane_of(x, 15), r1 = lane_of(x, 31), r2 = lane_of(x, 47);
  const double before = lane < 16 ? 0.0 : lane < 32 ? r0 : lane < 48 ? r0 + r1 : (r0 + r1) + r2;
  return before + x;
}

// One lane's entries [v0, v0 + 4) of a row: p and q, zeros past the vocabulary. WHOLE: there
// are four, at 16-byte aligned addresses.
template <bool WHOLE>
__device__ inline void load4(const Args& a, const Weights& w, int v0, float (&p)[4],
                             float (&q)[4]) {
  if constexpr (WHOLE) {
    const float4 x = *reinterpret_cast<const float4*>(w.p + v0);
    p[0] = x.x, p[1] = x.y, p[2] = x.z, p[3] = x.w;
    float4 y = {0.f, 0.f, 0.f, 0.f};
    if (w.q) y = *reinterpret_cast<const float4*>(w.q + v0);
    q[0] = y.x, q[1] = y.y, q[2] = y.z, q[3] = y.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = v0 < a.vocab - i;
      p[i] = in ? w.p[v0 + i] : 0.f;
      q[i] = in && w.q ? w.q[v0 + i] : 0.f;
    }
  }
  if (w.certain >= 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (v0 + i == w.certain) q[i] = __builtin_huge_valf();
  }
}

template <bool VEC>
__global__ __launch_bounds__(kThreads, 4) void verify_kernel(Args a) {
  __shared__ double s_sum[kWaves];
  __shared__ int s_flag, s_found[kWaves], s_some[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x / a.groups;
  const int group = blockIdx.x - b * a.groups;

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
  // (An id outside the vocabulary is no entry's.)
  const int own = id >= 0 && id < a.vocab ? (int)id : -1;
  w.certain = n < k && !a.q ? __builtin_amdgcn_readfirstlane(__shfl(own, n)) : -1;

  double* sums = a.sums + (int64_t)b * a.pieces * 2;
  // One piece: 16 entries per lane, four at a time.
  auto load_piece = [&](int c, float (&p)[4][4], float (&q)[4][4]) {
    const int v0 = c * kPiece + lane * 4;
    if (VEC && c < a.vocab / kPiece) {  // wavefront-uniform
#pragma unroll
      for (int j = 0; j < 4; ++j) load4<true>(a, w, v0 + j * 256, p[j], q[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) load4<false>(a, w, v0 + j * 256, p[j], q[j]);
    }
  };
  auto sum_piece = [&](int c, const float (&p)[4][4], const float (&q)[4][4]) {
    double sd = 0.0, sp = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sd += weight(p[j][i], q[j][i]);
        sp += weight(p[j][i], 0.f);
      }
    sd = wave_sum(sd);
    sp = wave_sum(sp);
    if (lane == 0) {
      // Device-coherent: the sequence's last workgroup may run on another XCD.
      __hip_atomic_store(sums + 2 * c, sd, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(sums + 2 * c + 1, sp, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  };
  const int stride = a.groups * kWaves;
  float p0[4][4], q0[4][4], p1[4][4], q1[4][4];
  int c = group * kWaves + wave;
  if (c < a.pieces) load_piece(c, p0, q0);
  while (c < a.pieces) {  // wavefront-uniform
    if (c + stride < a.pieces) load_piece(c + stride, p1, q1);
    sum_piece(c, p0, q0);
    c += stride;
    if (c >= a.pieces) break;
    if (c + stride < a.pieces) load_piece(c + stride, p0, q0);
    sum_piece(c, p1, q1);
    c += stride;
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_s_waitcnt(0);  // the sums have landed before the arrival counts
  __syncthreads();
  if (tid == 0)
    s_flag = __hip_atomic_fetch_add(a.cnt + b, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
             a.groups - 1;
  __syncthreads();
  if (!s_flag) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");

  // The piece of the crossing, by every wavefront for itself: batches of 256 pieces, four
  // consecutive ones per lane, both sums of each in one device-coherent read.
  const auto rs = tiles::tile_rsrc(sums, a.pieces * 16);
  double x[2][4];  // [whether of p alone][piece]
  auto take = [&](int first) {  // past the last piece: zeros
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 y = tiles::load_coherent16(rs, (first + lane * 4 + i) * 16);
      typedef double f64x2 __attribute__((ext_vector_type(2)));
      const f64x2 z = __builtin_bit_cast(f64x2, y);
      x[0][i] = z[0];
      x[1][i] = z[1];
    }
  };
  double of_diff = 0.0, of_p = 0.0;
  for (int first = 0; first < a.pieces; first += 256) {
    take(first);
    of_diff += wave_sum((x[0][0] + x[0][1]) + (x[0][2] + x[0][3]));
    of_p += wave_sum((x[1][0] + x[1][1]) + (x[1][2] + x[1][3]));
  }
  const bool whole = !(of_diff > 0.0);  // p <= q everywhere: the target's own row
  if (whole) {
    w.q = nullptr;
    w.certain = -1;
  }
  const double aim = (double)a.u_next[b] * (whole ? of_p : of_diff);
  // First piece whose inclusive sum exceeds aim, and the last with any weight.
  int at = -1, last = 0;
  double before = 0.0, last_before = 0.0, run = 0.0;
  for (int first = 0; first < a.pieces && at < 0; first += 256) {
    if (a.pieces > 256) take(first);
    double own4[4], mine = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      own4[i] = whole ? x[1][i] : x[0][i];
      mine += own4[i];
    }
    const double incl = wave_scan(mine, lane);
    double sum = run + (incl - mine);
    int over = -1, some = -1;
    double over_before = 0.0, some_before = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (own4[i] > 0.0) {
        if (over < 0 && sum + own4[i] > aim) {
          over = i;
          over_before = sum;
        }
        some = i;
        some_before = sum;
      }
      sum += own4[i];
    }
    const uint64_t overs = __ballot(over >= 0), somes = __ballot(some >= 0);
    if (overs) {
      const int l = (int)__builtin_ctzll(overs);
      at = first + 4 * l + __builtin_amdgcn_readlane(over, l);
      before = lane_of(over_before, l);
    }
    if (somes) {
      const int l = 63 - (int)__builtin_clzll(somes);
      last = first + 4 * l + __builtin_amdgcn_readlane(some, l);
      last_before = lane_of(some_before, l);
    }
    run += lane_of(incl, 63);
  }
  if (at < 0) {  // u' * total not below the sum of all, by rounding or u' >= 1
    at = last;
    before = last_before;
  }

  // The index within the piece: thread t now holds four consecutive entries.
  constexpr int kPer = kPiece / kThreads;
  static_assert(kPer == 4, "one load4 per thread");
  float ep[4], eq[4];
  if (VEC && at < a.vocab / kPiece)
    load4<true>(a, w, at * kPiece + tid * kPer, ep, eq);
  else
    load4<false>(a, w, at * kPiece + tid * kPer, ep, eq);
  double e[kPer], mine = 0.0;
  int some = -1;  // the thread's last entry with any weight
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    e[i] = weight(ep[i], eq[i]);
    mine += e[i];
    if (e[i] > 0.0) some = i;
  }
  const double incl = wave_scan(mine, lane);
  if (lane == 63) s_sum[wave] = incl;
  __syncthreads();
  double sum = before + (incl - mine);
  for (int i = 0; i < wave; ++i) sum += s_sum[i];
  int found = -1;  // and the first whose sum exceeds aim
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    sum += e[i];
    if (e[i] > 0.0 && sum > aim && found < 0) found = i;
  }
  // Per wavefront the first of the ones and the last of the others, or -1.
  const uint64_t founds = __ballot(found >= 0), somes = __ballot(some >= 0);
  const int fl = founds ? (int)__builtin_ctzll(founds) : 0;
  const int sl = somes ? 63 - (int)__builtin_clzll(somes) : 0;
  const int fi = __builtin_amdgcn_readlane(found, fl), si = __builtin_amdgcn_readlane(some, sl);
  if (lane == 0) {
    s_found[wave] = founds ? (wave * 64 + fl) * kPer + fi : -1;
    s_some[wave] = somes ? (wave * 64 + sl) * kPer + si : -1;
  }
  __syncthreads();
  int64_t* out = a.tokens + (int64_t)b * (a.k + 1);
  if (tid <= a.k) {
    int best = -1, spare = -1;
#pragma unroll
    for (int i = kWaves - 1; i >= 0; --i) {
      best = s_found[i] >= 0 ? s_found[i] : best;
      spare = spare >= 0 ? spare : s_some[i];
    }
    if (best < 0) best = spare;
    // With no weight anywhere: index 0. (Lane i of the first wavefront holds id i.)
    const int64_t next = best >= 0 ? (int64_t)at * kPiece + best : 0;
    out[tid] = tid < n ? id : (tid == n ? next : -1);
  }
  if (tid == 0) {
    a.accepted[b] = n;
    __hip_atomic_store(a.cnt + b, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

static int pieces_of(int vocab) { return (int)(((int64_t)vocab + kPiece - 1) / kPiece); }

// Workgroups per sequence: one wavefront per piece for a few sequences; for many, as many
// as fill kWavesPerCu wavefronts per compute unit over all sequences, the pieces dealt in
// whole rounds. (64 sequences at 4 / 8 / 12 / 16 on MI355X: 18.0 / 17.0 / 18.0 / 18.6 us.)
constexpr int kWavesPerCu = 8;
static int groups_of(int num_seqs, int pieces) {
  const int64_t waves = (int64_t)kWavesPerCu * device_cus() / num_seqs;
  const int64_t rounds = waves >= pieces ? 1 : (pieces + (waves > 0 ? waves : 1) - 1) / (waves > 0 ? waves : 1);
  const int64_t per_round = (pieces + rounds - 1) / rounds;
  return (int)((per_round + kWaves - 1) / kWaves);
}

}  // namespace verify
}  // namespace pa

using namespace pa;
using namespace pa::verify;

extern "C" {

size_t pa_verify_drafts_workspace_bytes(int num_seqs, int vocab) {
  if (num_seqs <= 0 || num_seqs > kMaxSeqs || vocab <= 0) return 0;
  return kCounterBytes + (size_t)num_seqs * pieces_of(vocab) * 2 * sizeof(double);
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
  if (vocab > (1 << 30)) {
    set_error("a vocabulary of %d is not built", vocab);
    return PA_ERR_UNSUPPORTED;
  }
  const size_t need = pa_verify_drafts_workspace_bytes(num_seqs, vocab);
  if (!workspace || workspace_bytes < need) {
    set_error("workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    return PA_ERR_WORKSPACE;
  }
  const int pieces = pieces_of(vocab);
  const int groups = groups_of(num_seqs, pieces);
  const int64_t grid = (int64_t)num_seqs * groups;
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
  a.k = max_drafts;
  a.vocab = vocab;
  a.pieces = pieces;
  a.groups = groups;
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
