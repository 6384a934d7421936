// Decode attention with capped, biased and windowed scores over the paged fp16 pool (gfx950).
//
//   s_j = softcap * tanh(scale q.k_j / softcap) - slope_h (p - j),  p = L - 1,
//   o = sum_j 2^(log2(e) s_j - m) v_j / sum_j 2^(log2(e) s_j - m),
//   over the keys j of [max(first, L - window), L)
//
// Work split, as for the 8-bit pool (pa_fp8_attend.h): the work is a list of (sequence, kv
// head) pairs, each of the 32-token chunks that its window touches plus a fixed cost; a grid
// of one workgroup per compute unit takes equal contiguous ranges of it, found by every
// wavefront for itself with lane scans over lengths and first keys. Where every pair is
// short a workgroup takes one pair whole. Within a pair's part of its range the wavefronts
// take the chunks in turn, each with an online softmax of its own for the whole query group,
// and meet in LDS; a pair cut by range boundaries leaves fp32 records, which the last of its
// workgroups combines in list order (the same bits on every run).
//
// Per chunk. K and V rows go from memory straight into LDS (buffer_load ... lds), the 16-byte
// pieces of a row permuted by its number so that neither K's operand reads nor V's transposing
// ones meet a bank twice. All fragments are in registers before the next chunk's loads are
// issued into the same LDS, and the arithmetic runs under those loads. Scores go to the exp2
// domain with cap (tanh as 1 - 2 / (1 + e^2x), and for caps above 128 a polynomial where that
// would cancel: see ScoreForm) and bias right after the products; that costs a few instructions
// per key and query head where memory costs hundreds of cycles per chunk.
// Keys outside the interval get no weight, and their V rows are cleared: what lies in freed
// blocks before the window never reaches a result.
//
// Probabilities are rounded to fp16 (the denominators sum the rounded ones), scaled by 2^14 so
// that they keep 11 bits down to 2^-28 of the largest: half a step, 2^-11 relative, as the
// output's own rounding.
//
// Bound by memory. In a run of calls on MI355X: 32 capped contexts of 256 to 8192 tokens at 28 / 4
// heads of 128 49.1 us (241 MB, 4.9 TB/s), 64 windows of 1024 with a bias at 16 / 16 heads of 64 52.2
// (258 MB, 4.9); one context of 300 tokens 5.1, a launch and its chain of dependent reads.
#include "../../include/paged_attention.h"
#include "pa_fp8_attend.h"

namespace pa {
namespace scored {

using namespace tiles;
using fp8::Cut;
using fp8::global_ptr;
using fp8::lds_ptr;
using fp8::load_to_lds;
using fp8::over_groups;
using fp8::over_row;
using fp8::pinned;
using fp8::record_size;
using fp8::swizzle;

constexpr int kChunk = 32;  // tokens a wavefront takes at a time
// The workspace starts with arrival counters at the same place for every call, one per
// pair of a call that is cut into ranges.
constexpr int kMaxCounters = 16384;
constexpr size_t kCounterBytes = (size_t)kMaxCounters * sizeof(int);
constexpr float kBias = 14.f;  // log2 of the factor on the probabilities

struct Args {
  const f16* q;
  int64_t q_sb, q_sh;
  const uint8_t* k;  // strides in bytes
  int64_t k_sb, k_st, k_sh;
  const uint8_t* v;
  int64_t v_sb, v_st, v_sh;
  const int32_t* bt;
  int64_t bt_sb, bt_sk;
  const int32_t* lens;
  const int32_t* starts;  // first key of each sequence, or null: 0
  const float* slopes;    // per query head, or null: no bias
  int64_t slope_s;
  f16* out;
  int64_t o_sb, o_sh;
  int* cnt;
  float* recs;
  int num_seqs, hkv, g, bs, num_blocks, max_blocks;
  int window;     // 0: none
  int ranged;     // 0: one workgroup per pair, no plan
  int min_range;  // list positions a range has at least
  int pair_cost;  // list positions a pair takes beside its chunks
  int rec_floats;
  float scale_log2, cap_log2, cap_out, cap_in, cap_t;  // see ScoreForm
};

template <int D, int BS, int NW>
__global__ __launch_bounds__(64 * NW, 2) void decode_scored_kernel(Args a) {
  constexpr int kThreads = 64 * NW;
  constexpr int RB = 2 * D;          // bytes of a row
  constexpr int NP = RB / 16;        // 16-byte pieces of it, one per lane
  constexpr int RPI = 64 / NP;       // rows per load instruction
  constexpr int NI = kChunk / RPI;   // load instructions per chunk, for K and for V
  constexpr bool UNIFORM = BS > 0;   // an instruction's rows lie in one block
  static_assert(BS % 16 == 0, "whole tiles per block, or any block size as 0");
  static_assert(RPI <= 16, "rows of one tile per instruction");
  constexpr int NC = D / 32;         // products per score tile
  constexpr int ND = D / 16;
  constexpr int D4 = D / 4;
  // Bytes per wavefront: K rows, then V rows; at the end its accumulators.
  constexpr int STAGE = 2 * kChunk * RB;
  static_assert(STAGE >= 16 * D * 4, "the accumulators fit");
  __shared__ __attribute__((aligned(16))) uint8_t s_stage[NW * STAGE];
  __shared__ __attribute__((aligned(16))) f32x4 s_part[kThreads];
  __shared__ float s_m[NW][16], s_l[NW][16];
  __shared__ int s_last;

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int row = lane & 15;
  const int grp = lane >> 4;
  const int bs = BS > 0 ? BS : a.bs;
  const int cap = a.max_blocks * bs;
  const int last_tile = (cap - 1) / 16;
  uint8_t* const stage = s_stage + wave * STAGE;
  // This lane's piece of a loaded row: row lrow of the instruction's. (The permutation is
  // linear in the bits of the row's number: instruction i's differs by swizzle(i * RPI).)
  const int lrow = lane / NP;
  const uint32_t lane_piece = (uint32_t)((lane % NP) ^ swizzle<NP>(lrow)) * 16;
  const uint32_t k_lrow = (uint32_t)(lrow * a.k_st), v_lrow = (uint32_t)(lrow * a.v_st);
  constexpr int kAll = 0x7fffffff;

  auto clamped = [&](int n) { return n < 0 ? 0 : (n > cap ? cap : n); };
  // First key of a sequence of n tokens (clamped); at most n.
  auto first_key = [&](int n, int start) {
    int f = start < 0 ? 0 : start;
    if (a.window > 0) f = max(f, n - a.window);
    return min(f, n);
  };
  auto chunks_of = [&](int n, int first) {
    return first < n ? (n + kChunk - 1) / kChunk - first / kChunk : 0;
  };

  // Chunks [c0, c1) of pair (b, h) of a sequence of L tokens, seen from key `from` on (not
  // ranged: all chunks, of a length found here). The pair is spread over nseg workgroups'
  // ranges, from range w0 on; this is its part `seg`.
  auto segment = [&](int b, int h, int L, int from, int c0, int c1, int w0, int seg, int nseg) {
    const int32_t* const btrow = pinned(a.bt + (int64_t)b * a.bt_sb);
    const int64_t bt_sk = pinned(a.bt_sk);
    const uint8_t* const kbase = pinned(a.k + h * a.k_sh);
    const uint8_t* const vbase = pinned(a.v + h * a.v_sh);
    const int64_t k_sb = pinned(a.k_sb), v_sb = pinned(a.v_sb);
    const int64_t k_st = pinned(a.k_st), v_st = pinned(a.v_st);
    const int last_id = pinned(a.num_blocks - 1);
    const int heads = a.g;
    if (!a.ranged) {
      L = clamped(load_uniform(a.lens + b));
      from = first_key(L, a.starts ? load_uniform(a.starts + b) : 0);
      c0 = from / kChunk;
      c1 = c0 + chunks_of(L, from);
    }
    // UNIFORM: the block ids of the chunk's two tiles; else those of the lane's row of each load.
    constexpr int NID = UNIFORM ? 2 : NI;
    int ids[NID];
    // Clamped to the table's width only: a tile past the end reads some block of the pool and
    // what it reads is masked.
    auto load_ids = [&](int c) {
#pragma unroll
      for (int i = 0; i < NID; ++i) {
        if constexpr (UNIFORM) {
          const int at = min(2 * c + i, last_tile);
          ids[i] = load_uniform(btrow + (int64_t)(at / (BS / 16)) * bt_sk);
        } else {
          ids[i] = btrow[(int64_t)(min(c * kChunk + i * RPI + lrow, cap - 1) / bs) * bt_sk];
        }
      }
    };
    const int first = c0 + wave;
    load_ids(first);
    // Q^T operands: column = query head `row` of the kv head's group.
    const int head = h * a.g + min(row, a.g - 1);
    f16x8 qf[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c)
      qf[c] = *reinterpret_cast<const f16x8*>(a.q + (int64_t)b * a.q_sb + (int64_t)head * a.q_sh +
                                              32 * c + grp * 8);
    const float slope = a.slopes ? a.slopes[head * a.slope_s] * kLog2e : 0.f;
    auto issue = [&](int c) {
      auto block = [&](int id) { return (int64_t)min(max(id, 0), last_id); };
      uint8_t* const to = s_stage + pinned(wave * STAGE);
      auto load_rows = [&](const uint8_t* base, int64_t sb, int64_t st, uint32_t row_off, uint8_t* to) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int64_t id = block(ids[UNIFORM ? i * RPI / 16 : i]);
          const uint32_t piece = lane_piece ^ (uint32_t)(swizzle<NP>(i * RPI) * 16);
          if constexpr (UNIFORM) {
            const int64_t off = (2 * c + i * RPI / 16) % (BS / 16) * 16 + i * RPI % 16;
            load_to_lds(tile_rsrc(base + id * sb + off * st, kAll), row_off + piece, to + i * 1024);
          } else {
            const int64_t off = (c * kChunk + i * RPI + lrow) % bs;
            load_to_lds(base + id * sb + off * st + piece, to + i * 1024);
          }
        }
      };
      load_rows(kbase, k_sb, k_st, k_lrow, to);
      load_rows(vbase, v_sb, v_st, v_lrow, to + kChunk * RB);
    };

    float m_run = kNegInf, l_run = 0.f;
    f32x4 acc[ND];
#pragma unroll
    for (int nd = 0; nd < ND; ++nd) acc[nd] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (first < c1) {
      issue(first);
      load_ids(first + NW);
    }
    for (int c = first; c < c1; c += NW) {
      const int t0 = c * kChunk;
      const bool whole = t0 >= from && t0 + kChunk <= L;  // wavefront-uniform
      // The chunk has landed; all of it into registers. Tile t's score row m is token
      // 8 (m / 4) + 4 t + m % 4: lane (., grp) then gets the scores of tokens 8 grp .. + 7,
      // those of its V fragments.
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
      wave_lds_fence();
      f16x8 kf[2][NC];
      f16x4 vf[ND][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int r = 8 * (row >> 2) + 4 * t + (row & 3);
#pragma unroll
        for (int c = 0; c < NC; ++c)
          kf[t][c] = *reinterpret_cast<const f16x8*>(stage + r * RB + ((c * 4 + grp) ^ swizzle<NP>(r)) * 16);
        // V^T: lanes 4 r + q of a group of 16 name halves [4 q, 4 q + 4) of four rows.
        const int rv = 8 * grp + 4 * t + (row >> 2);
        const uint8_t* vp = stage + kChunk * RB + rv * RB + (row & 1) * 8;
#pragma unroll
        for (int nd = 0; nd < ND; ++nd)
          vf[nd][t] = lds_read_tr16(reinterpret_cast<const f16*>(
              vp + ((nd * 2 + (row >> 1 & 1)) ^ swizzle<NP>(rv)) * 16));
      }
      wave_lds_fence();
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): nothing reads the LDS any more
      if (c + NW < c1) {
        issue(c + NW);
        load_ids(c + 2 * NW);
      }
      f32x4 s[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c)
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t][c], qf[c], s[t], 0, 0, 0);
      }
      const float away = (float)(t0 + 8 * grp - (L - 1));  // of the lane's first token
      if (a.cap_t != 0.f) {  // uniform
#pragma unroll
        for (int i = 0; i < 8; ++i)
          s[i / 4][i % 4] = wide_cap(s[i / 4][i % 4], a.scale_log2, a.cap_log2, a.cap_in, a.cap_t);
      } else if (a.cap_log2 != 0.f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float e = fast_exp2(s[i / 4][i % 4] * a.cap_in);
          s[i / 4][i % 4] = __builtin_fmaf(a.cap_out, __builtin_amdgcn_rcpf(e + 1.f), a.cap_log2);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i / 4][i % 4] *= a.scale_log2;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        s[i / 4][i % 4] = __builtin_fmaf(slope, away + (float)i, s[i / 4][i % 4]);
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = t0 + 8 * grp + i;
          const bool seen = key >= from && key < L;
          if (!seen) s[i / 4][i % 4] = kNegInf;
          // Rows that are not seen count as zeros: 0 * what lies there is never NaN.
#pragma unroll
          for (int nd = 0; nd < ND; ++nd)
            if (!seen) vf[nd][i / 4][i % 4] = (f16)0.f;
        }
      }
      float m = s[0][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) m = fmaxf(m, s[i / 4][i % 4]);
      const float m_new = fmaxf(m_run, over_groups(m, fp8::Max()));
      if (__ballot(m_new > m_run) != 0) {  // wavefront-uniform
        const float alpha = m_new == kNegInf ? 1.f : fast_exp2(m_run - m_new);
        l_run *= alpha;
#pragma unroll
        for (int nd = 0; nd < ND; ++nd) acc[nd] *= alpha;
        m_run = m_new;
      }
      // (First the maximum, then the factor: added to one another they round to some units of
      // large scores, and the probabilities to infinity.)
      const float m0 = m_run == kNegInf ? 0.f : m_run;
      f16x8 pb;
#pragma unroll
      for (int i = 0; i < 8; ++i) pb[i] = (f16)fast_exp2(s[i / 4][i % 4] - m0 + kBias);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        l_run = __builtin_amdgcn_fdot2(f16x2{pb[2 * i], pb[2 * i + 1]}, f16x2{(f16)1.f, (f16)1.f},
                                       l_run, false);
      // O^T += V^T P^T: operand index k = 8 grp + i stands for token 8 grp + i on both sides.
#pragma unroll
      for (int nd = 0; nd < ND; ++nd) {
        const f16x8 av = {vf[nd][0][0], vf[nd][0][1], vf[nd][0][2], vf[nd][0][3],
                          vf[nd][1][0], vf[nd][1][1], vf[nd][1][2], vf[nd][1][3]};
        acc[nd] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, pb, acc[nd], 0, 0, 0);
      }
    }

    // The wavefronts' states meet in LDS, four elements of accumulator row r at slot
    // (d / 4) ^ (r & 7). (Lane indices anew: see fresh_lane.)
    const int lane = fresh_lane();
    const int tid = wave * 64 + lane, row = lane & 15, grp = lane >> 4;
    // Part i of a cut pair lies in range w0 + i's slot 0 (the pair began before that range)
    // or, i = 0, in slot 1.
    const int64_t rec0 = (int64_t)(2 * w0 + 1) * a.rec_floats;
    auto record = [&](int i) { return (i ? 2 * i - 1 : 0) * a.rec_floats; };  // from rec0
    const auto rr = tile_rsrc(a.recs + rec0, (2 * nseg - 1) * a.rec_floats * 4);
    const int rb = record(seg) * 4;
    auto out_row = [&](int j) { return a.out + (int64_t)b * a.o_sb + (int64_t)(h * a.g + j) * a.o_sh; };
    float* my_acc = reinterpret_cast<float*>(stage);
    const float l_all = over_groups(l_run, fp8::Sum());
    if (grp == 0) {
      s_m[wave][row] = m_run;
      s_l[wave][row] = l_all;
    }
    if (row < heads) {
#pragma unroll
      for (int nd = 0; nd < ND; ++nd)
        *reinterpret_cast<f32x4*>(my_acc + row * D + ((nd * 4 + grp) ^ (row & 7)) * 4) = acc[nd];
    }
    __syncthreads();
    // (A state of no maximum holds zeros, or NaN that has to show.)
    auto share = [&](float m, float M) { return m == kNegInf ? 1.f : fast_exp2(m - M); };
#pragma unroll 1
    for (int i = tid; i < heads * D4; i += kThreads) {
      const int j = i / D4;
      const int d = (i - j * D4) * 4;
      float M = s_m[0][j];
#pragma unroll
      for (int w = 1; w < NW; ++w) M = fmaxf(M, s_m[w][j]);
      float l = 0.f;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = share(s_m[w][j], M);
        l += f * s_l[w][j];
        o += f * *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(s_stage + w * STAGE) +
                                                 j * D + ((d >> 2) ^ (j & 7)) * 4);
      }
      if (nseg == 1) {
        const float inv = l == 0.f ? 0.f : 1.f / l;  // 0: no key at all
        f16x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (f16)(o[e] * inv);
        *reinterpret_cast<f16x4*>(out_row(j) + d) = y;
      } else {
        store_coherent16(rr, rb + (j * D + d) * 4, o);
        if (d == 0) {
          __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, M), rr,
                                                rb + (heads * D + j) * 4, 0, 16);
          __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, l), rr,
                                                rb + (heads * D + heads + j) * 4, 0, 16);
        }
      }
    }
    if (nseg == 1) {
      __syncthreads();  // the next segment stages where this one's states lie
      return;
    }
    int* cnt = a.cnt + (int64_t)b * a.hkv + h;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);  // the record has landed before the arrival counts
    __syncthreads();
    if (tid == 0)
      s_last = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == nseg - 1;
    __syncthreads();
    if (!s_last) return;  // (the next segment writes s_last behind further barriers)
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");

    // Merge: the parts' maxima and denominators into LDS (batches of parts, as many as fit),
    // their maximum, sum and shares per head by 16 lanes each, and the accumulators by threads
    // (item: head and four of its elements; the parts of an item are dealt over as many threads
    // as there are for it), U parts a round trip. Part 0 lies apart from the others, which are
    // two records apart.
    float* s_max = s_m[0];  // (the wavefronts' states are spent)
    float* s_sum = s_l[0];
    const int batch = min(nseg, (int)(sizeof(s_stage) / 8) / heads);
    float* s_pm = reinterpret_cast<float*>(s_stage);
    float* s_pl = s_pm + heads * batch;
    const int items = heads * D4;
    const int parts = items < kThreads ? kThreads / items : 1;
    const int part = parts > 1 ? tid / items : 0;
    const int step = 2 * a.rec_floats * 4;  // bytes from part i to part i + 1, i > 0
    constexpr int U = 8;
    // Past the last part: zeros (by the lane's offset, whole).
    auto fetch = [&](int i, int j, int d, f32x4 (&y)[U]) {
      const int at = (record(i) + j * D + d) * 4;
#pragma unroll
      for (int u = 0; u < U; ++u) y[u] = load_coherent16(rr, at + u * parts * step);
    };
    // Maximum and denominator i of parts [s0, s1): of head i / (s1 - s0).
    auto load_ml = [&](int s0, int s1) {
#pragma unroll 1
      for (int i = tid; i < heads * (s1 - s0); i += kThreads) {
        const int j = i / (s1 - s0);
        const int p = i - j * (s1 - s0);
        const int at = (record(s0 + p) + heads * D + j) * 4;
        s_pm[j * batch + p] = load_coherent4(rr, at);
        s_pl[j * batch + p] = load_coherent4(rr, at + heads * 4);
      }
    };
#pragma unroll 1
    for (int base = 0; base < items; base += kThreads) {  // workgroup-uniform
      const int item = parts > 1 ? tid - part * items : base + tid;
      const bool live = part < parts && item < items;
      const int j = live ? item / D4 : 0;
      const int d = live ? (item - j * D4) * 4 : 0;
      const f32x4 y0 = load_coherent16(rr, (j * D + d) * 4);
      f32x4 y[U];
      fetch(1 + part, j, d, y);
      if (base == 0) {
#pragma unroll 1
        for (int s0 = 0; s0 < nseg; s0 += batch) {
          const int s1 = min(nseg, s0 + batch);
          if (s0) __syncthreads();
          load_ml(s0, s1);
          __syncthreads();
#pragma unroll 1
          for (int jj = tid / 16; jj < heads; jj += kThreads / 16) {
            const float had = s0 ? s_max[jj] : kNegInf;
            float M = had;
            for (int i = row; i < s1 - s0; i += 16) M = fmaxf(M, s_pm[jj * batch + i]);
            M = over_row(M, fp8::Max());
            float sum = 0.f;
            for (int i = row; i < s1 - s0; i += 16) {
              const float f = share(s_pm[jj * batch + i], M);
              sum += s_pl[jj * batch + i] * f;
              s_pm[jj * batch + i] = f;
            }
            sum = over_row(sum, fp8::Sum());
            if (s0) sum += s_sum[jj] * share(had, M);
            if (row == 0) {
              s_max[jj] = M;
              s_sum[jj] = sum;
            }
          }
        }
        __syncthreads();
      }
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int s0 = 0; s0 < nseg; s0 += batch) {
        const int s1 = min(nseg, s0 + batch);
        if (batch < nseg) {  // the batch's shares, of the maxima over all batches
          __syncthreads();
          load_ml(s0, s1);
          __syncthreads();
          for (int i = tid; i < heads * (s1 - s0); i += kThreads) {
            const int jj = i / (s1 - s0);
            float& x = s_pm[jj * batch + i - jj * (s1 - s0)];
            x = share(x, s_max[jj]);
          }
          __syncthreads();
        }
        if (!live) continue;
        const float* pm = s_pm + j * batch - s0;
        if (s0 == 0 && part == 0) o += pm[0] * y0;
#pragma unroll 1
        for (int i = s0 ? s0 + part : 1 + part; i < s1; i += U * parts) {
          if (i != 1 + part) fetch(i, j, d, y);
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (i + u * parts < s1) o += pm[i + u * parts] * y[u];
        }
      }
      if (parts > 1) {
        s_part[tid] = o;
        __syncthreads();
        if (part == 0)
          for (int p = 1; p < parts; ++p) o += s_part[tid + p * items];
      }
      if (live && part == 0) {
        const float sum = s_sum[j];
        const float inv = sum == 0.f ? 0.f : 1.f / sum;  // 0: no key at all
        f16x4 z;
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = (f16)(o[e] * inv);
        *reinterpret_cast<f16x4*>(out_row(j) + d) = z;
      }
    }
    if (tid == 0) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
  };

  if (!a.ranged) {
    const int pair = xcd_order(blockIdx.x, gridDim.x);
    const int b = pair / a.hkv;
    segment(b, pair - b * a.hkv, 0, 0, 0, 0, 0, 0, 1);
    return;
  }
  // This workgroup's part of the list: positions [x0, x1); `at` is the first of sequence b.
  // Each sequence takes hkv x (its chunks + pair_cost) positions. (The host sees to it that 31
  // bits hold their sum.) Lengths of 256 sequences a time, sequence base + 64 k + lane in
  // lens[k]: read together.
  constexpr int LK = 4;
  int lens[LK], firsts[LK], own[LK], incl[LK];
  auto take = [&](int base) {
#pragma unroll
    for (int k = 0; k < LK; ++k) {
      const int s = min(base + 64 * k + lane, a.num_seqs - 1);
      lens[k] = a.lens[s];
      firsts[k] = a.starts ? a.starts[s] : 0;
    }
#pragma unroll
    for (int k = 0; k < LK; ++k) {
      lens[k] = clamped(lens[k]);
      firsts[k] = first_key(lens[k], firsts[k]);
      own[k] = base + 64 * k + lane < a.num_seqs
                   ? a.hkv * (chunks_of(lens[k], firsts[k]) + a.pair_cost) : 0;
      incl[k] = wave_incl_scan(own[k]);
    }
  };
  int T = 0;
  for (int base = 0; base < a.num_seqs; base += 64 * LK) {
    take(base);
#pragma unroll
    for (int k = 0; k < LK; ++k) T += __builtin_amdgcn_readlane(incl[k], 63);
  }
  const int G = max(1, min((int)gridDim.x, T / a.min_range));
  if ((int)blockIdx.x >= G) return;
  const int w = xcd_order(blockIdx.x, G);
  const Cut ranges{T / G, T % G};
  const int x0 = ranges.start(w), x1 = ranges.start(w + 1);
  // The sequence that holds x0, and its first position.
  int at = 0, b = 0, h = 0;
  bool found = false;
  for (int base = 0; base < a.num_seqs && !found; base += 64 * LK) {
    if (a.num_seqs > 64 * LK) take(base);
#pragma unroll
    for (int k = 0; k < LK; ++k) {
      const int total = __builtin_amdgcn_readlane(incl[k], 63);
      if (!found && at + total > x0) {
        const int l = (int)__builtin_ctzll(__ballot(at + incl[k] > x0));
        b = base + 64 * k + l;
        at += __builtin_amdgcn_readlane(incl[k] - own[k], l);
        found = true;
      }
      if (!found) at += total;
    }
  }
  for (;;) {
    int L = 0, from = 0;
    if (a.num_seqs <= 64 * LK) {
#pragma unroll
      for (int k = 0; k < LK; ++k)
        if (b / 64 == k) {
          L = __builtin_amdgcn_readlane(lens[k], b % 64);
          from = __builtin_amdgcn_readlane(firsts[k], b % 64);
        }
    } else {
      L = clamped(load_uniform(a.lens + b));
      from = first_key(L, a.starts ? load_uniform(a.starts + b) : 0);
    }
    const int n = chunks_of(L, from);
    // The pair's positions: pair_cost of them, then its chunks.
    const int span = n + a.pair_cost;
    for (; h < a.hkv && at + span <= x0; ++h) at += span;
    if (h == a.hkv) {
      h = 0;
      if (++b == a.num_seqs) return;
      continue;
    }
    if (at >= x1) return;
    const int c0 = max(0, min(n, x0 - at - a.pair_cost));
    const int c1 = max(0, min(n, x1 - at - a.pair_cost));
    // The ranges that hold chunks of it (of no chunks: the one that holds its start).
    const int w0 = ranges.of(at + (n ? a.pair_cost : 0));
    const int w1 = n ? ranges.of(at + span - 1) : w0;
    at += span;
    if (w >= w0 && w <= w1)
      segment(b, h, L, from, from / kChunk + c0, from / kChunk + c1, w0, w - w0, w1 - w0 + 1);
    if (at >= x1) return;
    if (++h == a.hkv) {
      h = 0;
      if (++b == a.num_seqs) return;
    }
  }
}

// ---- launch plan ----

// List positions of 32 tokens: what a pair costs beside its chunks, and the fewest a range
// takes. Measured on MI355X (us; positions of a pair 2, 8, 16): 4 x 8000 tokens at 14 / 2 heads of
// 64 16.5, 15.5, 14.0; 100 ragged up to 4000 28.3, 27.7, 25.6; 64 ragged up to 8000 at 32 / 8 of 128
// 190.5 and 189.9 of the last two. Ranges of 8, 16 and 32 at least: one context of 24000 16.4, 14.7,
// 17.0.
// At head_dim 256, whose chunks are longer: 40 ragged up to 6000 at 16 / 8 heads 175 of 8, 182 of 16.
static int pair_cost(int head_dim) { return head_dim <= 128 ? 16 : 8; }
constexpr int kMinRange = 16;
// Windows (or tables) of at most this many tokens take one workgroup per pair: beyond, records and
// their merge cost less than the wait for one compute unit's reading. 8 contexts of 2000 tokens at
// 14 / 2 heads of 64 15.2 us in ranges, 11.9 whole; of 128, 1500 tokens 15.0 and 15.2, 2000 at 32 / 8
// 20.3 and 26.5; of 256, 1200 tokens 22.8 and 26.5.
static int whole_pairs(int head_dim) { return head_dim <= 64 ? 2048 : head_dim == 128 ? 1536 : 1024; }
// And where the pairs fill at least half the compute units (100 ragged up to 2040 at 14 / 2 heads of
// 64 15.3 whole, 20.3 in ranges).
constexpr int kWholePairsBusy = 2048;

struct Plan {
  int waves, ranged, grid, rec_floats;
  size_t ws_bytes;
};

static Plan plan_of(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim, int block_size,
                    int max_blocks, int window) {
  Plan p{};
  const int n = device_cus();
  int64_t seen = (int64_t)max_blocks * block_size;
  if (window > 0 && window < seen) seen = window;
  const int64_t chunks = (seen + 2 * kChunk - 2) / kChunk;  // that an interval of so many can touch
  const int64_t pairs = (int64_t)num_seqs * num_kv_heads;
  const bool few = pairs <= n;
  const int64_t whole = 2 * pairs >= n ? kWholePairsBusy : whole_pairs(head_dim);
  p.ranged = seen > whole && pairs <= kMaxCounters && pairs * (chunks + pair_cost(head_dim)) < 0x7fffffff;
  // One workgroup of eight wavefronts per compute unit, for few pairs or ranges (two of four: 64
  // ragged up to 8000 198.5 us, one of eight 190; 200 ragged up to 6000 at 16 / 8 heads of 64 213 and
  // 200); four wavefronts for many short pairs, several at a time, and at head_dim 256, for LDS.
  p.waves = head_dim <= 128 && (few || p.ranged) ? 8 : 4;
  p.grid = pairs > 0x7fffffff ? -1 : (int)pairs;
  if (p.ranged) {
    // No more ranges than the longest lengths fill.
    const int64_t most = pairs * (chunks + pair_cost(head_dim)) / kMinRange;
    p.grid = (int)(most < n ? (most < 1 ? 1 : most) : n);
    p.rec_floats = record_size(num_q_heads / num_kv_heads, head_dim);
    p.ws_bytes = kCounterBytes + (size_t)2 * p.grid * p.rec_floats * sizeof(float);
  }
  return p;
}

template <int D, int NW>
static hipError_t launch_nw(const Args& a, unsigned grid, hipStream_t s) {
  // (The uniform tiles' loads take 31-bit offsets within 16 rows.)
  const bool near = a.k_st < (1 << 26) && a.v_st < (1 << 26);
  if (a.bs == 16 && near)
    decode_scored_kernel<D, 16, NW><<<grid, 64 * NW, 0, s>>>(a);
  else if (a.bs == 32 && near)
    decode_scored_kernel<D, 32, NW><<<grid, 64 * NW, 0, s>>>(a);
  else
    decode_scored_kernel<D, 0, NW><<<grid, 64 * NW, 0, s>>>(a);
  return hipGetLastError();
}

static hipError_t launch(const Args& a, int D, const Plan& p, hipStream_t s) {
  const unsigned grid = (unsigned)p.grid;
  switch (D * 16 + p.waves) {
    case 32 * 16 + 4: return launch_nw<32, 4>(a, grid, s);
    case 32 * 16 + 8: return launch_nw<32, 8>(a, grid, s);
    case 64 * 16 + 4: return launch_nw<64, 4>(a, grid, s);
    case 64 * 16 + 8: return launch_nw<64, 8>(a, grid, s);
    case 128 * 16 + 4: return launch_nw<128, 4>(a, grid, s);
    case 128 * 16 + 8: return launch_nw<128, 8>(a, grid, s);
    case 256 * 16 + 4: return launch_nw<256, 4>(a, grid, s);
    default: return hipErrorInvalidValue;
  }
}

static bool sizes_ok(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim, int block_size,
                     int max_blocks) {
  return num_seqs > 0 && num_q_heads > 0 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0 &&
         num_q_heads / num_kv_heads <= 16 && block_size > 0 && max_blocks > 0 &&
         (int64_t)max_blocks * block_size <= 0x7fffffff - 4096 &&
         (head_dim == 32 || head_dim == 64 || head_dim == 128 || head_dim == 256);
}

}  // namespace scored
}  // namespace pa

using namespace pa;
using namespace pa::scored;

extern "C" {

size_t pa_decode_scored_workspace_bytes(int num_seqs, int num_q_heads, int num_kv_heads,
                                        int head_dim, int block_size, int max_blocks_per_seq,
                                        int window) {
  if (!sizes_ok(num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq)) return 0;
  return plan_of(num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq,
                 window).ws_bytes;
}

int pa_decode_scored_f16(const void* q, const int64_t q_strides[3], const void* k_cache,
                         const int64_t k_strides[4], const void* v_cache,
                         const int64_t v_strides[4], const int32_t* block_tables,
                         const int64_t bt_strides[2], const int32_t* seq_lens, void* out,
                         const int64_t out_strides[3], int num_seqs, int num_q_heads,
                         int num_kv_heads, int head_dim, int block_size, int num_blocks,
                         int max_blocks_per_seq, float scale, float softcap, const float* slopes,
                         int64_t slope_stride, int window, const int32_t* key_starts,
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
  if (!sizes_ok(num_seqs, num_q_heads, num_kv_heads, head_dim, block_size, max_blocks_per_seq)) {
    set_error("not built: head_dim %d (32, 64, 128, 256), query group size %d (at most 16), or "
              "tables of 2^31 tokens", head_dim, num_q_heads / num_kv_heads);
    return PA_ERR_UNSUPPORTED;
  }
  if (!q || !q_strides || !k_cache || !k_strides || !v_cache || !v_strides || !block_tables ||
      !bt_strides || !seq_lens || !out || !out_strides) {
    set_error("null pointer argument");
    return PA_ERR_ARG;
  }
  int rc = check_scores(scale, softcap, window);
  if (rc) return rc;
  for (int i = 0; i < 3; ++i) {
    if (k_strides[i] % 8 || v_strides[i] % 8 || k_strides[i] < 0 || v_strides[i] < 0) {
      set_error("cache strides must be non-negative multiples of 8 elements");
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
  const Plan p = plan_of(num_seqs, num_q_heads, num_kv_heads, head_dim, block_size,
                         max_blocks_per_seq, window);
  if (p.ws_bytes && (!workspace || workspace_bytes < p.ws_bytes)) {
    set_error("workspace of %zu bytes needed, %zu given", p.ws_bytes, workspace_bytes);
    return PA_ERR_WORKSPACE;
  }
  if (p.grid < 0) {
    set_error("%d sequences of %d kv heads exceed one launch", num_seqs, num_kv_heads);
    return PA_ERR_UNSUPPORTED;
  }
  Args a{};
  a.q = (const f16*)q;
  a.q_sb = q_strides[0];
  a.q_sh = q_strides[1];
  a.k = (const uint8_t*)k_cache;
  a.k_sb = k_strides[0] * 2;
  a.k_st = k_strides[1] * 2;
  a.k_sh = k_strides[2] * 2;
  a.v = (const uint8_t*)v_cache;
  a.v_sb = v_strides[0] * 2;
  a.v_st = v_strides[1] * 2;
  a.v_sh = v_strides[2] * 2;
  a.bt = block_tables;
  a.bt_sb = bt_strides[0];
  a.bt_sk = bt_strides[1];
  a.lens = seq_lens;
  a.starts = key_starts;
  a.slopes = slopes;
  a.slope_s = slope_stride;
  a.out = (f16*)out;
  a.o_sb = out_strides[0];
  a.o_sh = out_strides[1];
  a.num_seqs = num_seqs;
  a.hkv = num_kv_heads;
  a.g = num_q_heads / num_kv_heads;
  a.bs = block_size;
  a.num_blocks = num_blocks;
  a.max_blocks = max_blocks_per_seq;
  a.window = window;
  a.cnt = (int*)workspace;
  a.recs = (float*)((char*)workspace + (p.ws_bytes ? kCounterBytes : 0));
  a.ranged = p.ranged;
  a.min_range = kMinRange;
  a.pair_cost = pair_cost(head_dim);
  a.rec_floats = p.rec_floats;
  const ScoreForm f = score_form(scale, softcap);
  a.scale_log2 = f.scale_log2;
  a.cap_log2 = f.cap_log2;
  a.cap_out = f.cap_out;
  a.cap_in = f.cap_in;
  a.cap_t = f.cap_t;
  const hipError_t e = launch(a, head_dim, p, (hipStream_t)stream);
  if (e == hipSuccess) return PA_OK;
  set_error("HIP launch failed: %s", hipGetErrorString(e));
  return PA_ERR_HIP;
}

}  // extern "C"
