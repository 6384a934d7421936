// Decode attention over the 8-bit paged pool (gfx950): one query token per sequence.
//
//   o = sum_t p_t v_t / sum_t p_t,  p_t = 2^(scale log2(e) q.k_t - m),  m the maximum
//   so far, K and V rows = e4m3 code * scale[block, kv head]
//
// Work split. The work is a list of (sequence, group of HG adjacent kv heads) pairs, each
// of its 32-token chunks plus a fixed cost; a grid of a few workgroups per compute unit
// takes equal contiguous ranges of it, so every workgroup reads about the same bytes
// however lengths differ. Each wavefront derives the plan for itself, from the lengths,
// with lane scans: no memory, no barrier. Where every pair is short a workgroup takes one
// pair whole and there is no plan. Within a pair's part of its range, a workgroup's four
// wavefronts take the chunks in turn, each with its own online softmax for the whole
// query group, and meet in LDS at the end. A pair inside one range is written as fp16
// there; a pair cut by range boundaries leaves fp32 partial records, and the last of its
// workgroups to arrive combines them by log-sum-exp in list order (the same bits on
// every run).
//
// Per chunk. Lane (row, grp) loads 16 bytes of token `row`'s K row per 64: with the
// head's elements taken in that order on both sides these are the A operands of
// S^T = K Q^T (v_mfma_f32_16x16x32_f16), so K needs no LDS. Codes become fp16 in
// v_cvt_scalef32_pk_f16_fp8 with the scale applied, exactly: the products and sums are
// those of an fp16 cache that holds the same values. V rows take the same loads,
// conversion, and a pass through LDS (each wavefront's own, without barriers) for the
// transposed operand of O^T += V^T P^T. Registers of K and V are free for the next
// chunk's loads as soon as the scores exist and V is in LDS.
//
// Probabilities are rounded to fp16 (the denominators sum the rounded ones), scaled by
// 2^14 so that they keep 11 bits down to 2^-28 of the largest: half a step, 2^-12
// relative, next to the cache's own rounding of up to 2^-4.
#include "../../include/paged_attention.h"
#include "pa_fp8.h"
#include "pa_tiles.h"

namespace pa {
namespace fp8 {

using namespace tiles;

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kChunk = 32;  // tokens a wavefront takes at a time
// The workspace starts with arrival counters at the same place for every call, one per
// pair of a call that is cut into ranges.
constexpr int kMaxCounters = 16384;
constexpr size_t kCounterBytes = (size_t)kMaxCounters * sizeof(int);
constexpr float kBias = 14.f;  // log2 of the factor on the probabilities

struct DecodeFp8Args {
  const f16* q;
  int64_t q_sb, q_sh;
  const uint8_t* k;
  int64_t k_sb, k_st, k_sh;
  const uint8_t* v;
  int64_t v_sb, v_st, v_sh;
  const float* ks;
  int64_t ks_sb, ks_sh;
  const float* vs;
  int64_t vs_sb, vs_sh;
  const int32_t* bt;
  int64_t bt_sb, bt_sk;
  const int32_t* lens;
  f16* out;
  int64_t o_sb, o_sh;
  int* cnt;
  float* recs;
  int num_seqs, hkv, g, bs, num_blocks, max_blocks;
  int ranged;      // 0: one workgroup per pair, no plan
  int min_range;   // list positions a range has at least
  int pair_cost;   // list positions a pair takes beside its chunks
  int rec_floats;
  float scale_log2;
};

// Floats of a partial record: heads x dim accumulators, then maxima and denominators.
__host__ __device__ inline int record_size(int heads, int D) { return (heads * (D + 2) + 3) & ~3; }

// A wavefront-uniform value, in scalar registers.
__device__ inline int64_t uniform64(int64_t x) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)x);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)((uint64_t)x >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// Range w of G of a T-position list starts at w T / G; the range that holds position x.
__device__ inline int64_t range_start(int64_t w, int64_t T, int64_t G) { return w * T / G; }
__device__ inline int range_of(int64_t x, int64_t T, int64_t G) {
  return (int)(((x + 1) * G - 1) / T);
}

// A lane's load through a tile resource, with load_tile's cache policy.
template <typename W>
__device__ inline W load_words(__amdgpu_buffer_rsrc_t r, uint32_t lane_off, int off) {
  if constexpr (sizeof(W) == 16)
    return load_tile(r, lane_off, off);
  else
    return __builtin_bit_cast(W, __builtin_amdgcn_raw_buffer_load_b64(r, (int)lane_off, off, 3));
}

template <int D, int HG, int BS>
__global__ __launch_bounds__(kThreads) void decode_fp8_kernel(DecodeFp8Args a) {
  constexpr int LB = D >= 64 ? 16 : 8;  // bytes of one lane's load
  constexpr int SEG = D / (4 * LB);     // loads per head and 16-token tile
  constexpr int NF = LB / 8;            // MFMA operands per load
  constexpr int NC = D / 32;            // products per score tile
  constexpr int ND = D / 16;
  constexpr int D4 = D / 4;
  constexpr int LS = D + 16;  // LDS row stride of the staged V rows (halves)
  constexpr int AS = D + 4;   // LDS row stride of the accumulators (floats)
  constexpr int STAGE = HG * kChunk * LS;  // halves per wavefront
  static_assert(STAGE * 2 >= HG * 16 * AS * 4, "the accumulators reuse the staging area");
  typedef unsigned words __attribute__((ext_vector_type(LB / 4)));
  constexpr bool UNIFORM = BS > 0;  // a 16-token tile lies in one block
  static_assert(BS % 16 == 0, "whole tiles per block, or any block size as 0");
  __shared__ __attribute__((aligned(16))) f16 s_stage[kWaves * STAGE];
  __shared__ __attribute__((aligned(16))) f32x4 s_part[kThreads];
  __shared__ float s_m[kWaves][HG * 16], s_l[kWaves][HG * 16];
  __shared__ int s_last;

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int row = lane & 15;
  const int grp = lane >> 4;
  const int bs = BS > 0 ? BS : a.bs;
  const int groups = a.hkv / HG;
  const int heads = HG * a.g;  // query heads of a pair
  const int cap = a.max_blocks * bs;
  const int last_tile = (cap - 1) / 16;
  f16* stage = s_stage + wave * STAGE;
  const uint32_t k_lane = (uint32_t)(row * a.k_st + grp * LB);
  const uint32_t v_lane = (uint32_t)(row * a.v_st + grp * LB);
  constexpr int kAll = 0x7fffffff;

  auto clamped = [&](int n) { return n < 0 ? 0 : (n > cap ? cap : n); };
  auto chunks_of = [&](int n) { return (clamped(n) + kChunk - 1) / kChunk; };

  // Chunks [c0, c1) of pair (b, group from kv head h0) of a sequence of L tokens. The pair
  // is spread over nseg workgroups' ranges, from range w0 on; this is its part `seg`.
  auto segment = [&](int b, int h0, int L, int c0, int c1, int w0, int seg, int nseg) {
    const int32_t* btrow = a.bt + (int64_t)b * a.bt_sb;
    int ids[2];
    // Clamped to the table's width only, so that ids need no length: a tile past the end
    // reads some block of the pool and what it reads is masked.
    auto load_ids = [&](int c) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if constexpr (UNIFORM) {
          // A tile lies in one block: its id is wavefront-uniform.
          const int at = min(2 * c + t, last_tile);
          ids[t] = load_uniform(btrow + (int64_t)(at / (BS / 16)) * a.bt_sk);
        } else {
          ids[t] = btrow[(int64_t)(min(c * kChunk + t * 16 + row, cap - 1) / bs) * a.bt_sk];
        }
      }
    };
    const int first = c0 + wave;
    load_ids(first);
    // Q^T operands: column = query head `row` of a kv head's group, elements in the order
    // of the K loads.
    f16x8 qf[HG][NC];
#pragma unroll
    for (int hg = 0; hg < HG; ++hg) {
      const f16* qp = a.q + (int64_t)b * a.q_sb +
                      (int64_t)((h0 + hg) * a.g + min(row, a.g - 1)) * a.q_sh;
#pragma unroll
      for (int s = 0; s < SEG; ++s)
#pragma unroll
        for (int f = 0; f < NF; ++f)
          qf[hg][s * NF + f] =
              *reinterpret_cast<const f16x8*>(qp + s * 4 * LB + grp * LB + f * 8);
    }
    words kb[2][HG][SEG], vb[2][HG][SEG];
    float ksc[2][HG], vsc[2][HG];
    auto load_kv = [&](int c) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int64_t id = min(max(ids[t], 0), a.num_blocks - 1);
        if constexpr (UNIFORM) {
          // Row offsets within a tile are the lane's own, everything else is uniform.
          const int64_t off = (2 * c + t) % (BS / 16) * 16;
          const auto kr = tile_rsrc(a.k + id * a.k_sb + off * a.k_st + (int64_t)h0 * a.k_sh, kAll);
          const auto vr = tile_rsrc(a.v + id * a.v_sb + off * a.v_st + (int64_t)h0 * a.v_sh, kAll);
#pragma unroll
          for (int hg = 0; hg < HG; ++hg) {
#pragma unroll
            for (int s = 0; s < SEG; ++s) {
              kb[t][hg][s] = load_words<words>(kr, k_lane, (int)(hg * a.k_sh) + s * 4 * LB);
              vb[t][hg][s] = load_words<words>(vr, v_lane, (int)(hg * a.v_sh) + s * 4 * LB);
            }
            ksc[t][hg] = load_uniform(a.ks + id * a.ks_sb + (h0 + hg) * a.ks_sh);
            vsc[t][hg] = load_uniform(a.vs + id * a.vs_sb + (h0 + hg) * a.vs_sh);
          }
        } else {
          const int64_t off = (c * kChunk + t * 16 + row) % bs;
          const uint8_t* kp = a.k + id * a.k_sb + off * a.k_st + (int64_t)h0 * a.k_sh + grp * LB;
          const uint8_t* vp = a.v + id * a.v_sb + off * a.v_st + (int64_t)h0 * a.v_sh + grp * LB;
#pragma unroll
          for (int hg = 0; hg < HG; ++hg) {
#pragma unroll
            for (int s = 0; s < SEG; ++s) {
              kb[t][hg][s] = __builtin_nontemporal_load(
                  reinterpret_cast<const words*>(kp + hg * a.k_sh + s * 4 * LB));
              vb[t][hg][s] = __builtin_nontemporal_load(
                  reinterpret_cast<const words*>(vp + hg * a.v_sh + s * 4 * LB));
            }
            ksc[t][hg] = a.ks[id * a.ks_sb + (h0 + hg) * a.ks_sh];
            vsc[t][hg] = a.vs[id * a.vs_sb + (h0 + hg) * a.vs_sh];
          }
        }
      }
    };

    float m_run[HG], l_run[HG];
    f32x4 acc[HG][ND];
#pragma unroll
    for (int hg = 0; hg < HG; ++hg) {
      m_run[hg] = kNegInf;
      l_run[hg] = 0.f;
#pragma unroll
      for (int nd = 0; nd < ND; ++nd) acc[hg][nd] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (first < c1) {
      load_kv(first);
      load_ids(first + kWaves);
    }
    for (int c = first; c < c1; c += kWaves) {
      const int t0 = c * kChunk;
      const bool whole = t0 + kChunk <= L;  // wavefront-uniform: the last chunk may not be
      // Scores, and V into LDS.
      float x[HG][2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int hg = 0; hg < HG; ++hg) {
          f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < SEG; ++i)
#pragma unroll
            for (int f = 0; f < NF; ++f)
              s = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                  from_codes8(kb[t][hg][i][2 * f], kb[t][hg][i][2 * f + 1], ksc[t][hg]),
                  qf[hg][i * NF + f], s, 0, 0, 0);
#pragma unroll
          for (int r = 0; r < 4; ++r) x[hg][t][r] = s[r] * a.scale_log2;
          if (!whole) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (t0 + t * 16 + grp * 4 + r >= L) x[hg][t][r] = kNegInf;
          }
          f16* sp = stage + (hg * kChunk + t * 16 + row) * LS + grp * LB;
          // Rows past the end are staged as zeros: 0 * what lies there is never NaN.
          const bool in = whole || t0 + t * 16 + row < L;
#pragma unroll
          for (int i = 0; i < SEG; ++i)
#pragma unroll
            for (int f = 0; f < NF; ++f) {
              const f16x8 y = from_codes8(vb[t][hg][i][2 * f], vb[t][hg][i][2 * f + 1], vsc[t][hg]);
              *reinterpret_cast<f16x8*>(sp + i * 4 * LB + f * 8) = in ? y : zero8();
            }
        }
      if (c + kWaves < c1) {
        load_kv(c + kWaves);
        load_ids(c + 2 * kWaves);
      }
      // Softmax of the chunk.
      f16x8 pb[HG];
#pragma unroll
      for (int hg = 0; hg < HG; ++hg) {
        float m = kNegInf;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) m = fmaxf(m, x[hg][t][r]);
        m = fmaxf(m, __shfl_xor(m, 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        const float m_new = fmaxf(m_run[hg], m);
        const float alpha = fast_exp2(m_run[hg] - m_new);
        l_run[hg] *= alpha;
#pragma unroll
        for (int nd = 0; nd < ND; ++nd) acc[hg][nd] *= alpha;
        m_run[hg] = m_new;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const f16 p = (f16)fast_exp2(x[hg][t][r] - m_new + kBias);
            pb[hg][4 * t + r] = p;
            l_run[hg] += (float)p;
          }
      }
      wave_lds_fence();
      // O^T += V^T P^T: operand index k = 8 grp + i stands for token 4 grp + i of tile 0
      // (i < 4) or 4 grp + i - 4 of tile 1, on both sides.
#pragma unroll
      for (int hg = 0; hg < HG; ++hg) {
        const f16* v0 = stage + (hg * kChunk + grp * 4 + (row >> 2)) * LS + (row & 3) * 4;
#pragma unroll
        for (int nd = 0; nd < ND; ++nd) {
          const f16x4 a0 = lds_read_tr16(v0 + nd * 16);
          const f16x4 a1 = lds_read_tr16(v0 + 16 * LS + nd * 16);
          const f16x8 av = {a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]};
          acc[hg][nd] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, pb[hg], acc[hg][nd], 0, 0, 0);
        }
      }
      wave_lds_fence();
    }

    // The wavefronts' states meet in LDS. (Lane indices anew: see fresh_lane.)
    const int lane = fresh_lane();
    const int tid = wave * 64 + lane, row = lane & 15, grp = lane >> 4;
    float* my_acc = reinterpret_cast<float*>(stage);
#pragma unroll
    for (int hg = 0; hg < HG; ++hg) {
      float l = l_run[hg];
      l += __shfl_xor(l, 16);
      l += __shfl_xor(l, 32);
      if (grp == 0) {
        s_m[wave][hg * 16 + row] = m_run[hg];
        s_l[wave][hg * 16 + row] = l;
      }
      if (row < a.g) {
#pragma unroll
        for (int nd = 0; nd < ND; ++nd)
          *reinterpret_cast<f32x4*>(my_acc + (hg * 16 + row) * AS + nd * 16 + grp * 4) = acc[hg][nd];
      }
    }
    __syncthreads();
    // Part i of a cut pair lies in range w0 + i's slot 0 (the pair began before that range)
    // or, i = 0, in slot 1.
    const int64_t rec0 = (int64_t)(2 * w0 + 1) * a.rec_floats;
    auto record = [&](int i) { return (i ? 2 * i - 1 : 0) * a.rec_floats; };  // from rec0
    const auto rr = tile_rsrc(a.recs + rec0, (2 * nseg - 1) * a.rec_floats * 4);
    const int rb = record(seg) * 4;
    f16* out = a.out + (int64_t)b * a.o_sb + (int64_t)h0 * a.g * a.o_sh;
    for (int i = tid; i < heads * D4; i += kThreads) {
      const int j = i / D4;
      const int d = (i - j * D4) * 4;
      const int hg = j / a.g;
      const int r = hg * 16 + (j - hg * a.g);
      float M = s_m[0][r];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) M = fmaxf(M, s_m[w][r]);
      float l = 0.f;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = w < c1 - c0 ? fast_exp2(s_m[w][r] - M) : 0.f;  // 0: it had no chunk
        l += f * s_l[w][r];
        o += f * *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(s_stage + w * STAGE) +
                                                 r * AS + d);
      }
      if (nseg == 1) {
        const float inv = c1 > c0 ? 1.f / l : 0.f;
        f16x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (f16)(o[e] * inv);
        *reinterpret_cast<f16x4*>(out + (int64_t)j * a.o_sh + d) = y;
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
    int* cnt = a.cnt + (int64_t)b * groups + h0 / HG;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);  // the record has landed before the arrival counts
    __syncthreads();
    if (tid == 0)
      s_last = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == nseg - 1;
    __syncthreads();
    if (!s_last) return;  // (the next segment writes s_last behind further barriers)
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");

    // Merge. Maximum and sum over the parts per head (a wavefront takes every fourth head,
    // its lanes the parts), then batches of parts: their weights exp2(m - max) / sum into
    // LDS, their accumulators by threads (item: head and four of its elements; the parts
    // of an item are dealt over as many threads as there are for it).
    float* s_max = s_m[0];  // (the wavefronts' states are spent)
    float* s_inv = s_l[0];
    auto load_ml = [&](int j, int i, float& m, float& l) {
      const int at = (record(i) + heads * D) * 4;
      m = load_coherent4(rr, at + j * 4);
      l = load_coherent4(rr, at + (heads + j) * 4);
    };
#pragma unroll 1
    for (int j = wave; j < heads; j += kWaves) {
      float M = kNegInf, sum = 0.f;  // over this lane's parts
#pragma unroll 1
      for (int i = lane; i < nseg; i += 64) {
        float m, l;
        load_ml(j, i, m, l);
        const float m_new = fmaxf(M, m);
        if (m_new != kNegInf) sum = sum * fast_exp2(M - m_new) + l * fast_exp2(m - m_new);
        M = m_new;
      }
      float all = M;
#pragma unroll
      for (int off = 32; off; off >>= 1) all = fmaxf(all, __shfl_xor(all, off));
      sum = M == kNegInf ? 0.f : sum * fast_exp2(M - all);
#pragma unroll
      for (int off = 32; off; off >>= 1) sum += __shfl_xor(sum, off);
      if (lane == 0) {
        s_max[j] = all;
        s_inv[j] = all == kNegInf ? 0.f : 1.f / sum;  // no token at all: zeros
      }
    }
    float* s_w = reinterpret_cast<float*>(s_stage);
    const int batch = min(nseg, (int)(sizeof(s_stage) / 4) / heads);
    const int items = heads * D4;
    const int parts = items < kThreads ? kThreads / items : 1;
#pragma unroll 1
    for (int base = 0; base < items; base += kThreads) {  // workgroup-uniform
      const int part = parts > 1 ? tid / items : 0;
      const int item = parts > 1 ? tid - part * items : base + tid;
      const bool live = part < parts && item < items;
      const int j = live ? item / D4 : 0;
      const int d = live ? (item - j * D4) * 4 : 0;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int s0 = 0; s0 < nseg; s0 += batch) {
        const int s1 = min(nseg, s0 + batch);
        __syncthreads();
#pragma unroll 1
        for (int i = tid; i < heads * (s1 - s0); i += kThreads) {
          const int jj = i / (s1 - s0);
          const int k = i - jj * (s1 - s0);
          float m, l;
          load_ml(jj, s0 + k, m, l);
          s_w[jj * batch + k] = m == kNegInf ? 0.f : fast_exp2(m - s_max[jj]) * s_inv[jj];
        }
        __syncthreads();
        constexpr int U = 12;
        if (live)
#pragma unroll 1
          for (int i = s0 + part; i < s1; i += U * parts) {
            f32x4 y[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
              y[u] = load_coherent16(rr, (record(min(i + u * parts, s1 - 1)) + j * D + d) * 4);
#pragma unroll
            for (int u = 0; u < U; ++u)
              if (i + u * parts < s1) o += s_w[j * batch + i + u * parts - s0] * y[u];
          }
      }
      if (parts > 1) {
        s_part[tid] = o;
        __syncthreads();
        if (part == 0)
          for (int p = 1; p < parts; ++p) o += s_part[item + p * items];
      }
      if (live && part == 0) {
        f16x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (f16)o[e];
        *reinterpret_cast<f16x4*>(out + (int64_t)j * a.o_sh + d) = y;
      }
    }
    if (tid == 0) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
  };

  // This workgroup's part of the list: positions [x0, x1) of T, cut into G ranges; `at`
  // is the first position of sequence b.
  int64_t T = 0, G = 1, x0 = 0, x1 = 0, at = 0;
  int b = 0, g0 = 0, w = 0;
  if (a.ranged) {
    // Each sequence takes groups x (its chunks + pair_cost) positions.
    auto width = [&](int n) { return (int64_t)groups * (chunks_of(n) + a.pair_cost); };
    int64_t mine = 0;
    for (int i = lane; i < a.num_seqs; i += 64) mine += width(a.lens[i]);
#pragma unroll
    for (int off = 32; off; off >>= 1) mine += __shfl_xor(mine, off);
    T = uniform64(mine);
    G = max((int64_t)1, min((int64_t)gridDim.x, T / a.min_range));
    if (blockIdx.x >= G) return;
    w = xcd_order(blockIdx.x, (int)G);
    x0 = range_start(w, T, G);
    x1 = range_start(w + 1, T, G);
    for (int base = 0; base < a.num_seqs; base += 64) {
      const int64_t own = base + lane < a.num_seqs ? width(a.lens[base + lane]) : 0;
      int64_t incl = own;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int64_t y = __shfl_up(incl, off);
        if (lane >= off) incl += y;
      }
      const int64_t total = uniform64(__shfl(incl, 63));
      if (at + total > x0) {
        const int l = (int)__builtin_ctzll(__ballot(at + incl > x0));
        b = base + l;
        at += uniform64(__shfl(incl - own, l));
        break;
      }
      at += total;
    }
    b = __builtin_amdgcn_readfirstlane(b);
  } else {
    const int pair = xcd_order(blockIdx.x, gridDim.x);
    b = pair / groups;
    g0 = pair - b * groups;
  }
  for (;;) {
    const int L = clamped(load_uniform(a.lens + b));
    const int n = (L + kChunk - 1) / kChunk;
    int c0 = 0, c1 = n, w0 = 0, w1 = 0;
    if (a.ranged) {
      // The pair's positions: pair_cost of them, then its chunks.
      const int span = n + a.pair_cost;
      for (; g0 < groups && at + span <= x0; ++g0) at += span;
      if (g0 == groups) {
        g0 = 0;
        if (++b == a.num_seqs) return;
        continue;
      }
      if (at >= x1) return;
      c0 = (int)max((int64_t)0, min((int64_t)n, x0 - at - a.pair_cost));
      c1 = (int)max((int64_t)0, min((int64_t)n, x1 - at - a.pair_cost));
      w0 = range_of(at, T, G);
      w1 = range_of(at + span - 1, T, G);
      at += span;
    }
    segment(b, g0 * HG, L, c0, c1, w0, w - w0, w1 - w0 + 1);
    if (!a.ranged || at >= x1) return;
    if (++g0 == groups) {
      g0 = 0;
      if (++b == a.num_seqs) return;
    }
  }
}

// ---- plan, argument checks and the C entry points ----

struct DecodePlan {
  int head_group, ranged, grid;
  size_t ws_bytes;
};

// Workgroups per compute unit of a ranged launch.
constexpr int kRangesPerCu = 3;
// List positions of 32 tokens: what a pair costs beside its chunks, and the fewest a
// range takes.
constexpr int kPairCost = 8;
constexpr int kMinRange = 8;
// Tables of at most this many tokens take one workgroup per pair.
constexpr int kWholePairs = 512;

static DecodePlan decode_plan(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                              int block_size, int max_blocks) {
  DecodePlan p{};
  const int n = device_cus();
  p.head_group =
      head_dim <= 64 && num_kv_heads % 2 == 0 && (int64_t)num_seqs * num_kv_heads > n ? 2 : 1;
  const int64_t pairs = (int64_t)num_seqs * (num_kv_heads / p.head_group);
  const int64_t cap = (int64_t)max_blocks * block_size;
  p.ranged = cap > kWholePairs && pairs <= kMaxCounters;
  p.grid = pairs > 0x7fffffff ? -1 : (int)pairs;
  if (p.ranged) {
    // No more ranges than the longest lengths could fill.
    const int64_t most = pairs * ((cap + kChunk - 1) / kChunk + kPairCost) / kMinRange;
    p.grid = (int)(most < kRangesPerCu * n ? (most < 1 ? 1 : most) : kRangesPerCu * n);
    const int heads = num_q_heads / num_kv_heads * p.head_group;
    p.ws_bytes =
        kCounterBytes + (size_t)2 * p.grid * record_size(heads, head_dim) * sizeof(float);
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

template <int D, int HG>
static void launch_decode_bs(const DecodeFp8Args& a, unsigned grid, hipStream_t s) {
  // The uniform tiles' loads take 31-bit offsets within 16 rows of HG heads.
  const int64_t most = 1 << 26;
  const bool near = a.k_st < most && a.v_st < most && a.k_sh < most && a.v_sh < most;
  if (a.bs == 16 && near)
    decode_fp8_kernel<D, HG, 16><<<grid, kThreads, 0, s>>>(a);
  else if (a.bs == 32 && near)
    decode_fp8_kernel<D, HG, 32><<<grid, kThreads, 0, s>>>(a);
  else
    decode_fp8_kernel<D, HG, 0><<<grid, kThreads, 0, s>>>(a);
}

static void launch_decode(const DecodeFp8Args& a, int D, int hg, unsigned grid, hipStream_t s) {
  switch (D * 4 + hg) {
    case 32 * 4 + 1: return launch_decode_bs<32, 1>(a, grid, s);
    case 32 * 4 + 2: return launch_decode_bs<32, 2>(a, grid, s);
    case 64 * 4 + 1: return launch_decode_bs<64, 1>(a, grid, s);
    case 64 * 4 + 2: return launch_decode_bs<64, 2>(a, grid, s);
    case 128 * 4 + 1: return launch_decode_bs<128, 1>(a, grid, s);
    case 256 * 4 + 1: return launch_decode_bs<256, 1>(a, grid, s);
  }
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
                     max_blocks_per_seq).ws_bytes;
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
                                   max_blocks_per_seq);
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
  a.cnt = (int*)workspace;
  a.recs = (float*)((char*)workspace + (p.ws_bytes ? kCounterBytes : 0));
  a.num_seqs = num_seqs;
  a.hkv = num_kv_heads;
  a.g = num_q_heads / num_kv_heads;
  a.bs = block_size;
  a.num_blocks = num_blocks;
  a.max_blocks = max_blocks_per_seq;
  a.ranged = p.ranged;
  a.min_range = kMinRange;
  a.pair_cost = kPairCost;
  a.rec_floats = record_size(a.g * p.head_group, head_dim);
  a.scale_log2 = scale * kLog2e;
  launch_decode(a, head_dim, p.head_group, (unsigned)p.grid, (hipStream_t)stream);
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return PA_OK;
  set_error("HIP launch failed: %s", hipGetErrorString(e));
  return PA_ERR_HIP;
}

}  // extern "C"
