// Attention over the 8-bit paged pool (gfx950) for one query token per sequence, or a few.
//
//   o = sum_t p_t v_t / sum_t p_t,  p_t = 2^(scale log2(e) (q.k_t - m)),  m the maximum
//   so far, K and V rows = e4m3 code * scale[block, kv head]
//
// Work split. The work is a list of (sequence, group of HG adjacent kv heads) pairs, each
// of its 32-token chunks plus a fixed cost; a grid of one or two workgroups per compute unit
// takes equal contiguous ranges of it, so every workgroup reads about the same bytes
// however lengths differ. Each wavefront derives the plan for itself, from the lengths,
// with lane scans: no memory, no barrier (1.3 us). Where every pair is short a workgroup
// takes one pair whole and there is no plan. Within a pair's part of its range, a
// workgroup's wavefronts take the chunks in turn, each with its own online softmax for the
// whole query group, and meet in LDS at the end. A pair inside one range is written as fp16
// there; a pair cut by range boundaries leaves fp32 partial records, and the last of its
// workgroups to arrive combines them by log-sum-exp in list order (the same bits on
// every run).
//
// Per chunk. K and V codes go from memory straight into LDS (buffer_load ... lds), whole
// rows of HG heads by neighbouring lanes: no registers are held while they are on their
// way, and eight wavefronts per compute unit have 8 KB each in flight. From there K is read
// in the operand layout of S^T = K Q^T and V by transposing reads of bytes
// (ds_read_b64_tr_b8) in that of O^T += V^T P^T, both v_mfma_f32_16x16x32_f16. Codes become
// fp16 in v_cvt_scalef32_pk_f16_fp8 with the scale applied, exactly: the products and sums
// are those of an fp16 cache that holds the same values. All fragments are in registers
// before the next chunk's loads are issued into the same LDS, and the arithmetic runs under
// those loads. Each wavefront has its own LDS, without barriers. The 16-byte pieces of a row
// are permuted by the row's number (by the lanes' addresses when loading), so that neither
// kind of read meets a bank twice.
//
// Bounds on MI355X (head_dim 64, 14 / 2 heads, block 16, unless stated). 256 sequences of
// 1.2M tokens in all (316 MB): memory, 62.4 us, 5.1 TB/s, where a gather of such 2 KB blocks
// alone reaches 6.3. 8 sequences of 1k to 8k at 32 / 8 heads of 128 (73 MB): 22.3 us, of
// which the streaming takes about 12; the rest is the chain launch -> plan -> first ids ->
// first chunk, and meeting, arrival and merge. One sequence: chains alone, 13.1 us at 24001
// tokens (3.7 of them the merge of 47 parts) and 5.7 at 300 tokens.
//
// Probabilities are rounded to fp16 (the denominators sum the rounded ones), scaled by
// 2^14 so that they keep 11 bits down to 2^-28 of the largest: half a step, 2^-12
// relative, next to the cache's own rounding of up to 2^-4.
//
// A few tokens per sequence (MULTI: drafts to be checked). The (token, query head) columns
// of one sequence and kv head, token-major, fill up to CB blocks of 16, which share every
// K and V fragment; a column sees the keys up to its token's position. A NaN in a V row
// reaches only the columns that see it: where some column does not see the whole chunk,
// NaN codes are cleared and the probabilities of their tokens become NaN instead. 16
// sequences of 0.3k to 4k tokens and 5 drafts at 32 / 8 heads of 128 (90 MB): 30.9 us, about 14
// of them streaming.
#pragma once

#include <type_traits>

#include "pa_fp8.h"
#include "pa_tiles.h"

namespace pa {
namespace fp8 {

using namespace tiles;

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
  // MULTI: first query row of each sequence, query rows, and the most a sequence may have.
  const int32_t* qstart;
  int num_tokens, max_new;
  int ranged;      // 0: one workgroup per pair, no plan
  int min_range;   // list positions a range has at least
  int pair_cost;   // list positions a pair takes beside its chunks
  int rec_floats;
  float scale_log2;
};

// Floats of a partial record: heads x dim accumulators, then maxima and denominators.
__host__ __device__ inline int record_size(int heads, int D) { return (heads * (D + 2) + 3) & ~3; }

// A T-position list cut into G ranges that differ by one position at most: the first T % G
// hold T / G + 1. Where range w starts, and the range that holds position x.
struct Cut {
  int q, r;
  __device__ int start(int w) const { return w * q + (w < r ? w : r); }
  __device__ int of(int x) const {
    const int head = r * (q + 1);
    return x < head ? x / (q + 1) : r + (x - head) / q;
  }
};

// The power of two that conversions of codes take from a scale: its exponent alone.
__device__ inline float power_of(float scale) {
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, scale) & 0x7f800000u);
}

// Lane l's value, in a scalar register.
__device__ inline float lane_value(float x, int l) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), l));
}

typedef __attribute__((address_space(3))) void* lds_ptr;
typedef __attribute__((address_space(1))) const void* global_ptr;

// 16 bytes of every lane from memory into LDS, lane by lane from `to` (uniform) on, with
// load_tile's cache policy; through a resource, or from a lane's own address.
__device__ inline void load_to_lds(__amdgpu_buffer_rsrc_t r, uint32_t lane_off, uint8_t* to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)to, 16, (int)lane_off, 0, 0, 3);
}
__device__ inline void load_to_lds(const uint8_t* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds((global_ptr)from, (lds_ptr)to, 16, 0, 3);
}

// Transposing LDS read of bytes: within each group of 16 lanes, lane 2 r + q supplies the
// address of bytes [8 q, 8 q + 8) of row r of an 8 x 16 block, and lane j receives column j
// (rows 0 .. 7).
__device__ inline uint2 lds_read_tr8(const uint8_t* p) {
  typedef int v2i __attribute__((__vector_size__(8)));
  auto* lp = (__attribute__((address_space(3))) v2i*)(const_cast<uint8_t*>(p));
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(lp));
}

// op over lanes l, l ^ 16, l ^ 32 and l ^ 48, in all four. (The swaps exchange rows of 16 or
// 32 lanes between two registers: the copy has to be one of its own.)
template <typename Op>
__device__ inline float over_groups(float x, Op op) {
  auto bits = [](float v) { return __builtin_bit_cast(unsigned, v); };
  auto val = [](unsigned u) { return __builtin_bit_cast(float, u); };
  unsigned copy = bits(x);
  asm volatile("" : "+v"(copy));
  const auto a = __builtin_amdgcn_permlane16_swap(bits(x), copy, false, false);
  const float y = op(val(a[0]), val(a[1]));
  copy = bits(y);
  asm volatile("" : "+v"(copy));
  const auto b = __builtin_amdgcn_permlane32_swap(bits(y), copy, false, false);
  return op(val(b[0]), val(b[1]));
}

// op over the 16 lanes of a row, in all of them (rotations within the row).
template <typename Op>
__device__ inline float over_row(float x, Op op) {
  auto turned = [](float v, auto by) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v),
                                                                 0x120 + decltype(by)::value, 0xf,
                                                                 0xf, false));
  };
  x = op(x, turned(x, std::integral_constant<int, 8>()));
  x = op(x, turned(x, std::integral_constant<int, 4>()));
  x = op(x, turned(x, std::integral_constant<int, 2>()));
  return op(x, turned(x, std::integral_constant<int, 1>()));
}
__device__ inline unsigned or_over_row(unsigned x) {
  x |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, false);
  x |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xf, 0xf, false);
  x |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xf, 0xf, false);
  return x | (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xf, 0xf, false);
}
struct Max {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Sum {
  __device__ float operator()(float a, float b) const { return a + b; }
};

// A uniform value in scalar registers of its own from here on. (The arguments come in blocks
// of sixteen registers; what loops use straight from them keeps whole blocks alive, which
// then come back lane by lane from vector registers at every use.)
template <typename T>
__device__ inline T pinned(T x) {
  asm volatile("" : "+s"(x));
  return x;
}

// The permutation of a row's 16-byte pieces in LDS: piece p of chunk row r lies in slot
// p ^ swizzle(r) of NP. Eight rows whose same piece is read at once, 0 .. 7 (V) or 0 .. 3
// and 8 .. 11 (K), then lie in different banks.
template <int NP>
__device__ inline int swizzle(int r) {
  const int f = (r & 3) | (((r >> 2) ^ (r >> 3)) & 1) << 2;
  return NP >= 8 ? f : NP == 4 ? f >> 1 : f >> 2;
}

// Wavefronts per SIMD that the registers are kept to. (A workgroup of eight is its compute
// unit's only one, and spills no vector registers then. Every form keeps about 90 to 150
// scalar registers in lanes of vector ones; of four wavefronts, two heads of 64 in blocks of
// other sizes than 16 and 32 alone spill vector registers, 7.)
constexpr int waves_per_simd(int D, int NW, int CB) {
  return D == 256 || CB > 1 || NW > 4 ? 2 : 3;
}

// NW: wavefronts of a workgroup. One token per sequence: a block of 16 columns for each of
// HG heads; MULTI: CB blocks of one head.
template <int D, int HG, int BS, int NW, int CB, bool MULTI>
__global__ __launch_bounds__(64 * NW, waves_per_simd(D, NW, CB)) void attend_fp8_kernel(DecodeFp8Args a) {
  static_assert(MULTI ? HG == 1 : CB == 1, "column blocks of one head, or one of each head");
  constexpr int NS = HG * CB;  // blocks of 16 columns, each with its online softmax
  constexpr int kThreads = 64 * NW;
  constexpr int RB = HG * D;            // bytes of a loaded row
  constexpr int NP = RB / 16;           // 16-byte pieces of it, one per lane
  constexpr int RPI = 64 / NP;          // rows per load instruction
  constexpr int NI = kChunk / RPI;      // load instructions per chunk, for K and for V
  // Whether an instruction's rows lie in one block: their address is then uniform.
  constexpr bool UNIFORM = BS > 0 && RPI <= 16;
  static_assert(BS % 16 == 0, "whole tiles per block, or any block size as 0");
  constexpr int FB = D >= 64 ? 16 : 8;  // bytes of one lane's K fragment read
  constexpr int SEG = D / (4 * FB);     // such reads per head and 16-token tile
  constexpr int NF = FB / 8;            // MFMA operands of one
  constexpr int NC = D / 32;            // products per score tile
  constexpr int ND = D / 16;
  constexpr int D4 = D / 4;
  // Bytes per wavefront: K rows, then V rows; at the end its accumulators.
  constexpr int STAGE = NS * 16 * D * 4;
  static_assert(STAGE >= 2 * kChunk * RB, "the accumulators take the larger room");
  typedef unsigned frag __attribute__((ext_vector_type(FB / 4)));
  __shared__ __attribute__((aligned(16))) uint8_t s_stage[NW * STAGE];
  __shared__ __attribute__((aligned(16))) f32x4 s_part[kThreads];
  __shared__ float s_m[NW][NS * 16], s_l[NW][NS * 16];
  // Scales per token where they are not uniform: fp32 of K, fp16 of V.
  __shared__ float s_ks[UNIFORM ? 1 : NW][HG * kChunk];
  __shared__ __attribute__((aligned(16))) f16 s_vs[UNIFORM ? 1 : NW][HG * kChunk];
  __shared__ int s_last;

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int row = lane & 15;
  const int grp = lane >> 4;
  const int bs = BS > 0 ? BS : a.bs;
  const int groups = a.hkv / HG;
  const int cap = a.max_blocks * bs;
  const int last_tile = (cap - 1) / 16;
  uint8_t* const stage = s_stage + wave * STAGE;
  // This lane's piece of a loaded row: row lrow of the instruction's. (The swizzle of rows
  // 8 on differs by 4 from that of the rows before; a row of 16 pieces takes instructions of
  // four rows, whose swizzles differ by 4 every second one.) Byte offsets, for both.
  const int lrow = lane / NP;
  auto piece = [&](int flip) { return ((lane % NP) ^ swizzle<NP>(lrow) ^ flip) * 16; };
  constexpr int FLIP = NP >= 8 ? 4 : 0;
  auto lane_offset = [&](int64_t st, int64_t sh, int flip) {
    const int c = piece(flip);
    return (uint32_t)(lrow * st + c / D * sh + c % D);
  };
  const uint32_t k_lane = lane_offset(a.k_st, a.k_sh, 0), k_flip = lane_offset(a.k_st, a.k_sh, FLIP);
  const uint32_t v_lane = lane_offset(a.v_st, a.v_sh, 0), v_flip = lane_offset(a.v_st, a.v_sh, FLIP);
  // Whether instruction i's rows have the flipped swizzle: bits 2 and 3 of i * RPI (those of
  // lrow are in swizzle(lrow)).
  auto flipped = [](int i) { return ((i * RPI >> 2) ^ (i * RPI >> 3)) & 1; };
  constexpr int kAll = 0x7fffffff;

  auto clamped = [&](int n) { return n < 0 ? 0 : (n > cap ? cap : n); };
  auto chunks_of = [&](int n) { return (clamped(n) + kChunk - 1) / kChunk; };

  // Chunks [c0, c1) of pair (b, group from kv head h0) of a sequence of L tokens (not ranged:
  // all chunks, of a length found here, while the first ids are on their way). The pair is
  // spread over nseg workgroups' ranges, from range w0 on; this is its part `seg`.
  auto segment = [&](int b, int h0, int L, int c0, int c1, int w0, int seg, int nseg) {
    const int32_t* const btrow = pinned(a.bt + (int64_t)b * a.bt_sb);
    const int64_t bt_sk = pinned(a.bt_sk);
    const uint8_t* const kbase = pinned(a.k + h0 * a.k_sh);
    const uint8_t* const vbase = pinned(a.v + h0 * a.v_sh);
    const int64_t k_sb = pinned(a.k_sb), v_sb = pinned(a.v_sb);
    const int64_t k_st = pinned(a.k_st), v_st = pinned(a.v_st);
    const int last_id = pinned(a.num_blocks - 1);
    // The scale that the lane loads of each chunk: see issue().
    const int shead = UNIFORM ? (HG > 1 ? lane >> 1 & 1 : 0) : (HG > 1 ? lane >> 5 : 0);
    const bool of_v = UNIFORM && (lane & 4);
    const float* const sbase = (of_v ? a.vs : a.ks) + (h0 + shead) * (of_v ? a.vs_sh : a.ks_sh);
    const int64_t s_sb = of_v ? a.vs_sb : a.ks_sb;
    // The columns of the pair: its query heads, or times its tokens.
    int q0 = b, qall = 1, heads = HG * a.g;
    if constexpr (MULTI) {
      q0 = min(max(load_uniform(a.qstart + b), 0), a.num_tokens);
      qall = min(max(load_uniform(a.qstart + b + 1), q0), a.num_tokens) - q0;
      heads = min(qall, a.max_new) * a.g;
      if (heads == 0) return;  // (in every workgroup of the pair)
    }
    // UNIFORM: the block ids of the chunk's two tiles; else those of the lane's row of each
    // load, and of token lane % 32 (for the scales).
    constexpr int NID = UNIFORM ? 2 : NI + 1;
    int ids[NID];
    // Clamped to the table's width only, so that ids need no length: a tile past the end
    // reads some block of the pool and what it reads is masked.
    auto load_ids = [&](int c) {
#pragma unroll
      for (int i = 0; i < NID; ++i) {
        if constexpr (UNIFORM) {
          const int at = min(2 * c + i, last_tile);
          ids[i] = load_uniform(btrow + (int64_t)(at / (BS / 16)) * bt_sk);
        } else {
          const int t = i < NI ? i * RPI + lrow : lane & 31;
          ids[i] = btrow[(int64_t)(min(c * kChunk + t, cap - 1) / bs) * bt_sk];
        }
      }
    };
    const int first = c0 + wave;
    load_ids(first);
    // Q^T operands: column = query head `row` of a kv head's group, elements in the order
    // of the K operands; of the scale's sign, so that the largest product has the largest
    // score.
    const f16 sign = a.scale_log2 < 0.f ? (f16)-1.f : (f16)1.f;
    f16x8 qf[NS][NC];
    int token[NS];  // MULTI: the column's token
#pragma unroll
    for (int st = 0; st < NS; ++st) {
      int64_t at;  // of the query row and head
      if constexpr (MULTI) {
        const int col = min(st * 16 + row, heads - 1);
        token[st] = col / a.g;
        at = (int64_t)(q0 + token[st]) * a.q_sb + (int64_t)(h0 * a.g + col - token[st] * a.g) * a.q_sh;
      } else {
        at = (int64_t)b * a.q_sb + (int64_t)((h0 + st) * a.g + min(row, a.g - 1)) * a.q_sh;
      }
#pragma unroll
      for (int s = 0; s < SEG; ++s)
#pragma unroll
        for (int f = 0; f < NF; ++f)
          qf[st][s * NF + f] =
              sign * *reinterpret_cast<const f16x8*>(a.q + at + s * 4 * FB + grp * FB + f * 8);
    }
    // Issues a chunk's loads. UNIFORM: its scales by one vector load (scalar ones would make
    // LDS reads wait for their misses), lane t + 2 hg + 4 (0: keys, 1: values) for tile t;
    // else lane (token, head) those of token lane % 32.
    float scales = 1.f, vscales = 1.f;
    auto issue = [&](int c) {
      auto block = [&](int id) { return (int64_t)min(max(id, 0), last_id); };
      if constexpr (UNIFORM) {
        const int id0 = ids[0], id1 = ids[1];
        scales = sbase[block(lane & 1 ? id1 : id0) * s_sb];
      } else {
        const int64_t id = block(ids[NID - 1]);
        scales = sbase[id * s_sb];
        vscales = a.vs[id * a.vs_sb + (h0 + shead) * a.vs_sh];
      }
      uint8_t* const to = s_stage + pinned(wave * STAGE);  // (nor are 2 NI places kept)
      auto load_rows = [&](const uint8_t* base, int64_t sb, int64_t st, int64_t sh, uint32_t plain,
                           uint32_t flip, uint8_t* to) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int64_t id = block(ids[UNIFORM ? i * RPI / 16 : i]);
          if constexpr (UNIFORM) {
            const int64_t off = (2 * c + i * RPI / 16) % (BS / 16) * 16 + i * RPI % 16;
            load_to_lds(tile_rsrc(base + id * sb + off * st, kAll), flipped(i) ? flip : plain,
                        to + i * 1024);
          } else {
            const int64_t off = (c * kChunk + i * RPI + lrow) % bs;
            const int p = piece(flipped(i) ? FLIP : 0);
            load_to_lds(base + id * sb + off * st + p / D * sh + p % D, to + i * 1024);
          }
        }
      };
      load_rows(kbase, k_sb, k_st, a.k_sh, k_lane, k_flip, to);
      load_rows(vbase, v_sb, v_st, a.v_sh, v_lane, v_flip, to + kChunk * RB);
    };

    if (!a.ranged) {
      L = clamped(load_uniform(a.lens + b));
      c1 = (L + kChunk - 1) / kChunk;
    }
    // The last position each column sees, and how many all of them see.
    int last[NS];
#pragma unroll
    for (int st = 0; st < NS; ++st) last[st] = MULTI ? L - qall + token[st] : L - 1;
    const int all_see = MULTI ? L - qall + 1 : L;
    float m_run[NS], l_run[NS];
    f32x4 acc[NS][ND];
#pragma unroll
    for (int st = 0; st < NS; ++st) {
      m_run[st] = kNegInf;
      l_run[st] = 0.f;
#pragma unroll
      for (int nd = 0; nd < ND; ++nd) acc[st][nd] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (first < c1) {
      issue(first);
      load_ids(first + NW);
    }
    const float scale = fabsf(a.scale_log2);
    for (int c = first; c < c1; c += NW) {
      const int t0 = c * kChunk;
      const bool whole = t0 + kChunk <= all_see;  // wavefront-uniform: the last may not be
      // The chunk has landed; all of it into registers. Tile t's score row m is token
      // 8 (m / 4) + 4 t + m % 4: lane (., grp) then gets the scores of tokens 8 grp .. + 7,
      // those of its V fragments.
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
      wave_lds_fence();
      frag kf[2][HG][SEG];
      uint2 vf[HG][ND];
      float kfs[2][HG];  // K scales of the lane's fragments
      float vfs[HG];     // V scale of the lane's tokens,
      f16x8 vft[HG];     // or one for each
      if constexpr (UNIFORM) {
#pragma unroll
        for (int hg = 0; hg < HG; ++hg) {
          // (A tile past the end has some block's scale: its codes are cleared below.)
          const float v0 = lane_value(scales, 2 * hg + 4);
          const float v1 = t0 + 16 < L ? lane_value(scales, 2 * hg + 5) : 1.f;
          vfs[hg] = grp < 2 ? v0 : v1;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            // Score rows 0 .. 7 of either are tokens of the block's first half.
            const float s0 = lane_value(scales, 2 * hg), s1 = lane_value(scales, 2 * hg + 1);
            kfs[t][hg] = row < 8 ? s0 : s1;
          }
        }
      } else {
        const int t = lane & 31, hg = HG > 1 ? lane >> 5 : 0;
        s_ks[wave][hg * kChunk + t] = scales;
        s_vs[wave][hg * kChunk + t] = (f16)(t0 + t < L ? power_of(vscales) : 1.f);
        wave_lds_fence();
      }
#pragma unroll
      for (int hg = 0; hg < HG; ++hg) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int r = 8 * (row >> 2) + 4 * t + (row & 3);
#pragma unroll
          for (int s = 0; s < SEG; ++s) {
            const int at = hg * D + s * 4 * FB + grp * FB;  // byte of the row
            kf[t][hg][s] = *reinterpret_cast<const frag*>(
                stage + r * RB + ((at / 16) ^ swizzle<NP>(r)) * 16 + at % 16);
          }
          if constexpr (!UNIFORM) kfs[t][hg] = s_ks[wave][hg * kChunk + r];
        }
        const int r = 8 * grp + (row >> 1);
        const uint8_t* vp = stage + kChunk * RB + r * RB + (row & 1) * 8;
#pragma unroll
        for (int nd = 0; nd < ND; ++nd)
          vf[hg][nd] = lds_read_tr8(vp + ((hg * ND + nd) ^ swizzle<NP>(r)) * 16);
        if constexpr (!UNIFORM)
          vft[hg] = *reinterpret_cast<const f16x8*>(&s_vs[wave][hg * kChunk + 8 * grp]);
      }
      wave_lds_fence();
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): nothing reads the LDS any more
      if (c + NW < c1) {
        issue(c + NW);
        load_ids(c + 2 * NW);
      }
      unsigned nan_lo = 0, nan_hi = 0;  // MULTI: bit 8 i + 7, token 8 grp + i has a NaN in V
      if (!whole) {
        // Codes of rows past the end as 0: 0 * what lies there is never NaN.
        const int n = L - t0 - 8 * grp;  // the lane's tokens that count
        const unsigned lo = n >= 4 ? ~0u : n <= 0 ? 0u : (1u << 8 * n) - 1;
        const unsigned hi = n >= 8 ? ~0u : n <= 4 ? 0u : (1u << 8 * (n - 4)) - 1;
#pragma unroll
        for (int hg = 0; hg < HG; ++hg)
#pragma unroll
          for (int nd = 0; nd < ND; ++nd) {
            vf[hg][nd].x &= lo;
            vf[hg][nd].y &= hi;
            if constexpr (MULTI) {
              // The top bit of every byte that holds 0x7f or 0xff.
              const unsigned x = ((vf[hg][nd].x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
              const unsigned y = ((vf[hg][nd].y & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
              nan_lo |= x;
              nan_hi |= y;
              vf[hg][nd].x &= ~((x >> 7) * 0xffu);
              vf[hg][nd].y &= ~((y >> 7) * 0xffu);
            }
          }
        if constexpr (MULTI) {
          nan_lo = or_over_row(nan_lo);
          nan_hi = or_over_row(nan_hi);
        }
      }
      // Every step for all blocks of columns: their chains of dependent instructions overlap.
      // (Block st is of head st, or all are of one head.)
      constexpr int CPH = MULTI ? NS : 1;  // blocks per head
      f32x4 s[NS][2];
#pragma unroll
      for (int hg = 0; hg < HG; ++hg)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int cb = 0; cb < CPH; ++cb) s[hg * CPH + cb][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < NC; ++i) {
            const frag& w = kf[t][hg][i / NF];
            const f16x8 kk = from_codes8(w[i % NF * 2], w[i % NF * 2 + 1], kfs[t][hg]);
#pragma unroll
            for (int cb = 0; cb < CPH; ++cb)
              s[hg * CPH + cb][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                  kk, qf[hg * CPH + cb][i], s[hg * CPH + cb][t], 0, 0, 0);
          }
        }
      auto unseen = [&](int st, int t, int r) { return t0 + 8 * grp + 4 * t + r > last[st]; };
      if (!whole) {
#pragma unroll
        for (int st = 0; st < NS; ++st)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (unseen(st, i / 4, i % 4)) s[st][i / 4][i % 4] = kNegInf;
      }
      float m_new[NS];
      bool grown = false;
#pragma unroll
      for (int st = 0; st < NS; ++st) {
        float m = s[st][0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) m = fmaxf(m, s[st][i / 4][i % 4]);
        m_new[st] = fmaxf(m_run[st], over_groups(m, Max()));
        grown |= m_new[st] > m_run[st];
      }
      if (__ballot(grown) != 0) {  // wavefront-uniform
#pragma unroll
        for (int st = 0; st < NS; ++st) {
          // (Nothing seen yet: 0, whatever the scale; 0 * -inf would be NaN.)
          const float alpha = m_new[st] == kNegInf ? 1.f
                              : m_run[st] == kNegInf ? 0.f
                                                     : fast_exp2((m_run[st] - m_new[st]) * scale);
          l_run[st] *= alpha;
#pragma unroll
          for (int nd = 0; nd < ND; ++nd) acc[st][nd] *= alpha;
          m_run[st] = m_new[st];
        }
      }
      f16x8 pb[NS];
#pragma unroll
      for (int st = 0; st < NS; ++st) {
        // (Scaled after the subtraction: products of many millions, which fp32 holds to some
        // units only, still give the largest one's probability.)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          pb[st][i] = (f16)fast_exp2(__builtin_fmaf(s[st][i / 4][i % 4] - m_run[st], scale, kBias));
      }
      if (!whole) {
#pragma unroll
        for (int st = 0; st < NS; ++st)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if constexpr (MULTI)
              if ((i / 4 ? nan_hi : nan_lo) >> (8 * (i % 4) + 7) & 1) pb[st][i] = (f16)__builtin_nanf("");
            if (unseen(st, i / 4, i % 4)) pb[st][i] = (f16)0.f;
          }
      }
#pragma unroll
      for (int st = 0; st < NS; ++st)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          l_run[st] = __builtin_amdgcn_fdot2(f16x2{pb[st][2 * i], pb[st][2 * i + 1]},
                                             f16x2{(f16)1.f, (f16)1.f}, l_run[st], false);
      // O^T += V^T P^T: operand index k = 8 grp + i stands for token 8 grp + i on both sides.
#pragma unroll
      for (int hg = 0; hg < HG; ++hg)
#pragma unroll
        for (int nd = 0; nd < ND; ++nd) {
          f16x8 av;
          if constexpr (UNIFORM)
            av = from_codes8(vf[hg][nd].x, vf[hg][nd].y, vfs[hg]);
          else
            av = from_codes8(vf[hg][nd].x, vf[hg][nd].y, 1.f) * vft[hg];
#pragma unroll
          for (int cb = 0; cb < CPH; ++cb)
            acc[hg * CPH + cb][nd] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                av, pb[hg * CPH + cb], acc[hg * CPH + cb][nd], 0, 0, 0);
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
    auto out_row = [&](int j) {  // of column j
      const int t = MULTI ? j / a.g : 0;
      return a.out + (int64_t)(q0 + t) * a.o_sb + (int64_t)(h0 * a.g + j - t * a.g) * a.o_sh;
    };
    float* my_acc = reinterpret_cast<float*>(stage);
#pragma unroll
    for (int st = 0; st < NS; ++st) {
      const float l = over_groups(l_run[st], Sum());
      if (grp == 0) {
        s_m[wave][st * 16 + row] = m_run[st] == kNegInf ? kNegInf : m_run[st] * scale;
        s_l[wave][st * 16 + row] = l;
      }
      if (MULTI ? st * 16 + row < heads : row < a.g) {
#pragma unroll
        for (int nd = 0; nd < ND; ++nd)
          *reinterpret_cast<f32x4*>(my_acc + (st * 16 + row) * D +
                                    ((nd * 4 + grp) ^ (row & 7)) * 4) = acc[st][nd];
      }
    }
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < heads * D4; i += kThreads) {
      const int j = i / D4;
      const int d = (i - j * D4) * 4;
      const int r = HG > 1 && j >= a.g ? 16 + j - a.g : j;  // row of the accumulators
      float M = s_m[0][r];
#pragma unroll
      for (int w = 1; w < NW; ++w) M = fmaxf(M, s_m[w][r]);
      float l = 0.f;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        // A state of no maximum holds zeros, or NaN that has to show.
        const float m = s_m[w][r];
        const float f = m == kNegInf ? 1.f : fast_exp2(m - M);
        l += f * s_l[w][r];
        o += f * *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(s_stage + w * STAGE) +
                                                 r * D + ((d >> 2) ^ (r & 7)) * 4);
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
    int* cnt = a.cnt + (int64_t)b * groups + h0 / HG;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_waitcnt(0);  // the record has landed before the arrival counts
    __syncthreads();
    if (tid == 0)
      s_last = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == nseg - 1;
    __syncthreads();
    if (!s_last) return;  // (the next segment writes s_last behind further barriers)
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");

    // Merge: every part's maxima and denominators into LDS (batches of parts, as many as
    // fit), their maximum, sum and shares per head by 16 lanes each, and the accumulators by
    // threads (item: head and four of its elements; the parts of an item are dealt over as
    // many threads as there are for it), U parts a round trip, the first ones on their way
    // before anything else. Part 0 lies apart from the others, which are two records apart.
    float* s_max = s_m[0];  // (the wavefronts' states are spent)
    float* s_sum = s_l[0];
    const int batch = min(nseg, (int)(sizeof(s_stage) / 8) / heads);
    float* s_pm = reinterpret_cast<float*>(s_stage);
    float* s_pl = s_pm + heads * batch;
    const int items = heads * D4;
    const int parts = items < kThreads ? kThreads / items : 1;
    const int part = parts > 1 ? tid / items : 0;
    const int step = 2 * a.rec_floats * 4;  // bytes from part i to part i + 1, i > 0
    // U parts a round trip, for each of IPT items of a thread.
    constexpr int IPT = MULTI && NW == 4 ? 4 : 1;
    constexpr int U = NW > 4 ? 8 : 16 / IPT;
    // Past the last part: zeros. (By the lane's offset, whole: a scalar offset's part in the
    // check against the resource's end is not specified.)
    auto fetch = [&](int i, int j, int d, f32x4 (&y)[U]) {
      const int at = (record(i) + j * D + d) * 4;
#pragma unroll
      for (int u = 0; u < U; ++u) y[u] = load_coherent16(rr, at + u * parts * step);
    };
    // (As above: no maximum, and so zeros or NaN.)
    auto share = [&](float m, float M) { return m == kNegInf ? 1.f : fast_exp2(m - M); };
    // Maximum and denominator i of parts [s0, s1): of head i / (s1 - s0).
    auto fetch_ml = [&](int i, int s0, int s1) {
      const int j = i / (s1 - s0);
      const int at = (record(s0 + i - j * (s1 - s0)) + heads * D + j) * 4;
      return float2{load_coherent4(rr, at), load_coherent4(rr, at + heads * 4)};
    };
    auto keep_ml = [&](int i, int s0, int s1, float2 ml) {
      const int j = i / (s1 - s0);
      s_pm[j * batch + i - j * (s1 - s0)] = ml.x;
      s_pl[j * batch + i - j * (s1 - s0)] = ml.y;
    };
    auto load_ml = [&](int from, int s0, int s1) {
#pragma unroll 1
      for (int i = from; i < heads * (s1 - s0); i += kThreads) keep_ml(i, s0, s1, fetch_ml(i, s0, s1));
    };
    // The first ones before the accumulators: maxima and sums are formed while those are on
    // their way (1 us of 24001 tokens, when it was added). Not where it costs spills: at one
    // token in workgroups of four (316 MB: 65.5 -> 69.2 in a graph).
    constexpr bool EARLY = MULTI || NW > 4;
    const int early = EARLY ? min(nseg, batch) : 0;
    float2 ml0 = {0.f, 0.f};
    if (tid < heads * early) ml0 = fetch_ml(tid, 0, early);
#pragma unroll 1
    for (int base = 0; base < items; base += IPT * kThreads) {  // workgroup-uniform
      bool live[IPT];
      int j[IPT], d[IPT];
      f32x4 y0[IPT], y[IPT][U];
#pragma unroll
      for (int k = 0; k < IPT; ++k) {
        if (base + k * kThreads >= items) {  // workgroup-uniform
          live[k] = false;
          continue;
        }
        const int item = parts > 1 ? tid - part * items : base + k * kThreads + tid;
        live[k] = part < parts && item < items;
        j[k] = live[k] ? item / D4 : 0;
        d[k] = live[k] ? (item - j[k] * D4) * 4 : 0;
        y0[k] = load_coherent16(rr, (j[k] * D + d[k]) * 4);
        fetch(1 + part, j[k], d[k], y[k]);
      }
      if (base == 0) {
#pragma unroll 1
        for (int s0 = 0; s0 < nseg; s0 += batch) {
          const int s1 = min(nseg, s0 + batch);
          if (s0) __syncthreads();
          if (s0 == 0 && tid < heads * early) keep_ml(tid, 0, early, ml0);
          load_ml(s0 || !EARLY ? tid : tid + kThreads, s0, s1);
          __syncthreads();
#pragma unroll 1
          for (int jj = tid / 16; jj < heads; jj += kThreads / 16) {
            const float had = s0 ? s_max[jj] : kNegInf;
            float M = had;
            for (int i = row; i < s1 - s0; i += 16) M = fmaxf(M, s_pm[jj * batch + i]);
            M = over_row(M, Max());
            float sum = 0.f;
            for (int i = row; i < s1 - s0; i += 16) {
              const float f = share(s_pm[jj * batch + i], M);
              sum += s_pl[jj * batch + i] * f;
              s_pm[jj * batch + i] = f;
            }
            sum = over_row(sum, Sum());
            if (s0) sum += s_sum[jj] * share(had, M);
            if (row == 0) {
              s_max[jj] = M;
              s_sum[jj] = sum;
            }
          }
        }
        __syncthreads();
      }
      f32x4 o[IPT];
#pragma unroll
      for (int k = 0; k < IPT; ++k) o[k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int s0 = 0; s0 < nseg; s0 += batch) {
        const int s1 = min(nseg, s0 + batch);
        if (batch < nseg) {  // the batch's shares, of the maxima over all batches
          __syncthreads();
          load_ml(tid, s0, s1);
          __syncthreads();
          for (int i = tid; i < heads * (s1 - s0); i += kThreads) {
            const int j = i / (s1 - s0);
            float& x = s_pm[j * batch + i - j * (s1 - s0)];
            x = share(x, s_max[j]);
          }
          __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < IPT; ++k) {
          if (!live[k]) continue;
          const float* pm = s_pm + j[k] * batch - s0;
          if (s0 == 0 && part == 0) o[k] += pm[0] * y0[k];
#pragma unroll 1
          for (int i = s0 ? s0 + part : 1 + part; i < s1; i += U * parts) {
            if (i != 1 + part) fetch(i, j[k], d[k], y[k]);
#pragma unroll
            for (int u = 0; u < U; ++u)
              if (i + u * parts < s1) o[k] += pm[i + u * parts] * y[k][u];
          }
        }
      }
      if (parts > 1) {
        s_part[tid] = o[0];
        __syncthreads();
        if (part == 0)
          for (int p = 1; p < parts; ++p) o[0] += s_part[tid + p * items];
      }
#pragma unroll
      for (int k = 0; k < IPT; ++k) {
        if (!live[k] || part != 0) continue;
        const float sum = s_sum[j[k]];
        const float inv = sum == 0.f ? 0.f : 1.f / sum;  // 0: no key at all
        f16x4 z;
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = (f16)(o[k][e] * inv);
        *reinterpret_cast<f16x4*>(out_row(j[k]) + d[k]) = z;
      }
    }
    if (tid == 0) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
  };

  // This workgroup's part of the list: positions [x0, x1); `at` is the first of sequence b.
  Cut ranges{0, 0};
  int x0 = 0, x1 = 0, at = 0, b = 0, g0 = 0, w = 0;
  // Lengths of 256 sequences a time, sequence base + 64 k + lane in lens[k]: read together.
  constexpr int LK = 4;
  int lens[LK] = {0, 0, 0, 0}, own[LK], incl[LK];
  if (a.ranged) {
    // Each sequence takes groups x (its chunks + pair_cost) positions. (The host sees to it
    // that 31 bits hold their sum.)
    auto take = [&](int base) {
#pragma unroll
      for (int k = 0; k < LK; ++k) lens[k] = a.lens[min(base + 64 * k + lane, a.num_seqs - 1)];
#pragma unroll
      for (int k = 0; k < LK; ++k) {
        lens[k] = clamped(lens[k]);
        own[k] = base + 64 * k + lane < a.num_seqs ? groups * (chunks_of(lens[k]) + a.pair_cost) : 0;
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
    w = xcd_order(blockIdx.x, G);
    ranges = Cut{T / G, T % G};
    x0 = ranges.start(w);
    x1 = ranges.start(w + 1);
    // The sequence that holds x0, and its first position.
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
  } else {
    const int pair = xcd_order(blockIdx.x, gridDim.x);
    b = pair / groups;
    g0 = pair - b * groups;
  }
  for (;;) {
    int L = 0;
    if (a.ranged && a.num_seqs <= 64 * LK) {
#pragma unroll
      for (int k = 0; k < LK; ++k)
        if (b / 64 == k) L = __builtin_amdgcn_readlane(lens[k], b % 64);
    } else if (a.ranged) {
      L = clamped(load_uniform(a.lens + b));
    }
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
      c0 = max(0, min(n, x0 - at - a.pair_cost));
      c1 = max(0, min(n, x1 - at - a.pair_cost));
      // The ranges that hold chunks of it (of no chunks: the one that holds its start).
      w0 = ranges.of(at + (n ? a.pair_cost : 0));
      w1 = n ? ranges.of(at + span - 1) : w0;
      at += span;
    }
    if (w >= w0 && w <= w1) segment(b, g0 * HG, L, c0, c1, w0, w - w0, w1 - w0 + 1);
    if (!a.ranged || at >= x1) return;
    if (++g0 == groups) {
      g0 = 0;
      if (++b == a.num_seqs) return;
    }
  }
}

// ---- launch plan, shared by the two sources that launch the kernel ----

// List positions of 32 tokens: what a pair costs beside its chunks (its beginning, meeting,
// arrival and merge), and the fewest a range takes. Measured on MI355X at 8 / 16 / 32: the
// cost, 256 x ~4.6k tokens 62.3 / 62.3 / 64.8 us, 16 x 5 drafts 31.7 / 31.2 / 32.8, 20 x 4
// drafts at head_dim 64 15.6 / 13.4 / 13.3, 64 x 5 drafts of up to 4k 72.5 / 76.9 / 76.9; the
// range, one sequence of 24001 tokens 15.1 / 13.3 / 14.4, 8 of 1k to 8k 22.6 / 22.8 / 22.5.
constexpr int kPairCost = 16;
constexpr int kMinRange = 16;
// Tables of at most this many tokens take one workgroup per pair; of the second, where
// the pairs fill at least half the compute units. Whole pairs against ranges, measured: 8 x
// 1024 tokens at 32 / 8 heads 12.5 against 13.5 us, 8 x 2k 20.1 against 14.3; at 14 / 2 heads
// 128 x 1088 10.6 against 16.8, 64 x 2k 14.0 against 16.0, 512 x 2k 34.4 against 40.1; 64 x 5
// drafts of up to 4k 79.6 against 76.8.
constexpr int kWholePairs = 1024;
constexpr int kWholePairsBusy = 2048;

struct DecodePlan {
  int head_group, waves, ranged, grid, rec_floats;
  size_t ws_bytes;

  // The launch's part of the arguments.
  void fill(DecodeFp8Args& a, void* workspace) const {
    a.cnt = (int*)workspace;
    a.recs = (float*)((char*)workspace + (ws_bytes ? kCounterBytes : 0));
    a.ranged = ranged;
    a.min_range = kMinRange;
    a.pair_cost = kPairCost;
    a.rec_floats = rec_floats;
  }
};

// For the form of up to new_tokens query tokens per sequence, or 0: the one-token form.
DecodePlan decode_plan(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim,
                       int block_size, int max_blocks, int new_tokens);

// Whether the uniform tiles' loads, which take 31-bit offsets within 16 rows of two heads,
// serve these strides.
inline bool near_strides(const DecodeFp8Args& a) {
  const int64_t most = 1 << 26;
  return a.k_st < most && a.v_st < most && a.k_sh < most && a.v_sh < most;
}

}  // namespace fp8
}  // namespace pa
