// Sampling from logits: temperature, top-k, top-p and min-p, by given random numbers (gfx950).
//
// A row's weights are w = exp((z - max z) / T). Its entries are ordered by z, largest first,
// equal ones by index; the first top_k stay, of them the shortest beginning that weighs
// top_p of their sum, of those the ones with w >= min_p. The token is the first index whose
// cumulative kept weight exceeds u times the sum; or the row of probabilities is written.
//
// A row is read once, in pieces of 1024 entries by wavefronts of several workgroups: the
// maximum of each cell of 128 entries, of each piece, and where the settings need the whole
// sum, the piece's sum of weights go to the workspace. The last of the row's workgroups to
// arrive decides. It does not sort. The cells' maxima give a lower bound on what can be
// kept: for top-k, the k-th largest of them (k entries at least reach it); for min-p its
// own logit; for top-p, entries below (1 - p) / vocab of the sum, which together weigh less
// than 1 - p. Only cells that reach the bound are read again, and their entries above it
// listed: tens to hundreds for usual settings. A short list is ranked by comparing all
// with all; a longer one by radix passes over the logits' bits with counts and weights.
// Where more are listed than fit LDS (flat distributions), two more launches share the row
// among workgroups. The first counts entries and adds up their places per interval of logits,
// without weighing one: an interval's weight is at least that of its number at their mean
// (the exponential is convex) and at most that of as many on the chord over it, which brackets
// the border to an interval or two. The second sums the weights above the bracket per piece and
// lists what lies in it, and the last of its workgroups decides. Lists beyond their room (equal
// logits) have the row done by one workgroup alone, narrowing by intervals of logits and by
// their bits. (Rows without such a list leave these launches at once.)
//
// Weights and sums. w is computed in 64 bits (2^-45 relative) and summed as whole numbers of
// 2^-44: sums do not depend on the order, so that LDS atomics may form them, and the 2^19
// entries that a row may have cannot overflow 64 bits. (Sums of whole pieces, formed while
// the row is read, are in 64-bit floating point in a fixed order.) The token differs from the
// definition's only where u times the sum lies within about 2^-44 per entry of a border.
//
// What bounds it: for many rows the 64-bit arithmetic of the weights, for one row the chain of
// dependent steps. In a run of calls on MI355X: one fp16 row of 151936 with temperature, top-k
// and top-p 17 us (12-14 the first launch, 2 each of the others, which find nothing to do); 256
// rows of mixed settings 99 (45 + 18 + 40 under the profiler; a copy of the logits would take 15); 32
// bf16 rows of 100003 at high temperatures and wide top-p 55.7; probabilities of 80 rows of 151936
// 77, of which writing 16 (4.5 TB/s).
#include "../../include/paged_attention.h"
#include "pa_tiles.h"

namespace pa {
namespace sample {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kPiece = 1024;  // entries of a wavefront's step, 16 per lane
constexpr int kCell = 128;    // entries of 16 lanes, eight each
constexpr int kMaxVocab = 1 << 19;
constexpr int kMaxPieces = kMaxVocab / kPiece;
constexpr int kMaxCells = kMaxVocab / kCell;
// The workspace starts with one arrival counter per row, at the same place for every call.
constexpr int kMaxRows = 16384;
constexpr size_t kCounterBytes = (size_t)kMaxRows * sizeof(int);
constexpr int kList = 2048;   // listed entries
constexpr int kShort = 512;   // of them, ranked by comparing all with all: one per thread
constexpr int kCellBins = 512;
constexpr int kBins = 2048;
constexpr int kRoom = 2048;  // words of a shared row's room
static_assert(kRoom >= kBins && kRoom >= kList, "counts, then the list");
// Pieces that a workgroup looks through by itself, though most of them reach the bound.
constexpr int kAlonePieces = 32;
constexpr int kMaxShared = 2048;  // rows with room to be shared by
constexpr uint32_t kDead = 0x007fffffu;  // order key of -inf; NaN counts as -inf
constexpr double kUnit = 17592186044416.0;  // 2^44

// What the deciding workgroup leaves for the launch that writes probabilities.
typedef unsigned long long u64;

struct Decision {
  float max;
  uint32_t key;   // kept: order keys above this one,
  int last;       // or equal to it up to this index
  float min_p;
  double c;       // log2(e) / T
  double sum;
};

struct Piece {
  float max, pad;
  double sum;  // (of a shared row in the end: the kept weight, in units)
};

// A row whose list does not fit, between the launches.
enum { kDecided = 0, kCount = 1, kShare = 2, kKeepAll = 3, kAlone = 4 };
struct alignas(16) Shared_row {
  float max;
  uint32_t floor;     // keys below are out of the question
  float lo, scale;    // the intervals of the logits' line,
  int first, end;     // and those of the bracket
  int pad[2];
  u64 counts;         // entries in the bracket (listed), and 2^32 times those above it
  u64 aim, whole;
};

struct Args {
  const void* logits;
  int64_t s_seq, s_row;  // elements from sequence to sequence and row to row
  int rows, each, vocab;
  const float* temperature;  // per sequence, or null: t_all
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  float t_all, p_all, m_all;
  int k_all;
  const float* u;  // per row, strides; null: decisions for the probabilities
  int64_t u_seq, u_row;
  int64_t* tokens;
  float* probs;
  int* cnt;
  int* modes;     // per row: of the Shared_row
  char* records;  // per row: Decision, Shared_row, pieces, cells
  u64* rooms;     // of the first `shared_rows` rows: kBins counts and places, then kList keys and indexes
  int row_bytes, pieces, cells, groups;
  int shared_rows, shared_groups, cus;
};

constexpr int kHead = sizeof(Decision) + sizeof(Shared_row);
static_assert(sizeof(Decision) % 16 == 0 && sizeof(Shared_row) % 16 == 0, "16-byte reads behind them");
__host__ __device__ inline int row_record(int pieces, int cells) {
  return kHead + pieces * (int)sizeof(Piece) + (cells + 3) / 4 * 16;
}

// ---- entries -----------------------------------------------------------------------

// Logits in memory at any alignment of their own.
struct Half {
  typedef uint16_t E;
  static constexpr E kLow = 0xfc00;  // -inf
  __device__ static float get(E x) { return (float)__builtin_bit_cast(f16, x); }
};
struct Brain {
  typedef uint16_t E;
  static constexpr E kLow = 0xff80;
  __device__ static float get(E x) { return __builtin_bit_cast(float, (uint32_t)x << 16); }
};
struct Single {
  typedef uint32_t E;
  static constexpr E kLow = 0xff800000u;
  __device__ static float get(E x) { return __builtin_bit_cast(float, x); }
};

// Eight entries as they lie in memory; the floats they stand for, NaN as -inf.
template <typename T>
struct Eight {
  typedef typename T::E E;
  typedef E words __attribute__((ext_vector_type(8), aligned(sizeof(E))));
  words w;

  // Entries v0 .. v0 + 7 of a row of eight and more. A lane whose entries reach past the end
  // gets the row's last eight, those before v0 as -inf, and is told where they begin.
  __device__ __forceinline__ int load(const E* row, int v0, int vocab) {
    const int at = min(v0, vocab - 8);
    w = *reinterpret_cast<const words*>(row + at);
    if (at != v0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = at + i < v0 ? T::kLow : w[i];
    }
    return at;
  }
  __device__ __forceinline__ float operator[](int i) const { return fmaxf(T::get(w[i]), kNegInf); }
  __device__ __forceinline__ float raw(int i) const { return T::get(w[i]); }  // NaN as it is
};

// Unsigned numbers in the logits' order; both zeros are one.
__device__ inline uint32_t order_key(float z) {
  const uint32_t b = __builtin_bit_cast(uint32_t, z + 0.f);
  return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ inline float of_key(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// 2^d for -1000 <= d <= 0, to 2^-45 relative: the whole part, by an addition that leaves it in
// the low bits, goes to the exponent; the rest by the polynomial through 2^f at the ten Chebyshev
// nodes of [-1/2, 1/2], its constant rounded to 1: the largest weighs exactly that.
// N of them step by step, so that their chains of dependent instructions overlap (one after
// the other, as the compiler orders them by itself, a pass over flat rows took 100 us where it
// takes 94).
template <int N>
__device__ inline void exp2_of(double (&d)[N]) {
  constexpr double kWhole = 6755399441055744.0;  // 1.5 * 2^52
  constexpr double kC[9] = {1.3259945262689143e-06, 1.5252640059770786e-05, 0.00015403432339553542,
                            0.001333355825801874,   0.009618129195951041,   0.05550410866428854,
                            0.24022650695631514,    0.6931471805599526,     1.0};
  int n[N];
  double p[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const double t = d[e] + kWhole;
    n[e] = (int)__builtin_bit_cast(uint2, t).x;
    d[e] -= t - kWhole;
    p[e] = 1.0212097549811005e-07;
  }
#pragma unroll
  for (int i = 0; i < 9; ++i) {
#pragma unroll
    for (int e = 0; e < N; ++e) p[e] = __builtin_fma(p[e], d[e], kC[i]);
    if constexpr (N > 1) __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int e = 0; e < N; ++e) {
    uint2 b = __builtin_bit_cast(uint2, p[e]);
    asm("v_lshl_add_u32 %0, %1, 20, %0" : "+v"(b.y) : "v"(n[e]));  // (the 64-bit sum takes five)
    d[e] = __builtin_bit_cast(double, b);
  }
}
__device__ inline double exp2_of(double d) {
  double x[1] = {d};
  exp2_of(x);
  return x[0];
}

// The weight of z next to a maximum m: 2^(c (z - m)), c = log2(e) / T; as good as 0 from 2^-1000
// down and for z = -inf. Where m is +inf the entries of +inf alone count: they are told by
// comparing, and weigh 1.
struct Scale {
  double m, c, low;
  bool top_only;
  __device__ Scale() {}
  __device__ Scale(float max, double per_logit) {
    top_only = max == -kNegInf;
    m = top_only ? 0.0 : (double)max;
    c = top_only ? 0.0 : per_logit;
    low = top_only ? 0.0 : -1000.0;
  }
  __device__ double weight(float z) const { return exp2_of(fmax(((double)z - m) * c, low)); }
  template <int N>
  __device__ void weights(const float (&z)[N], double (&w)[N]) const {
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = fmax(((double)z[e] - m) * c, low);
    exp2_of(w);
  }
};
__device__ inline u64 units(double w) { return (u64)(w * kUnit + 0.5); }
// The same for w up to 1, by an addition that leaves the rounded number in the low bits (half a
// unit counts as none).
__device__ inline u64 units1(double w) {
  return __builtin_bit_cast(u64, __builtin_fma(w, kUnit, 4503599627370496.0)) & 0xfffffffffffffull;
}
// The sum of units1 over an array's chosen entries: of those numbers as they are, then without
// what is in the high bits of each.
template <typename F>
__device__ __forceinline__ u64 sum_units1(const double (&w)[8], F chosen) {
  u64 x = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    x += __builtin_bit_cast(u64, __builtin_fma(chosen(i) ? w[i] : 0.0, kUnit, 4503599627370496.0));
  return x - 8 * 0x4330000000000000ull;
}

// ---- sums over lanes ---------------------------------------------------------------

template <int CTRL>
__device__ inline double row_lane(double x) {
  const uint2 v = __builtin_bit_cast(uint2, x);
  return __builtin_bit_cast(
      double, make_uint2((unsigned)__builtin_amdgcn_update_dpp(0, (int)v.x, CTRL, 0xf, 0xf, false),
                         (unsigned)__builtin_amdgcn_update_dpp(0, (int)v.y, CTRL, 0xf, 0xf, false)));
}
template <int CTRL>
__device__ inline u64 row_lane(u64 x) {
  return __builtin_bit_cast(u64, row_lane<CTRL>(__builtin_bit_cast(double, x)));
}
template <typename X>
__device__ inline X lane_of(X x, int l) {  // of 64 bits, l uniform
  const uint2 v = __builtin_bit_cast(uint2, x);
  return __builtin_bit_cast(X, make_uint2((unsigned)__builtin_amdgcn_readlane((int)v.x, l),
                                          (unsigned)__builtin_amdgcn_readlane((int)v.y, l)));
}
// Over a wavefront, in every lane: rotations within rows of 16, then the rows.
template <typename X>
__device__ inline X wave_sum(X x) {
  x += row_lane<0x128>(x);
  x += row_lane<0x124>(x);
  x += row_lane<0x122>(x);
  x += row_lane<0x121>(x);
  return (lane_of(x, 0) + lane_of(x, 16)) + (lane_of(x, 32) + lane_of(x, 48));
}
// Over the lanes up to each.
__device__ inline u64 wave_scan(u64 x, int lane) {
  x += row_lane<0x111>(x);
  x += row_lane<0x112>(x);
  x += row_lane<0x114>(x);
  x += row_lane<0x118>(x);
  const u64 r0 = lane_of(x, 15), r1 = lane_of(x, 31), r2 = lane_of(x, 47);
  return x + (lane < 16 ? 0 : lane < 32 ? r0 : lane < 48 ? r0 + r1 : r0 + r1 + r2);
}
// Maximum over rows of 16 lanes, in all of them.
__device__ inline float row_max(float x) {
  auto turned = [](float v, auto by) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v),
                                                                 0x120 + decltype(by)::value, 0xf,
                                                                 0xf, false));
  };
  x = fmaxf(x, turned(x, std::integral_constant<int, 8>()));
  x = fmaxf(x, turned(x, std::integral_constant<int, 4>()));
  x = fmaxf(x, turned(x, std::integral_constant<int, 2>()));
  return fmaxf(x, turned(x, std::integral_constant<int, 1>()));
}
__device__ inline float wave_max_of_rows(float x) {  // x: equal within rows of 16
  auto at = [&](int l) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), l));
  };
  return fmaxf(fmaxf(at(0), at(16)), fmaxf(at(32), at(48)));
}

// ---- settings ----------------------------------------------------------------------

struct Settings {
  double c;      // log2(e) / T
  int k;         // entries that top-k keeps, 0: all
  float p;       // top-p, 1: off
  float min_p;   // 0: off
  bool whole;    // the sum over all entries is needed
  bool filtered;
};

__device__ inline Settings settings_of(const Args& a, int seq) {
  Settings s;
  const float t = a.temperature ? a.temperature[seq] : a.t_all;
  s.k = a.top_k ? a.top_k[seq] : a.k_all;
  s.p = a.top_p ? a.top_p[seq] : a.p_all;
  s.min_p = a.min_p ? a.min_p[seq] : a.m_all;
  if (s.k <= 0 || s.k >= a.vocab) s.k = 0;
  if (!(s.p < 1.f)) s.p = 1.f;
  s.min_p = s.min_p > 0.f ? fminf(s.min_p, 1.f) : 0.f;
  if (!(t > 0.f)) {  // greedy: the first of the largest
    s.c = 1.0;
    s.k = 1;
    s.p = 1.f;
    s.min_p = 0.f;
  } else {
    s.c = 1.4426950408889634 / (double)t;
    if (s.p <= 0.f) {  // the first alone, too
      s.k = 1;
      s.p = 1.f;
    }
  }
  s.filtered = s.k > 0 || s.p < 1.f || s.min_p > 0.f;
  s.whole = !s.filtered || (s.k == 0 && s.p < 1.f);
  return s;
}

// ---- the deciding workgroup ---------------------------------------------------------

struct Shared {
  uint32_t key[kList];
  int idx[kList];
  union {
    struct {
      u64 w[kBins];
      uint32_t n[kBins];
    } bin;
    uint16_t cells[kMaxCells];
    struct {
      ulonglong2 entry[kShort];  // order or index, weight
      u64 more[kShort / 2];
    } brief;
  };
  u64 psum[kMaxPieces];
  int pcount[kMaxPieces];
  u64 part[kWaves];
  int part_n[kWaves];
  int count;
  uint32_t found_key;
  int found, found2;
  u64 found_w;
};

// The entries that are still in question: those in interval `bin` of the logits' line (of
// scale 0: all are in interval 0), with these leading bits of their key. What lies above is
// kept for sure.
struct Range {
  uint32_t floor;  // keys below are out of the question
  float lo, scale;
  int bin;
  uint32_t mask, bits;
  __device__ int bin_of(float z) const {
    const float t = (z - lo) * scale;
    return t > 0.f ? (t < (float)(kBins - 1) ? (int)t : kBins - 1) : 0;
  }
  // 0: no, 1: in question, 2: kept
  __device__ int place(float z, uint32_t key) const {
    if (key < floor) return 0;
    const int b = bin_of(z);
    if (b != bin) return b > bin ? 2 : 0;
    const uint32_t x = key & mask;
    return x == bits ? 1 : x > bits ? 2 : 0;
  }
};

template <typename T>
struct Decider {
  typedef typename T::E E;
  const Args& a;
  Shared& sh;
  const E* row;
  Settings s;
  int tid, lane, wave;
  float m = kNegInf;      // the row's maximum
  Scale sc;               // and its weights
  int listed_cells = -1;  // -1: all pieces are read

  __device__ Decider(const Args& a_, Shared& sh_, const E* row_, const Settings& s_, int tid_, int lane_,
                     int wave_)
      : a(a_), sh(sh_), row(row_), s(s_), tid(tid_), lane(lane_), wave(wave_) {}
  __device__ __forceinline__ void set_max(float x) {
    m = x;
    sc = Scale(x, s.c);
  }

  // f(x, v0) for entries v0 .. v0 + 7 of every lane, by whole wavefronts: 512 entries a time,
  // kAhead times read before the first is looked at.
  static constexpr int kAhead = 4;
  template <typename F>
  __device__ __forceinline__ void each_entry(F f) {
    const bool dense = listed_cells < 0;
    const int steps = dense ? (a.vocab + 511) / 512 : (listed_cells + 3) / 4;
    for (int i0 = wave; i0 < steps; i0 += kWaves * kAhead) {  // wavefront-uniform
      Eight<T> x[kAhead];
      int v0[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int i = i0 + j * kWaves;
        v0[j] = a.vocab;
        if (dense)
          v0[j] = i * 512 + lane * 8;
        else if (i * 4 + (lane >> 4) < listed_cells)
          v0[j] = (int)sh.cells[i * 4 + (lane >> 4)] * kCell + (lane & 15) * 8;
        if (i < steps) v0[j] = x[j].load(row, v0[j], a.vocab);
      }
      // (One copy of f's code.)
#pragma unroll 1
      for (int j = 0; j < kAhead && i0 + j * kWaves < steps; ++j) {
        Eight<T> y;
        int v;
        switch (j) {
          case 0: y = x[0], v = v0[0]; break;
          case 1: y = x[1], v = v0[1]; break;
          case 2: y = x[2], v = v0[2]; break;
          default: y = x[3], v = v0[3]; break;
        }
        f(y, v);
      }
    }
  }

  // Sum over the workgroup, in every thread.
  __device__ __forceinline__ u64 block_sum(u64 x) {
    x = wave_sum(x);
    __syncthreads();
    if (lane == 0) sh.part[wave] = x;
    __syncthreads();
    u64 t = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) t += sh.part[i];
    return t;
  }

  __device__ __forceinline__ float block_max(float x) {
    x = wave_max_of_rows(row_max(x));
    __syncthreads();
    if (lane == 0) sh.part[wave] = (u64)__builtin_bit_cast(uint32_t, x);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) x = fmaxf(x, __builtin_bit_cast(float, (uint32_t)sh.part[i]));
    return x;
  }

  // The cells' maxima, eight per thread: cell (j * kThreads + tid) * 4 + i at [j * 4 + i].
  static constexpr int kCells = kMaxCells / kThreads;
  static_assert(kCells == 8, "two loads of four per thread");
  float cell[kCells];
  __device__ __forceinline__ int cell_of(int i) const { return (i / 4 * kThreads + tid) * 4 + i % 4; }
  __device__ __forceinline__ void load_cells(const __amdgpu_buffer_rsrc_t& rc) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f32x4 y = {kNegInf, kNegInf, kNegInf, kNegInf};
      if (j * kThreads * 4 < a.cells)  // uniform
        y = tiles::load_coherent16(rc, (j * kThreads + tid) * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) cell[j * 4 + i] = cell_of(j * 4 + i) < a.cells ? y[i] : kNegInf;
    }
  }

  // A key that the k-th largest entry has at least: the k-th largest of the cells' maxima, to a
  // bin of their range.
  __device__ __forceinline__ uint32_t cell_bound(int k) {
    float low = -kNegInf;
#pragma unroll
    for (int i = 0; i < kCells; ++i)
      if (cell[i] != kNegInf) low = fminf(low, cell[i]);
    low = -block_max(-low);
    const float width = m - low;
    if (!(width > 0.f && width < 3e38f)) return 0;
    const float scale = (float)kCellBins / width;
    auto bin = [&](float z) { return min((int)((z - low) * scale), kCellBins - 1); };
    for (int i = tid; i < kCellBins; i += kThreads) {
      sh.bin.n[i] = 0;
      sh.bin.w[i] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kCells; ++i)
      if (cell[i] != kNegInf) atomicAdd(&sh.bin.n[bin(cell[i])], 1u);
    walk_bins<kCellBins>(0, 0, k, ~0ull);
    const int b = sh.found;
    __syncthreads();
    if (b < 0) return 0;  // fewer cells than k
    return order_key(low + (float)b / scale - 1e-6f * (fabsf(low) + fabsf(m)));
  }

  // Lists the cells whose maximum reaches the bound; whether few enough are listed.
  __device__ __forceinline__ bool list_cells(uint32_t floor) {
    if (tid == 0) sh.count = 0;
    __syncthreads();
    unsigned in = 0;
#pragma unroll
    for (int i = 0; i < kCells; ++i) in |= (unsigned)(order_key(cell[i]) >= floor) << i;
    const int mine = __builtin_popcount(in);
    const int incl = tiles::wave_incl_scan(mine);
    int at = 0;
    if (lane == 63 && incl) at = atomicAdd(&sh.count, incl);
    at = __builtin_amdgcn_readlane(at, 63) + incl - mine;
#pragma unroll
    for (int i = 0; i < kCells; ++i)
      if (in >> i & 1) sh.cells[at++] = (uint16_t)cell_of(i);
    __syncthreads();
    const int n = sh.count;
    __syncthreads();
    listed_cells = n;
    return n * 4 <= a.cells || a.cells <= 64;
  }

  // Lists the entries in question; how many there are (more than kList: not all listed).
  __device__ __forceinline__ int list_entries(const Range& r) {
    if (tid == 0) sh.count = 0;
    __syncthreads();
    each_entry([&](const Eight<T>& x, int v0) __attribute__((always_inline)) {
      unsigned in = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) in |= (unsigned)(r.place(x[i], order_key(x[i])) == 1) << i;
      if (__ballot(in != 0) == 0) return;
      const int mine = __builtin_popcount(in);
      const int incl = tiles::wave_incl_scan(mine);
      int at = 0;
      if (lane == 63) at = atomicAdd(&sh.count, incl);
      at = __builtin_amdgcn_readlane(at, 63) + incl - mine;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (in >> i & 1) {
          if (at < kList) {
            sh.key[at] = order_key(x[i]);
            sh.idx[at] = v0 + i;
          }
          ++at;
        }
    });
    __syncthreads();
    const int n = sh.count;
    __syncthreads();
    return n;
  }

  // Of the bins' counts and weights, from the last bin down: the first at which k entries
  // or a weight of `aim` are reached, in sh.found (-1: none), and what lies above it (then:
  // all) in sh.found2 and sh.found_w. (k 0 or aim ~0: no such limit.)
  // BINS: each thread BINS / kThreads neighbouring ones, the last threads the first bins.
  template <int BINS>
  __device__ __forceinline__ void walk_bins(int have, u64 have_w, int k, u64 aim) {
    constexpr int PER = BINS > kThreads ? BINS / kThreads : 1;
    static_assert(PER * kThreads >= BINS && BINS % 64 == 0, "whole wavefronts of bins");
    __syncthreads();
    const int b0 = BINS - 1 - tid * PER;  // and down from there
    const bool live = tid * PER < BINS;
    int own[PER], mine = 0;
    u64 own_w[PER], mine_w = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      mine += own[i] = live ? (int)sh.bin.n[b0 - i] : 0;
      mine_w += own_w[i] = live ? sh.bin.w[b0 - i] : 0;
    }
    const int incl = tiles::wave_incl_scan(mine);
    const u64 incl_w = wave_scan(mine_w, lane);
    if (lane == 63) {
      sh.part[wave] = incl_w;
      sh.part_n[wave] = incl;
    }
    if (tid == 0) sh.found = 0x7fffffff;
    __syncthreads();
    int sum = have + incl - mine;
    u64 sum_w = have_w + incl_w - mine_w;
    int all = have;
    u64 all_w = have_w;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if (i < wave) {
        sum += sh.part_n[i];
        sum_w += sh.part[i];
      }
      all += sh.part_n[i];
      all_w += sh.part[i];
    }
    int hit = -1, before = 0;
    u64 before_w = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (hit < 0 && own[i] > 0 && ((k > 0 && sum + own[i] >= k) || sum_w + own_w[i] >= aim)) {
        hit = b0 - i;
        before = sum;
        before_w = sum_w;
      }
      sum += own[i];
      sum_w += own_w[i];
    }
    const uint64_t hits = __ballot(hit >= 0);
    if (hits && lane == (int)__builtin_ctzll(hits)) atomicMin(&sh.found, tid);
    __syncthreads();
    const int first = sh.found;
    __syncthreads();
    if (tid == (first == 0x7fffffff ? 0 : first)) {
      sh.found = hit;
      sh.found2 = hit < 0 ? all : before;
      sh.found_w = hit < 0 ? all_w : before_w;
    }
    __syncthreads();
  }

  // Where the kept ones end: keys above `key`, and of those equal to it `ties`; `count` and
  // `w` of the entries above it. ties -1: everything down to the bound is kept.
  struct Cut {
    uint32_t key;
    int ties, all;  // kept ones of that key, and all of it
    int above;
    u64 above_w;
    Range range;    // in which the listed entries lie (narrowed where they did not fit)
    bool in_list;   // the entries of range are listed
    int n;
  };

  // Where the kept ones end: the first k entries (0: no such limit), or the shortest beginning
  // that weighs aim, of what c.range and c.above stand for, all c.n entries in question listed.
  __device__ __forceinline__ void cut_list(Cut& c, int k, u64 aim) {
    c.in_list = true;
    // Radix passes over the list.
    uint32_t prefix = 0;
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kThreads) {
        sh.bin.n[i] = 0;
        sh.bin.w[i] = 0;
      }
      __syncthreads();
#pragma unroll 1
      for (int i = tid; i < c.n; i += kThreads) {
        const uint32_t key = sh.key[i];
        if (shift == 24 || key >> (shift + 8) == prefix) {
          atomicAdd(&sh.bin.n[key >> shift & 255], 1u);
          atomicAdd(&sh.bin.w[key >> shift & 255], units1(sc.weight(of_key(key))));
        }
      }
      walk_bins<256>(c.above, c.above_w, k, aim);
      if (sh.found < 0) {  // the limit is not reached (in the first pass, if at all)
        keep_all(c);
        __syncthreads();
        return;
      }
      prefix = prefix << 8 | (uint32_t)sh.found;
      c.above = sh.found2;
      c.above_w = sh.found_w;
      c.all = (int)sh.bin.n[sh.found];
      __syncthreads();
    }
    c.key = prefix;
    finish(c, k, aim);
  }

  // The same for at most kShort listed entries, by their places in the order; `last` too.
  __device__ __forceinline__ void cut_brief(Cut& c, int k, u64 aim, int& last) {
    const int e = entry_of(c.n);
    u64 order = 0, w = 0;
    if (e < c.n) {
      order = (u64)sh.key[e] << 32 | (uint32_t)~sh.idx[e];
      w = units1(sc.weight(of_key(sh.key[e])));
    }
    __syncthreads();  // (the bins are spent)
    if (e == tid) sh.brief.entry[e] = ulonglong2{order, w};
    if (tid == 0) sh.count = -1;
    __syncthreads();
    const u64 first = places(c.n, order);
    const int rank = (int)(first >> 53);
    const u64 before = c.above_w + (first & ((1ull << 53) - 1));
    const bool kept = tid < c.n && (k == 0 || c.above + rank < k) &&
                      (before < aim || (c.above == 0 && rank == 0));
    if (kept) atomicMax(&sh.count, rank);
    __syncthreads();
    if (kept && rank == sh.count) {
      sh.found_key = sh.key[e];
      sh.found = sh.idx[e];
    }
    __syncthreads();
    if (sh.count < 0) {  // none of them (none listed)
      keep_all(c);
      last = 0x7fffffff;
    } else {
      c.key = sh.found_key;
      last = sh.found;
    }
    __syncthreads();
  }

  // Everything down to the bound is kept.
  __device__ __forceinline__ void keep_all(Cut& c) {
    c.key = c.range.floor;
    c.ties = -1;
    c.all = 0;
  }

  // The intervals of the logits' line from the bound to the maximum.
  __device__ __forceinline__ void lay_bins(Range& r) {
    r.lo = r.floor > kDead + 1 ? of_key(r.floor) : (float)((double)m - 46.0 / s.c);
    const float width = m - r.lo;
    r.scale = width > 0.f && width < 3e38f ? (float)kBins / width : 0.f;
  }

  // The same of all entries from c.range.floor on, more than fit the list: by this workgroup
  // alone, narrowed by intervals first and then, if more than fit are in one, by the bits of
  // their keys.
  __device__ __forceinline__ void cut_alone(Cut& c, int k, u64 aim) {
    listed_cells = -1;
    lay_bins(c.range);
    int shift = 32;
    bool first = c.range.scale > 0.f;
#pragma unroll 1
    for (;;) {
      // A round: the bins of what is in question.
      for (int i = tid; i < kBins; i += kThreads) {
        sh.bin.n[i] = 0;
        sh.bin.w[i] = 0;
      }
      __syncthreads();
      const int low = first ? 0 : shift > 10 ? shift - 10 : 0;
      const int bits = first ? 10 : shift - low;
      each_entry([&](const Eight<T>& x, int) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t key = order_key(x[i]);
          if (first ? key >= c.range.floor : c.range.place(x[i], key) == 1) {
            const int b = first ? c.range.bin_of(x[i]) : (int)((key >> low) & ((1u << bits) - 1));
            atomicAdd(&sh.bin.n[b], 1u);
            atomicAdd(&sh.bin.w[b], units1(sc.weight(x[i])));
          }
        }
      });
      walk_bins<kBins>(c.above, c.above_w, k, aim);
      const int b = sh.found;
      c.above = sh.found2;
      c.above_w = sh.found_w;
      if (b < 0) {  // the limit is not reached (in the first round, if at all)
        c.n = 0;
        keep_all(c);
        __syncthreads();
        return;
      }
      const int held = (int)sh.bin.n[b];
      if (first) {
        c.range.bin = b;
        first = false;
      } else {
        shift = low;
        c.range.bits |= (uint32_t)b << low;
        c.range.mask = low == 0 ? ~0u : ~((1u << low) - 1);
      }
      __syncthreads();
      if (c.range.mask == ~0u) {  // equal logits alone
        c.key = c.range.bits;
        c.all = held;
        finish(c, k, aim);
        return;
      }
      if (held <= kList) break;
    }
    c.n = list_entries(c.range);
    cut_list(c, k, aim);
  }

  // How many of the equal logits at the border are kept.
  __device__ __forceinline__ void finish(Cut& c, int k, u64 aim) {
    int t = c.all;
    if (k > 0) t = min(t, k - c.above);
    const u64 w = units1(sc.weight(of_key(c.key)));
    if (aim != ~0ull && w > 0) {
      const u64 need = aim > c.above_w ? (aim - c.above_w + w - 1) / w : 0;
      if (need < (u64)t) t = (int)need;
    }
    c.ties = t > 0 ? t : (c.above > 0 ? 0 : 1);
  }

  // The index up to which entries of key c.key are kept.
  __device__ __forceinline__ int last_tie(const Cut& c) {
    if (c.ties < 0 || c.ties >= c.all) return 0x7fffffff;
    if (c.ties == 0) return -1;
    for (int i = tid; i < kMaxPieces; i += kThreads) sh.pcount[i] = 0;
    __syncthreads();
    if (c.in_list) {
      for (int i = tid; i < c.n; i += kThreads)
        if (sh.key[i] == c.key) atomicAdd(&sh.pcount[sh.idx[i] / kPiece], 1);
    } else {
      each_entry([&](const Eight<T>& x, int v0) __attribute__((always_inline)) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) n += order_key(x[i]) == c.key;
        if (n) atomicAdd(&sh.pcount[(v0 + 7) / kPiece], n);
      });
    }
    __syncthreads();
    if (wave == 0) {
      // Lane l: pieces 8 l .. 8 l + 7.
      constexpr int PER = kMaxPieces / 64;
      int own[PER], mine = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) mine += own[i] = sh.pcount[lane * PER + i];
      int sum = tiles::wave_incl_scan(mine) - mine, hit = -1, before = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (hit < 0 && sum + own[i] >= c.ties) {
          hit = lane * PER + i;
          before = sum;
        }
        sum += own[i];
      }
      const uint64_t hits = __ballot(hit >= 0);
      const int l = (int)__builtin_ctzll(hits);  // (the kept ones are among all)
      const int piece = __builtin_amdgcn_readlane(hit, l);
      int left = c.ties - __builtin_amdgcn_readlane(before, l);
      int found = -1;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        Eight<T> x;
        const int v0 = x.load(row, piece * kPiece + j * 512 + lane * 8, a.vocab);
        int n = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) n += order_key(x[i]) == c.key;
        const int incl = tiles::wave_incl_scan(n);
        int run = incl - n;
        int at = -1;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (order_key(x[i]) == c.key && ++run == left) at = v0 + i;
        const uint64_t got = __ballot(at >= 0);
        if (got && found < 0) found = __builtin_amdgcn_readlane(at, (int)__builtin_ctzll(got));
        left -= __builtin_amdgcn_readlane(incl, 63);
      }
      if (lane == 0) sh.found = found;
    }
    __syncthreads();
    const int last = sh.found;
    __syncthreads();
    return last;
  }

  // Weight of a kept entry, or 0.
  __device__ __forceinline__ u64 kept_units(float z, int v, uint32_t key_above, int last) const {
    const uint32_t key = order_key(z);
    const double w = sc.weight(z);
    const unsigned kept = (unsigned)(key > kDead) & (unsigned)(w >= (double)s.min_p) &
                          ((unsigned)(key > key_above) | ((unsigned)(key == key_above) & (unsigned)(v <= last)));
    return units1(w) & (0 - (u64)kept);
  }

  // The first index whose cumulative kept weight exceeds u times the sum, of the pieces'
  // kept weights in psum. The last with any weight where there is none.
  __device__ __forceinline__ void draw(int r, uint32_t key_above, int last, u64 sum) {
    __syncthreads();
    if (wave != 0) return;
    const int seq = r / a.each;
    const float u = a.u[seq * a.u_seq + (r - seq * a.each) * a.u_row];
    const double aim = (double)u * (double)sum;
    constexpr int PER = kMaxPieces / 64;
    u64 own[PER], mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) mine += own[i] = lane * PER + i < a.pieces ? sh.psum[lane * PER + i] : 0;
    u64 run = wave_scan(mine, lane) - mine;
    int hit = -1, some = -1;
    u64 hit_before = 0, some_before = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (own[i] > 0) {
        if (hit < 0 && (double)(run + own[i]) > aim) {
          hit = lane * PER + i;
          hit_before = run;
        }
        some = lane * PER + i;
        some_before = run;
      }
      run += own[i];
    }
    const uint64_t hits = __ballot(hit >= 0), somes = __ballot(some >= 0);
    int64_t token = 0;
    if (hits || somes) {
      const int l = hits ? (int)__builtin_ctzll(hits) : 63 - (int)__builtin_clzll(somes);
      const int piece = __builtin_amdgcn_readlane(hits ? hit : some, l);
      u64 before = lane_of(hits ? hit_before : some_before, l);
      int found = -1, spare = -1;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        Eight<T> x;
        const int v0 = x.load(row, piece * kPiece + j * 512 + lane * 8, a.vocab);
        u64 w[8], mine = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) mine += w[i] = kept_units(x[i], v0 + i, key_above, last);
        const u64 incl = wave_scan(mine, lane);
        u64 run = before + incl - mine;
        int at = -1, any = -1;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (w[i] > 0) {
            run += w[i];
            if (at < 0 && (double)run > aim) at = v0 + i;
            any = v0 + i;
          }
        const uint64_t ats = __ballot(at >= 0), anys = __ballot(any >= 0);
        if (ats && found < 0) found = __builtin_amdgcn_readlane(at, (int)__builtin_ctzll(ats));
        if (anys) spare = __builtin_amdgcn_readlane(any, 63 - (int)__builtin_clzll(anys));
        before += lane_of(incl, 63);
      }
      token = found >= 0 ? found : spare >= 0 ? spare : 0;
    }
    if (lane == 0) a.tokens[r] = token;
  }

  __device__ __forceinline__ void leave(int r, uint32_t key, int last, u64 sum) {
    if (tid == 0) {
      Decision d;
      d.max = m;
      d.key = key;
      d.last = last;
      d.min_p = s.min_p;
      d.c = s.c;
      d.sum = (double)sum / kUnit;
      *reinterpret_cast<Decision*>(a.records + (int64_t)r * a.row_bytes) = d;
    }
  }

  // No entry has a weight.
  __device__ __forceinline__ void nothing(int r) {
    if (!a.u)
      leave(r, ~0u, -1, 0);
    else if (tid == 0)
      a.tokens[r] = 0;
  }

  // The logit at which a weight is `share` of the maximum's, a little less for the rounding.
  __device__ __forceinline__ uint32_t floor_of(double share) const {
    const double z = (double)m + log2(share) / s.c;
    const double lo = z - 1e-6 * (fabs((double)m) + fabs(z)) - 1e-30;
    return lo > -3.4e38 ? order_key((float)lo) : 0;  // (NaN too: no bound)
  }

  // The first of the largest logits: of the first cell whose maximum is the row's.
  __device__ __forceinline__ void first_of_largest(int r) {
    const uint32_t top = order_key(m);
    int c = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < kCells; ++i)
      if (order_key(cell[i]) == top) c = min(c, cell_of(i));
    if (tid == 0) sh.found = 0x7fffffff;
    __syncthreads();
    if (c != 0x7fffffff) atomicMin(&sh.found, c);
    __syncthreads();
    if (wave != 0) return;
    const int v0 = sh.found * kCell;
    const int v1 = v0 + lane, v2 = v0 + 64 + lane;
    const uint64_t low = __ballot(v1 < a.vocab && order_key(T::get(row[min(v1, a.vocab - 1)])) == top);
    const uint64_t high = __ballot(v2 < a.vocab && order_key(T::get(row[min(v2, a.vocab - 1)])) == top);
    const int v = v0 + (low ? (int)__builtin_ctzll(low) : 64 + (high ? (int)__builtin_ctzll(high) : 0));
    if (!a.u)
      leave(r, top, v, (u64)kUnit);
    else if (lane == 0)
      a.tokens[r] = v;
  }

  // What is kept of a row: keys above `key`, or equal to it up to index `last`; `in_list`: all of
  // it is among the n listed entries, else the row is read again. Its token or its decision.
  __device__ __forceinline__ void conclude(int r, uint32_t key, int last, bool in_list, int n) {
    for (int i = tid; i < kMaxPieces; i += kThreads) sh.psum[i] = 0;
    __syncthreads();
    if (in_list) {
      add_listed(key, last, n);
    } else {
      listed_cells = -1;
      each_entry([&](const Eight<T>& x, int v0) __attribute__((always_inline)) {
        u64 w = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) w += kept_units(x[i], v0 + i, key, last);
        w = wave_sum(w);
        if (lane == 0 && w) atomicAdd(&sh.psum[(v0 + 7) / kPiece], w);
      });
    }
    sum_up(r, key, last);
  }

  // The kept ones of the list, into their pieces' sums.
  __device__ __forceinline__ void add_listed(uint32_t key, int last, int n) {
#pragma unroll 1
    for (int i = tid; i < n; i += kThreads) {
      const u64 w = kept_units(of_key(sh.key[i]), sh.idx[i], key, last);
      if (w) atomicAdd(&sh.psum[sh.idx[i] / kPiece], w);
    }
  }

  __device__ __forceinline__ void sum_up(int r, uint32_t key, int last) {
    __syncthreads();
    const u64 sum = block_sum(sh.psum[tid]);
    if (a.u)
      draw(r, key, last, sum);
    else
      leave(r, key, last, sum);
  }

  // The whole way of a row whose list does not fit, by this workgroup alone.
  __device__ __forceinline__ void alone(int r, uint32_t floor, u64 whole) {
    // (With top-k and top-p, the former's cut gives the sum for the latter's.)
    u64 aim = ~0ull, total = whole;
    Cut c;
#pragma unroll 1
    for (int pass = s.k > 0 && s.p < 1.f ? 0 : 1; pass < 2; ++pass) {
      if (pass == 1 && s.p < 1.f) aim = (u64)ceil((double)s.p * (double)total);
      c = Cut{};
      c.range = Range{floor, 0.f, 0.f, 0, 0, 0};
      cut_alone(c, s.k, aim);
      if (pass == 0) total = weight_to(c);
    }
    conclude(r, c.key, last_tie(c), false, 0);
  }

  // Weight of the entries up to a cut.
  __device__ __forceinline__ u64 weight_to(const Cut& c) {
    if (c.ties < 0) return c.above_w + everything(c.n);
    return c.above_w + (u64)c.ties * units1(sc.weight(of_key(c.key)));
  }

  __device__ __forceinline__ void decide(int r) {
    char* const rec = a.records + (int64_t)r * a.row_bytes;
    Shared_row* const state = reinterpret_cast<Shared_row*>(rec + sizeof(Decision));
    const auto rp = tiles::tile_rsrc(rec + kHead, a.pieces * (int)sizeof(Piece));
    const auto rc = tiles::tile_rsrc(rec + kHead + a.pieces * sizeof(Piece), (a.cells + 3) / 4 * 16);
    if (tid == 0) a.modes[r] = kDecided;  // (unless the row is shared, below)
    // Each thread its piece; maximum and sum of all.
    static_assert(kMaxPieces == kThreads, "one piece per thread");
    const f32x4 y = tiles::load_coherent16(rp, tid * 16);
    load_cells(rc);
    typedef double f64x2 __attribute__((ext_vector_type(2)));
    const float pm = tid < a.pieces ? y[0] : kNegInf;
    const double ps = tid < a.pieces ? __builtin_bit_cast(f64x2, y)[1] : 0.0;
    set_max(block_max(pm));
    if (m == kNegInf) {
      nothing(r);
      return;
    }
    if (s.k == 1) {
      first_of_largest(r);
      return;
    }
    u64 whole = 0;
    if (s.whole) {
      // (A piece none of whose entries has a unit of weight counts as nothing.)
      const double top = sc.top_only ? (pm == m ? 1.0 : 0.0) : sc.weight(pm);
      const u64 w = pm == kNegInf || units1(top) == 0 ? 0 : units(ps * top);
      if (tid < a.pieces) sh.psum[tid] = w;
      whole = block_sum(w);
    }
    const uint32_t lowest = sc.top_only ? order_key(m) : kDead + 1;  // key with a weight
    if (!s.filtered) {
      if (a.u)
        draw(r, lowest, 0x7fffffff, whole);
      else
        leave(r, lowest, 0x7fffffff, whole);
      return;
    }
    uint32_t floor = lowest;
    if (s.k > 0)
      floor = cell_bound(s.k);
    else if (s.p < 1.f)
      floor = floor_of((1.0 - (double)s.p) * ((double)whole / kUnit) / a.vocab);
    if (s.min_p > 0.f && (s.k == 0 || s.p == 1.f)) floor = max(floor, floor_of((double)s.min_p));
    floor = max(floor, lowest);
    // (Where most cells of a long row reach the bound, its entries are not even counted here:
    // with top-p or min-p they are nearly always too many, and one workgroup takes 25 us for
    // 150,000. With top-k this begins at k of a quarter of the cells, whose list may be short: one
    // row of 33000 takes 18.6 us at k = 58 and 32.4 at 70, of 151936 38.9 at 290 and 32.2 at 302. With
    // top-p as well the row then takes the two cuts of a workgroup alone: 17.6 and 67.5, 37.9 and 182.)
    const bool few = list_cells(floor);
    if (!few) listed_cells = -1;
    const int n = few || a.pieces <= kAlonePieces || r >= a.shared_rows
                      ? list_entries(Range{floor, 0.f, 0.f, 0, 0, 0}) : kList + 1;
    if (n <= kShort) {
      brief(r, n, whole);
      return;
    }
    const bool limited = s.k > 0 || s.p < 1.f;  // (with min-p alone, only the weights decide)
    if (n > kList) {
      share_or_not(r, floor, whole, limited, state);
      return;
    }
    uint32_t key = floor;
    int last = 0x7fffffff;
    if (limited) {
      u64 aim = ~0ull, total = whole;
      Cut c;
#pragma unroll 1
      for (int pass = s.k > 0 && s.p < 1.f ? 0 : 1; pass < 2; ++pass) {
        if (pass == 1 && s.p < 1.f) aim = (u64)ceil((double)s.p * (double)total);
        c = Cut{};
        c.range = Range{floor, 0.f, 0.f, 0, 0, 0};
        c.n = n;
        cut_list(c, s.k, aim);
        if (pass == 0) total = weight_to(c);
      }
      key = c.key;
      last = last_tie(c);
    }
    conclude(r, key, last, true, n);
  }

  // ---- a row shared by workgroups ----

  // Who does a row whose list does not fit: several workgroups, or one in the next launch. Top-k
  // and top-p together would take two cuts; lists may have run out; and the intervals have to
  // be wider than the slack of the bound for min-p.
  __device__ __forceinline__ void share_or_not(int r, uint32_t floor, u64 whole, bool limited,
                                               Shared_row* state) {
    Range range{floor, 0.f, 0.f, 0, 0, 0};
    lay_bins(range);
    const bool fine = range.scale > 0.f &&
                      (s.min_p == 0.f || m - range.lo > 0.0164f * (fabsf(m) + fabsf(range.lo)));
    const int mode = r >= a.shared_rows ? kAlone
                     : !limited         ? kKeepAll
                     : fine && !(s.k > 0 && s.p < 1.f) ? kCount : kAlone;
    if (mode == kCount) {
      for (int i = tid; i < kBins; i += kThreads) room_of(r)[i] = 0;
    }
    if (tid == 0) {
      Shared_row x{};
      a.modes[r] = mode;
      x.max = m;
      x.floor = floor;
      x.lo = range.lo;
      x.scale = range.scale;
      x.end = kBins;
      x.aim = s.p < 1.f ? (u64)ceil((double)s.p * (double)whole) : ~0ull;
      x.whole = whole;
      *state = x;
    }
  }

  __device__ __forceinline__ u64* room_of(int r) const { return a.rooms + (int64_t)r * kRoom; }

  // f(p, x, v0) for this workgroup's pieces, by whole wavefronts: piece p's entries, from v0 on,
  // the next piece's on their way.
  int groups = 1;  // workgroups that share the row
  template <typename F>
  __device__ __forceinline__ void each_piece(int group, F f) {
    const int stride = groups * kWaves;
    Eight<T> next[2];
    int at[2];
    auto take = [&](int p) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 2; ++j) at[j] = next[j].load(row, p * kPiece + j * 512 + lane * 8, a.vocab);
    };
    int p = group * kWaves + wave;
    if (p < a.pieces) take(p);
#pragma unroll 1
    for (; p < a.pieces; p += stride) {  // wavefront-uniform
      const Eight<T> x[2] = {next[0], next[1]};
      const int v0[2] = {at[0], at[1]};
      if (p + stride < a.pieces) take(p + stride);
      f(p, x, v0);
    }
  }

  // This workgroup's pieces into the row's counts (of 2^40) and places (of 2^-16 interval).
  __device__ __forceinline__ void count(int r, int group, const Shared_row& state) {
    for (int i = tid; i < kBins; i += kThreads) sh.bin.w[i] = 0;
    __syncthreads();
    const float lowest = of_key(state.floor), lo = state.lo, scale = state.scale;
    each_piece(group, [&](int, const Eight<T> (&x)[2], const int (&)[2]) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float z = x[j][i];
          const float t = fmaxf((z - lo) * scale, 0.f);
          const int b = min((int)t, kBins - 1);
          const unsigned place = (unsigned)((t - (float)b) * 65536.f);
          if (z >= lowest) atomicAdd(&sh.bin.w[b], (u64)place | 1ull << 40);
        }
    });
    __syncthreads();
    u64* const room = room_of(r);
    for (int i = tid; i < kBins; i += kThreads) {
      const u64 x = sh.bin.w[i];
      if (x) __hip_atomic_fetch_add(room + i, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }

  // Of all of them, the intervals that can hold the border: with top-k the one that does; with
  // top-p, from the first that reaches aim by the upper bounds of the weights down to the first
  // that does by the lower ones. (Ends and means are taken a thousandth of an interval further:
  // the numbers that intervals go by are rounded. The first interval may hold entries below it.)
  __device__ __forceinline__ void bracket(int r, Shared_row* state) {
    const u64* const room = room_of(r);
    constexpr int PER = kBins / kThreads;
    u64 x[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i)
      x[i] = __hip_atomic_load(room + i * kThreads + tid, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const double wide = 1.0 / (double)state->scale, lo = state->lo;
    auto weight_at = [&](double t) {
      return exp2_of(fmax((fmin(lo + t * wide, (double)m) - sc.m) * sc.c, sc.low));
    };
    const u64 aim = state->aim;
    int ends[2];  // by the upper bounds, by the lower ones
#pragma unroll 1
    for (int lower = s.k > 0 ? 1 : 0; lower < 2; ++lower) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int b = i * kThreads + tid;
        const int n = (int)(x[i] >> 40);
        double w = 0.0;
        if (n > 0 && s.k == 0) {
          const double mean = (double)(x[i] & 0xffffffffffull) / (65536.0 * n);
          if (lower) {
            w = b > 0 ? weight_at(b + mean - 1e-3) : 0.0;
          } else {
            const double w0 = weight_at(b - 1e-3), w1 = weight_at(b + 1.001);
            w = w0 + (w1 - w0) * fmin((mean + 2e-3) / 1.002, 1.0);
          }
        }
        sh.bin.n[b] = n;
        sh.bin.w[b] = units((double)n * w);
      }
      walk_bins<kBins>(0, 0, s.k, aim);
      ends[lower] = sh.found;
      __syncthreads();
    }
    if (s.k > 0) ends[0] = ends[1];
    if (tid == 0) {
      a.modes[r] = kShare;
      state->first = max(ends[1], 0);
      state->end = ends[0] < 0 ? 1 : ends[0] + 1;
    }
  }

  // This workgroup's pieces: the weight above the bracket into the pieces' sums, what lies in it
  // into the row's list. (Sums of every entry's own units, as the draw looks for them: of many
  // entries of less than half a unit the sum would have some, and no entry the token.)
  __device__ __forceinline__ void share(int r, int group, bool all, Shared_row* state, Piece* pieces) {
    const float lowest = of_key(state->floor), lo = state->lo, scale = state->scale;
    const float from = state->first > 0 ? (float)state->first : kNegInf;
    const float to = state->end < kBins ? (float)state->end : -kNegInf;
    u64* const list = room_of(r);
    each_piece(group, [&](int p, const Eight<T> (&x)[2], const int (&v0)[2]) __attribute__((always_inline)) {
      u64 w = 0;
      uint64_t any = 0;  // lanes with an entry in the bracket (or with top-k above it)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // (Without branches around an entry: their chains of dependent instructions overlap. What
        // is no number compares as neither.)
        float z[8];
        double y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = x[j].raw(i);
        if (all) {
          sc.weights(z, y);
          w += sum_units1(y, [&](int i) __attribute__((always_inline)) {
            return (unsigned)(z[i] >= lowest) & (unsigned)(y[i] >= (double)s.min_p);
          });
          continue;
        }
        uint64_t over = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float t = (z[i] - lo) * scale;
          const uint64_t high = __ballot(t >= to), low = __ballot(t >= from);
          over |= high;
          any |= (s.k > 0 ? low : low & ~high) & __ballot(z[i] >= lowest);
        }
        if (over != 0) {  // (above the bracket every entry weighs min_p, too: see share_or_not)
          sc.weights(z, y);
          w += sum_units1(y, [&](int i) __attribute__((always_inline)) {
            return (z[i] - lo) * scale >= to;
          });
        }
      }
      if (any != 0) {
        unsigned in[2] = {0, 0};
        int counts = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          unsigned over = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float z = x[j].raw(i), t = (z - lo) * scale;
            const unsigned high = t >= to;
            over |= high << i;
            in[j] |= ((unsigned)(z >= lowest) & (unsigned)(t >= from) & ~high) << i;
          }
          counts += __builtin_popcount(in[j]);
          if (s.k > 0) counts += __builtin_popcount(over) << 16;
        }
        const int incl = tiles::wave_incl_scan(counts);  // (1024 of each at most)
        const int total = __builtin_amdgcn_readlane(incl, 63);
        int at = 0;
        if (lane == 63)
          at = (int)(uint32_t)__hip_atomic_fetch_add(
              &state->counts, (u64)(total & 0xffff) | (u64)(total >> 16) << 32, __ATOMIC_RELAXED,
              __HIP_MEMORY_SCOPE_AGENT);
        at = __builtin_amdgcn_readlane(at, 63) + ((incl - counts) & 0xffff);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (in[j] >> i & 1) {
              if (at < kList)
                __hip_atomic_store(list + at, (u64)order_key(x[j][i]) << 32 | (uint32_t)(v0[j] + i),
                                   __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
              ++at;
            }
      }
      w = wave_sum(w);
      if (lane == 0)
        __hip_atomic_store(reinterpret_cast<u64*>(&pieces[p].sum), w, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
    });
  }

  // The end of a shared row, of all workgroups' lists and sums.
  __device__ __forceinline__ void end(int r, bool all, Shared_row* state, Piece* pieces) {
    sh.psum[tid] = tid < a.pieces
                       ? __hip_atomic_load(reinterpret_cast<const u64*>(&pieces[tid].sum),
                                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                       : 0;
    Cut c{};
    c.range.floor = state->floor;
    keep_all(c);
    int last = 0x7fffffff;
    if (!all) {
      const u64 counts = __hip_atomic_load(&state->counts, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const u64 aim = state->aim;
      const u64* const list = room_of(r);
      c.n = (int)min(counts & 0xffffffffu, (u64)0x7fffffff);
      for (int i = tid; i < min(c.n, kList); i += kThreads) {
        const u64 x = __hip_atomic_load(list + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sh.key[i] = (uint32_t)(x >> 32);
        sh.idx[i] = (int)(uint32_t)x;
      }
      c.above = (int)(counts >> 32);
      c.above_w = block_sum(sh.psum[tid]);
      bool fits = c.n <= kList;
      if (fits) {  // and the border is in the bracket, as it should be
        const u64 w = everything(c.n);
        fits = s.k > 0 ? c.above < s.k && (c.above + c.n >= s.k || state->first == 0)
                       : c.above_w < aim && (c.above_w + w >= aim || state->first == 0);
      }
      if (!fits) {
        alone(r, state->floor, state->whole);
        return;
      }
      if (c.above_w > 0 && c.above == 0) c.above = 1;  // (not counted: some)
      if (c.n <= kShort) {
        cut_brief(c, s.k, aim, last);
      } else {
        cut_list(c, s.k, aim);
        last = last_tie(c);
      }
      add_listed(c.key, last, c.n);
    }
    sum_up(r, c.key, last);
  }

  // Weight of all listed entries.
  __device__ __forceinline__ u64 everything(int n) {
    u64 w = 0;
    for (int i = tid; i < n; i += kThreads) w += units1(sc.weight(of_key(sh.key[i])));
    return block_sum(w);
  }

  // A row of at most kShort entries, one per thread.
  __device__ __forceinline__ void decide_short(int r) {
    const float z = tid < a.vocab ? fmaxf(T::get(row[tid]), kNegInf) : kNegInf;
    set_max(block_max(z));
    if (m == kNegInf) {
      nothing(r);
      return;
    }
    const bool out = z == kNegInf || (sc.top_only && z != m);
    if (tid < a.vocab) {
      sh.key[tid] = out ? kDead : order_key(z);
      sh.idx[tid] = tid;
    }
    const u64 whole = block_sum(out ? 0 : units1(sc.weight(z)));
    brief(r, a.vocab, whole);
  }

  // Which entry of n in sh.brief is this thread's: of up to kShort / 2, thread e + kShort / 2 is
  // entry e's partner.
  __device__ __forceinline__ int entry_of(int n) const {
    return n <= kShort / 2 ? tid & (kShort / 2 - 1) : tid;
  }
  // The sum over the n entries in sh.brief of what f makes of each, for the thread's entry; of a
  // pair the first thread gets it.
  template <typename F>
  __device__ __forceinline__ u64 over_brief(int n, F f) {
    static_assert(kThreads == kShort, "a thread per entry, or two");
    const bool pairs = n <= kShort / 2;
    // (Behind the n there are entries that add nothing, up to a multiple of 16.)
    const int per = pairs ? (n + 15) / 16 * 8 : (n + 7) / 8 * 8;
    const int from = pairs && tid >= kShort / 2 ? per : 0;
    u64 x = 0;
    if (entry_of(n) < ((n + 63) & ~63)) {  // wavefront-uniform
#pragma unroll 1
      for (int i = from; i < from + per; i += 8)
#pragma unroll
        for (int j = 0; j < 8; ++j) x += f(sh.brief.entry[i + j]);
    }
    if (pairs) {  // uniform
      if (tid >= kShort / 2) sh.brief.more[tid - kShort / 2] = x;
      __syncthreads();
      if (tid < kShort / 2) x += sh.brief.more[tid];
    }
    return x;
  }

  // How many of the entries in sh.brief come before `order`, times 2^53, and their weight.
  // (Weights of 2^44 at most: 512 of them leave room for their number in the same sum.)
  __device__ __forceinline__ u64 places(int n, u64 order) {
    return over_brief(n, [&](ulonglong2 x) __attribute__((always_inline)) {
      return x.x > order ? x.y + (1ull << 53) : 0;
    });
  }

  // The end for at most kShort listed entries, one per thread: every entry's
  // place in the order and the weight before it.
  __device__ __forceinline__ void brief(int r, int n, u64 whole) {
    const int e = entry_of(n);
    u64 order = 0, w = 0;
    uint32_t key = 0;
    int v = 0;
    if (e < n) {
      key = sh.key[e];
      v = sh.idx[e];
      order = (u64)key << 32 | (uint32_t)~v;
      w = units1(sc.weight(of_key(key)));
    }
    if (e == tid) sh.brief.entry[e] = ulonglong2{order, w};
    __syncthreads();
    const u64 first = places(n, order);
    const int rank = (int)(first >> 53);
    const u64 before = first & ((1ull << 53) - 1);
    bool kept = tid < n && key > kDead && (s.k == 0 || rank < s.k);
    if (s.p < 1.f) {
      u64 total = whole;
      if (s.k > 0) total = block_sum(kept ? w : 0);
      const u64 aim = (u64)ceil((double)s.p * (double)total);
      kept = kept && (rank == 0 || before < aim);
    }
    if (kept && s.min_p > 0.f) kept = sc.weight(of_key(key)) >= (double)s.min_p;
    const u64 sum = block_sum(kept ? w : 0);
    if (!a.u) {
      // The last kept one in the order.
      if (tid == 0) sh.count = 0;
      __syncthreads();
      if (kept) atomicMax(&sh.count, rank);
      __syncthreads();
      if (kept && rank == sh.count) {
        sh.found_key = key;
        sh.found = v;
      }
      __syncthreads();
      leave(r, sh.found_key, sh.found, sum);
      return;
    }
    // By the index now. (All have left the first walk behind block_sum's barriers.)
    if (e == tid) sh.brief.entry[e] = ulonglong2{(u64)v, kept ? w : 0};
    if (tid == 0) sh.found = sh.found2 = -1;
    __syncthreads();
    const u64 run = over_brief(n, [&](ulonglong2 x) __attribute__((always_inline)) {
      return (int)x.x <= v ? x.y : 0;
    });
    if (kept && w > 0) {
      const int seq = r / a.each;
      const double aim = (double)a.u[seq * a.u_seq + (r - seq * a.each) * a.u_row] * (double)sum;
      if ((double)run > aim && (run == w || !((double)(run - w) > aim))) sh.found = v;  // one, or none
      atomicMax(&sh.found2, v);
    }
    __syncthreads();
    if (tid == 0) a.tokens[r] = sh.found >= 0 ? sh.found : sh.found2;
  }
};

template <typename T>
__device__ __forceinline__ const typename T::E* row_of(const Args& a, int r, int seq) {
  return (const typename T::E*)a.logits + seq * a.s_seq + (int64_t)(r - seq * a.each) * a.s_row;
}

// Counts this workgroup's arrival at row r; whether it is the last of `groups`.
__device__ __forceinline__ bool arrive_last(const Args& a, int r, int groups, int tid, int& s_last) {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_s_waitcnt(0);  // what it leaves has landed before the arrival counts
  __syncthreads();
  if (tid == 0)
    s_last = __hip_atomic_fetch_add(a.cnt + r, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
             groups - 1;
  __syncthreads();
  if (!s_last) return false;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  if (tid == 0) __hip_atomic_store(a.cnt + r, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return true;
}

// One reading of the row: its pieces of this workgroup.
template <typename T>
__device__ __forceinline__ void read_row(const Args& a, const typename T::E* row, const Settings& s,
                                         char* rec, int group, int wave, int lane) {
  Piece* const pieces = reinterpret_cast<Piece*>(rec + kHead);
  float* const cells = reinterpret_cast<float*>(rec + kHead + a.pieces * sizeof(Piece));
  auto take = [&](int p, Eight<T> (&x)[2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) x[j].load(row, p * kPiece + j * 512 + lane * 8, a.vocab);
  };
  auto reduce = [&](int p, const Eight<T> (&w)[2]) {
    float x[2][8];
    float mp = kNegInf;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[j][i] = w[j][i];
      float y = fmaxf(fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3])),
                      fmaxf(fmaxf(x[j][4], x[j][5]), fmaxf(x[j][6], x[j][7])));
      y = row_max(y);
      const int c = p * (kPiece / kCell) + j * 4 + (lane >> 4);
      // Device-coherent, as all that the deciding workgroup reads: it may run on another XCD.
      if ((lane & 15) == 0 && c < a.cells) tiles::store_coherent(cells + c, y);
      mp = fmaxf(mp, y);
    }
    mp = wave_max_of_rows(mp);
    double sum = 0.0;
    if (s.whole && mp != kNegInf) {  // wavefront-uniform
      const Scale sc(mp, s.c);
      if (sc.top_only) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) sum += x[j][i] == mp ? 1.0 : 0.0;
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          double y[8];
          sc.weights(x[j], y);
          sum += ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
        }
      }
      sum = wave_sum(sum);
    }
    if (lane == 0) {
      tiles::store_coherent(&pieces[p].max, mp);
      __hip_atomic_store(&pieces[p].sum, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  };
  const int stride = a.groups * kWaves;
  Eight<T> x0[2], x1[2];
  int p = group * kWaves + wave;
  if (p < a.pieces) take(p, x0);
  while (p < a.pieces) {  // wavefront-uniform
    if (p + stride < a.pieces) take(p + stride, x1);
    reduce(p, x0);
    p += stride;
    if (p >= a.pieces) break;
    if (p + stride < a.pieces) take(p + stride, x0);
    reduce(p, x1);
    p += stride;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads, 4) void sample_kernel(Args a) {
  __shared__ Shared sh;
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = blockIdx.x / a.groups;
  const int seq = r / a.each;
  const typename T::E* row = row_of<T>(a, r, seq);
  const Settings s = settings_of(a, seq);
  Decider<T> d(a, sh, row, s, tid, lane, wave);
  if (a.vocab <= kShort) {
    d.decide_short(r);
    return;
  }
  char* const rec = a.records + (int64_t)r * a.row_bytes;
  read_row<T>(a, row, s, rec, blockIdx.x - r * a.groups, wave, lane);
  if (arrive_last(a, r, a.groups, tid, s_last)) d.decide(r);
}

// The launches that share a row whose list does not fit: END false, its counts per interval;
// END true, the bracket's list and the end.
template <typename T, bool END>
__global__ __launch_bounds__(kThreads, 4) void shared_kernel(Args a) {
  __shared__ Shared sh;
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // The rows that take part (kCount turns into kShare under these reads, and counts as well), as
  // many workgroups for each as fill the GPU once over all, results not depending on their
  // number; the workgroups are numbered over those that have work. (Numbered over all rows, the
  // ones that leave at once take their turns with the dispatcher all the same, and the others
  // pile up on some compute units: 256 rows at top-p 0.9 179 us where they take 114.)
  auto takes_part = [&](int row) {
    if (row >= a.rows) return false;
    const int x = __hip_atomic_load(a.modes + row, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return END ? x != kDecided : x == kCount || x == kShare;
  };
  auto in_group = [&](int base, int& before) {  // rows base + tid: whether; how many before, in all
    const uint64_t b = __ballot(takes_part(base + tid));
    if (lane == 0) sh.part_n[wave] = __popcll(b);
    __syncthreads();
    before = __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0u));
    int all = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      before += i < wave ? sh.part_n[i] : 0;
      all += sh.part_n[i];
    }
    __syncthreads();
    return (b >> lane & 1) ? all : ~all;
  };
  int n = 0, before;
  for (int base = 0; base < a.rows; base += kThreads) {
    const int x = in_group(base, before);
    n += x < 0 ? ~x : x;
  }
  if (n == 0) return;
  // One workgroup per compute unit for few rows (each adds up to 2048 counts to its row's room: 32
  // rows of 100003 at T 1.4, top-p 0.97 62.0 us with two, 55.6 with one), else two (100 rows of
  // 151936 at top-p 0.9 81.8 us with one, 73.3 with two; 256 rows 130.9 and 114.0).
  const int groups = max(1, min(a.shared_groups, (4 * n <= a.cus ? 1 : 2) * a.cus / n));
  const int nth = blockIdx.x / groups, group = blockIdx.x - nth * groups;
  if (nth >= n) return;
  int seen = 0;
  for (int base = 0; base < a.rows; base += kThreads) {
    const int x = in_group(base, before);
    if (x >= 0 && seen + before == nth) sh.found = base + tid;
    seen += x < 0 ? ~x : x;
  }
  __syncthreads();
  const int r = sh.found;
  __syncthreads();
  const int mode = a.modes[r];
  if (!END && mode != kCount) return;  // (cannot be: it ends with its last workgroup)
  char* const rec = a.records + (int64_t)r * a.row_bytes;
  Shared_row* const state = reinterpret_cast<Shared_row*>(rec + sizeof(Decision));
  Piece* const pieces = reinterpret_cast<Piece*>(rec + kHead);
  const int seq = r / a.each;
  Decider<T> d(a, sh, row_of<T>(a, r, seq), settings_of(a, seq), tid, lane, wave);
  d.groups = groups;
  d.set_max(state->max);
  if constexpr (!END) {
    d.count(r, group, *state);
    if (arrive_last(a, r, d.groups, tid, s_last)) d.bracket(r, state);
  } else if (mode == kAlone) {
    if (group == 0) d.alone(r, state->floor, state->whole);
  } else {
    d.share(r, group, mode == kKeepAll, state, pieces);
    if (arrive_last(a, r, d.groups, tid, s_last)) d.end(r, mode == kKeepAll, state, pieces);
  }
}

// Probabilities of one piece per wavefront.
template <typename T>
__global__ __launch_bounds__(256) void probs_kernel(Args a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = (int64_t)blockIdx.x * 4 + wave;
  const int r = (int)(item / a.pieces), p = (int)(item - (int64_t)r * a.pieces);
  if (r >= a.rows) return;
  const int seq = r / a.each;
  const typename T::E* row = (const typename T::E*)a.logits + seq * a.s_seq +
                             (int64_t)(r - seq * a.each) * a.s_row;
  const Decision d = *reinterpret_cast<const Decision*>(a.records + (int64_t)r * a.row_bytes);
  float* out = a.probs + (int64_t)r * a.vocab;
  const Scale sc(d.max, d.c);
  const double inv = d.sum > 0.0 ? 1.0 / d.sum : 0.0;
  if (a.vocab <= kShort) {  // (one piece)
    for (int v = lane; v < a.vocab; v += 64) {
      const float z = fmaxf(T::get(row[v]), kNegInf);
      const uint32_t key = order_key(z);
      const double w = sc.weight(z);
      out[v] = key > kDead && (key > d.key || (key == d.key && v <= d.last)) && w >= (double)d.min_p
                   ? (float)(w * inv) : 0.f;
    }
    return;
  }
  Eight<T> x[2];
  int at[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) at[j] = x[j].load(row, p * kPiece + j * 512 + lane * 8, a.vocab);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int v0 = at[j];
    float y[8];
    bool in[8], any = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t key = order_key(x[j][i]);
      in[i] = key > kDead && (key > d.key || (key == d.key && v0 + i <= d.last));
      any |= in[i];
      y[i] = 0.f;
    }
    if (__ballot(any) != 0) {
      float z[8];
      double w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = x[j][i];
      sc.weights(z, w);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (in[i] && w[i] >= (double)d.min_p) y[i] = (float)(w[i] * inv);
    }
    typedef float quad __attribute__((ext_vector_type(4), aligned(4)));
    const int first = p * kPiece + j * 512 + lane * 8;
    if (first == v0) {
      *reinterpret_cast<quad*>(out + v0) = quad{y[0], y[1], y[2], y[3]};
      *reinterpret_cast<quad*>(out + v0 + 4) = quad{y[4], y[5], y[6], y[7]};
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (v0 + i >= first) out[v0 + i] = y[i];
    }
  }
}

static size_t modes_bytes(int rows) { return (size_t)(rows + 3) / 4 * 16; }
static int pieces_of(int vocab) { return (vocab + kPiece - 1) / kPiece; }
static int cells_of(int vocab) { return (vocab + kCell - 1) / kCell; }

// Workgroups per row: one wavefront per piece for a few rows; for many, as many as fill
// kWavesPerCu wavefronts per compute unit over all rows, the pieces dealt in whole rounds.
constexpr int kWavesPerCu = 16;
static int groups_of(int rows, int pieces) {
  int64_t waves = (int64_t)kWavesPerCu * device_cus() / rows;
  if (waves < 1) waves = 1;
  const int64_t rounds = (pieces + waves - 1) / waves;
  const int64_t per_round = (pieces + rounds - 1) / rounds;
  return (int)((per_round + kWaves - 1) / kWaves);
}

// Whether no row's list can be too long: short rows, and settings of all rows that list nothing.
static bool never_shared(const Args& a) {
  if (a.vocab <= kList) return true;
  const bool greedy = !a.temperature && !(a.t_all > 0.f);
  const bool one = !a.top_k && a.k_all == 1;
  const bool plain = !a.top_k && (a.k_all <= 0 || a.k_all >= a.vocab) && !a.top_p &&
                     !(a.p_all < 1.f) && !a.min_p && !(a.m_all > 0.f);
  return greedy || one || plain;
}

template <typename T>
static hipError_t launch(const Args& a, hipStream_t stream) {
  sample_kernel<T><<<(unsigned)(a.rows * (int64_t)a.groups), kThreads, 0, stream>>>(a);
  if (!never_shared(a)) {
    const unsigned grid = (unsigned)(a.rows * (int64_t)a.shared_groups);
    shared_kernel<T, false><<<grid, kThreads, 0, stream>>>(a);
    shared_kernel<T, true><<<grid, kThreads, 0, stream>>>(a);
  }
  if (a.probs)
    probs_kernel<T><<<(unsigned)(((int64_t)a.rows * a.pieces + 3) / 4), 256, 0, stream>>>(a);
  return hipGetLastError();
}

// Workgroups that may share a row of a long list, at most: one wavefront per piece, or as many
// as a launch of kMostShared (most of which have nothing to do and cost 2 us in all) has for it.
constexpr int kMostShared = 2048;
static int shared_groups_of(int rows, int pieces) {
  const int most = (pieces + kWaves - 1) / kWaves, fair = kMostShared / rows;
  return fair < 1 ? 1 : fair < most ? fair : most;
}
static int shared_rows_of(int rows, int vocab) {
  return vocab <= kList ? 0 : rows < kMaxShared ? rows : kMaxShared;
}

static int run(const Args& a, int dtype, hipStream_t stream) {
  const hipError_t e = dtype == PA_F16    ? launch<Half>(a, stream)
                       : dtype == PA_BF16 ? launch<Brain>(a, stream)
                                          : launch<Single>(a, stream);
  if (e == hipSuccess) return PA_OK;
  set_error("HIP launch failed: %s", hipGetErrorString(e));
  return PA_ERR_HIP;
}

}  // namespace sample
}  // namespace pa

using namespace pa;
using namespace pa::sample;

extern "C" {

size_t pa_sample_workspace_bytes(int num_seqs, int rows_per_seq, int vocab) {
  const int64_t rows = (int64_t)num_seqs * rows_per_seq;
  if (num_seqs <= 0 || rows_per_seq <= 0 || rows > kMaxRows || vocab <= 0 || vocab > kMaxVocab) return 0;
  return kCounterBytes + modes_bytes((int)rows) +
         (size_t)rows * row_record(pieces_of(vocab), cells_of(vocab)) +
         (size_t)shared_rows_of((int)rows, vocab) * kRoom * sizeof(u64);
}

static int start(Args& a, const void* logits, int dtype, const int64_t* strides, int num_seqs,
                 int rows_per_seq, int vocab, const float* temperature, float temperature_all,
                 const int32_t* top_k, int top_k_all, const float* top_p, float top_p_all,
                 const float* min_p, float min_p_all, const void* out, void* workspace,
                 size_t workspace_bytes) {
  clear_error();
  if (num_seqs < 0 || rows_per_seq < 0 || vocab <= 0) {
    set_error("num_seqs (%d) and rows_per_seq (%d) must be >= 0, vocab (%d) positive", num_seqs,
              rows_per_seq, vocab);
    return PA_ERR_ARG;
  }
  if (dtype != PA_F16 && dtype != PA_BF16 && dtype != PA_F32) {
    set_error("unknown type of logits %d", dtype);
    return PA_ERR_ARG;
  }
  if (num_seqs == 0 || rows_per_seq == 0) return PA_OK;
  if ((int64_t)num_seqs * rows_per_seq > kMaxRows || vocab > kMaxVocab) {
    set_error("at most %d rows of %d logits, %d x %d of %d given", kMaxRows, kMaxVocab, num_seqs,
              rows_per_seq, vocab);
    return PA_ERR_UNSUPPORTED;
  }
  if (!logits || !strides || !out) {
    set_error("null pointer argument");
    return PA_ERR_ARG;
  }
  if (strides[2] != 1 && vocab > 1) {
    set_error("the rows of logits need unit vocabulary stride");
    return PA_ERR_ARG;
  }
  if ((uintptr_t)logits % (dtype == PA_F32 ? 4 : 2)) {
    set_error("logits must be aligned to their type");
    return PA_ERR_ARG;
  }
  const size_t need = pa_sample_workspace_bytes(num_seqs, rows_per_seq, vocab);
  if (!workspace || workspace_bytes < need) {
    set_error("workspace of %zu bytes needed, %zu given", need, workspace_bytes);
    return PA_ERR_WORKSPACE;
  }
  a.logits = logits;
  a.s_seq = strides[0];
  a.s_row = strides[1];
  a.rows = num_seqs * rows_per_seq;
  a.each = rows_per_seq;
  a.vocab = vocab;
  a.temperature = temperature;
  a.t_all = temperature_all;
  a.top_k = top_k;
  a.k_all = top_k_all;
  a.top_p = top_p;
  a.p_all = top_p_all;
  a.min_p = min_p;
  a.m_all = min_p_all;
  a.pieces = pieces_of(vocab);
  a.cells = cells_of(vocab);
  a.groups = groups_of(a.rows, a.pieces);
  a.row_bytes = row_record(a.pieces, a.cells);
  a.cnt = (int*)workspace;
  a.modes = (int*)((char*)workspace + kCounterBytes);
  a.records = (char*)workspace + kCounterBytes + modes_bytes(a.rows);
  a.rooms = (u64*)(a.records + (size_t)a.rows * a.row_bytes);
  a.shared_rows = shared_rows_of(a.rows, vocab);
  a.shared_groups = shared_groups_of(a.rows, a.pieces);
  a.cus = device_cus();
  return PA_OK;
}

int pa_sample_tokens(const void* logits, int dtype, const int64_t logits_strides[3],
                     const float* u, const int64_t u_strides[2], const float* temperature,
                     float temperature_all, const int32_t* top_k, int top_k_all,
                     const float* top_p, float top_p_all, const float* min_p, float min_p_all,
                     int64_t* tokens, int num_seqs, int rows_per_seq, int vocab, void* workspace,
                     size_t workspace_bytes, void* stream) {
  Args a{};
  const int status = start(a, logits, dtype, logits_strides, num_seqs, rows_per_seq, vocab,
                           temperature, temperature_all, top_k, top_k_all, top_p, top_p_all, min_p,
                           min_p_all, tokens, workspace, workspace_bytes);
  if (status != PA_OK || a.rows == 0) return status;
  if (!u || !u_strides) {
    set_error("null pointer argument");
    return PA_ERR_ARG;
  }
  a.u = u;
  a.u_seq = u_strides[0];
  a.u_row = u_strides[1];
  a.tokens = tokens;
  return run(a, dtype, (hipStream_t)stream);
}

int pa_sampling_probs(const void* logits, int dtype, const int64_t logits_strides[3],
                      const float* temperature, float temperature_all, const int32_t* top_k,
                      int top_k_all, const float* top_p, float top_p_all, const float* min_p,
                      float min_p_all, float* probs, int num_seqs, int rows_per_seq, int vocab,
                      void* workspace, size_t workspace_bytes, void* stream) {
  Args a{};
  const int status = start(a, logits, dtype, logits_strides, num_seqs, rows_per_seq, vocab,
                           temperature, temperature_all, top_k, top_k_all, top_p, top_p_all, min_p,
                           min_p_all, probs, workspace, workspace_bytes);
  if (status != PA_OK || a.rows == 0) return status;
  a.probs = probs;
  return run(a, dtype, (hipStream_t)stream);
}

}  // extern "C"
