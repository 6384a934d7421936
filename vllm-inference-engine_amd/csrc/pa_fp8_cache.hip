// Writing fp16 K/V rows into the 8-bit paged pool, and reading them back (gfx950).
//
// Write. For every block b, kv head h and cache that gets new rows x:
//   a = max |x| (each |x| kept at most 61440, NaN skipped)
//   e = smallest exponent of [-15, 8] with a <= 448 * 2^e; where rows before the
//       new ones stay in the block, at least the block's present exponent
//   code = e4m3(x * 2^-e), rounded to nearest even; the rows before are coded
//       again as e4m3(code * 2^(e_old - e)) where the exponent grew.
// With powers of two the product is exact, so a value is rounded once, and a row
// coded again changes only where its code falls below e4m3's normal range.
//
// One wavefront takes one (block, kv head, cache): the maximum is a reduction over
// its lanes, no other wavefront reads or writes that scale or those rows, and the
// fp16 rows are read once (up to 256 pieces of 16 bytes stay in registers between
// the maximum and the codes; each lane finds its pieces by steps, not divisions: prompts
// 18.2 -> 16.2 us in a graph). Bound by memory at prompts, by the chain length -> table
// entry -> scale -> store at single tokens. On MI355X: four prompts of 9.6k rows in all at
// 8 heads of 128 (59 MB) 15.4 us, 3.8 TB/s; a decode step's row for each of 128 sequences at 2
// heads of 64 4.3 us, little more than a launch.
#include "../../include/paged_attention.h"
#include "pa_fp8.h"

namespace pa {
namespace fp8 {

// |x| of a row's value for the maximum: NaN does not count, infinities are the
// largest value.
__device__ inline float finite_abs(float x) {
  return __builtin_fminf(__builtin_fmaxf(__builtin_fabsf(x), 0.f), kMaxValue);
}

// What is coded: NaN stays NaN, everything else is kept in range.
__device__ inline float in_range(float x) {
  return x != x ? x : __builtin_fminf(__builtin_fmaxf(x, -kMaxValue), kMaxValue);
}

// A piece is 8 values with VEC (16-byte source and 8-byte code accesses), else one.
template <bool VEC>
struct Piece;
template <>
struct Piece<true> {
  static constexpr int N = 8;
  f16x8 x;
  __device__ void load(const uint16_t* p) { x = *reinterpret_cast<const f16x8*>(p); }
  __device__ void store(uint8_t* p, float inv) const {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = in_range((float)x[i]) * inv;
    uint2 w;
    w.x = (unsigned)to_codes<true>(y[2], y[3], to_codes<false>(y[0], y[1], 0));
    w.y = (unsigned)to_codes<true>(y[6], y[7], to_codes<false>(y[4], y[5], 0));
    *reinterpret_cast<uint2*>(p) = w;
  }
  __device__ float amax() const {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = __builtin_fmaxf(m, finite_abs((float)x[i]));
    return m;
  }
  __device__ static void recode(uint8_t* p, float shift) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const f16x8 v = from_codes8(w.x, w.y, 1.f);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = (float)v[i] * shift;
    uint2 o;
    o.x = (unsigned)to_codes<true>(y[2], y[3], to_codes<false>(y[0], y[1], 0));
    o.y = (unsigned)to_codes<true>(y[6], y[7], to_codes<false>(y[4], y[5], 0));
    *reinterpret_cast<uint2*>(p) = o;
  }
};
template <>
struct Piece<false> {
  static constexpr int N = 1;
  f16 x;
  __device__ void load(const uint16_t* p) { x = *reinterpret_cast<const f16*>(p); }
  __device__ void store(uint8_t* p, float inv) const {
    *p = (uint8_t)to_codes<false>(in_range((float)x) * inv, 0.f, 0);
  }
  __device__ float amax() const { return finite_abs((float)x); }
  __device__ static void recode(uint8_t* p, float shift) {
    *p = (uint8_t)to_codes<false>((float)from_codes<false>(*p, 1.f)[0] * shift, 0.f, 0);
  }
};

template <bool VEC>
__global__ __launch_bounds__(256) void write_kernel(WriteArgs a) {
  typedef Piece<VEC> P;
  constexpr int HELD = 4;  // pieces per lane kept between the maximum and the codes
  const int lane = threadIdx.x & 63;
  const int unit = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per_slot = 2 * a.hkv;
  const int slot = unit / per_slot;
  if (slot >= a.slots) return;
  const int c = (unit - slot * per_slot) & 1;  // 0: keys, 1: values
  const int h = (unit - slot * per_slot) >> 1;
  const Rows& r = a.r;

  // Slots are numbered so that sequence b owns those from rows-before-b / bs + 2 b
  // on: its n rows touch at most n / bs + 2 blocks.
  const int b = r.qstart ? wave_search(r.num_seqs, slot, lane,
                                       [&](int i) { return row_start(r, i) / r.bs + 2 * i; })
                         : slot;
  const int q0 = row_start(r, b);
  const int n = row_start(r, b + 1) - q0;
  if (n <= 0) return;
  const int64_t L = r.lens[b];
  const int64_t from = L - n;  // position of the sequence's first new row
  const int p0 = from > 0 ? (int)from : 0;
  const int64_t blk = p0 / r.bs + (r.qstart ? slot - (q0 / r.bs + 2 * b) : 0);
  if (blk >= r.max_blocks) return;
  const int64_t lo = blk * r.bs > p0 ? blk * r.bs : p0;
  const int64_t hi = (blk + 1) * r.bs < L ? (blk + 1) * r.bs : L;
  if (lo >= hi) return;
  const int id = r.bt[(int64_t)b * r.bt_sb + blk * r.bt_sk];
  if (id < 0 || id >= r.num_blocks) return;
  const int r0 = (int)(lo - blk * r.bs);
  const int rows = (int)(hi - lo);

  const uint16_t* src = a.src[c] + (q0 + (lo - from)) * a.s_t[c] + (int64_t)h * a.s_h[c];
  uint8_t* dst = a.cache[c] + (int64_t)id * a.c_sb[c] + (int64_t)h * a.c_sh[c];
  float* sp = a.scale[c] + (int64_t)id * a.x_sb[c] + (int64_t)h * a.x_sh[c];
  const int e_old = r0 > 0 ? scale_exp(*sp) : kExpMin;

  // This lane's pieces are lane, lane + 64, ...; piece i is piece i % per_row of row
  // i / per_row. (The host sees to it that 31 bits hold a block's pieces.)
  const int per_row = a.D / P::N;
  const int pieces = rows * per_row;
  struct Place {
    int row, col;
  };
  const Place start{lane / per_row, lane % per_row};
  const int down = 64 / per_row, along = 64 % per_row;
  auto next = [&](Place& at) {
    at.row += down;
    at.col += along;
    if (at.col >= per_row) {
      at.col -= per_row;
      ++at.row;
    }
  };
  auto source = [&](Place at) { return src + at.row * a.s_t[c] + at.col * P::N * a.s_d[c]; };
  auto target = [&](Place at, int first) {
    return dst + (first + at.row) * a.c_st[c] + at.col * P::N;
  };
  P held[HELD];
  Place at[HELD];
  float m = 0.f;
  Place rest = start;
#pragma unroll
  for (int k = 0; k < HELD; ++k) {
    at[k] = rest;
    if (lane + 64 * k < pieces) held[k].load(source(rest));
    next(rest);
  }
#pragma unroll
  for (int k = 0; k < HELD; ++k)
    if (lane + 64 * k < pieces) m = __builtin_fmaxf(m, held[k].amax());
  Place more = rest;
  for (int i = lane + 64 * HELD; i < pieces; i += 64, next(more)) {
    P x;
    x.load(source(more));
    m = __builtin_fmaxf(m, x.amax());
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) m = __builtin_fmaxf(m, __shfl_xor(m, off));

  const int e_new = exp_for(m);
  const int e = e_old > e_new ? e_old : e_new;
  if (r0 > 0 && e > e_old) {
    const float shift = exp2i(e_old - e);
    more = start;
    for (int i = lane; i < r0 * per_row; i += 64, next(more)) P::recode(target(more, 0), shift);
  }
  const float inv = exp2i(-e);
#pragma unroll
  for (int k = 0; k < HELD; ++k)
    if (lane + 64 * k < pieces) held[k].store(target(at[k], r0), inv);
  for (int i = lane + 64 * HELD; i < pieces; i += 64, next(rest)) {
    P x;
    x.load(source(rest));
    x.store(target(rest, r0), inv);
  }
  if (lane == 0) *sp = exp2i(e);
}

// Read. A workgroup takes 16 output rows. Each row's sequence, block and row in the
// block are found once (16 lanes, the first row's sequence by a wavefront search and
// the others' from there) and kept in LDS; then the threads take 16-code pieces of
// the rows' keys and values. Rows without a slot are written as zeros. Bound by
// memory: one byte read and two written per value. On MI355X 37.5k rows at 8 heads of 128
// (231 MB) in 57.7 us, 4.0 TB/s where a large copy reaches 4.75; 8192 rows at 2 heads of 64
// (6.3 MB) in 5.4. Two, four or eight pieces per
// thread on their way at a time (54.1 us for 51.9 in a graph), and stores past the caches
// (54.5), were slower than one piece after the other in many workgroups.
constexpr int kReadRows = 16;

template <bool VEC>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a) {
  constexpr int N = VEC ? 16 : 1;
  __shared__ int s_id[kReadRows], s_off[kReadRows];
  const Rows& r = a.r;
  const int lane = threadIdx.x & 63;
  const int first = blockIdx.x * kReadRows;
  const int rows = r.num_tokens - first < kReadRows ? r.num_tokens - first : kReadRows;
  if (threadIdx.x < 64) {
    int b = wave_search(r.num_seqs, first, lane, [&](int i) { return row_start(r, i); });
    if (lane < rows) {
      int id = -1, off = 0;
      if (r.num_seqs > 0) {
        const int t = first + lane;
        while (b + 1 < r.num_seqs && row_start(r, b + 1) <= t) ++b;
        const int q0 = row_start(r, b), q1 = row_start(r, b + 1);
        const int64_t pos = (int64_t)r.lens[b] - (q1 - q0) + (t - q0);
        const int64_t blk = pos / r.bs;
        if (t >= q0 && t < q1 && pos >= 0 && blk < r.max_blocks) {
          id = r.bt[(int64_t)b * r.bt_sb + blk * r.bt_sk];
          if (id >= r.num_blocks) id = -1;
          off = (int)(pos - blk * r.bs);
        }
      }
      s_id[lane] = id;
      s_off[lane] = off;
    }
  }
  __syncthreads();
  const int per_head = a.D / N;
  const int per_row = a.hkv * per_head;
  const int per_cache = rows * per_row;
  for (int i = threadIdx.x; i < 2 * per_cache; i += 256) {
    const int c = i >= per_cache;
    const int j = i - c * per_cache;
    const int row = j / per_row;
    const int k = j - row * per_row;
    const int h = k / per_head;
    const int d = (k - h * per_head) * N;
    const int id = s_id[row];
    f16* o = a.out[c] + (int64_t)(first + row) * a.o_t[c] + (int64_t)h * a.o_h[c] + d;
    const uint8_t* p = a.cache[c] + (int64_t)id * a.c_sb[c] + (int64_t)s_off[row] * a.c_st[c] +
                       (int64_t)h * a.c_sh[c] + d;
    const float* sp = a.scale[c] + (int64_t)id * a.x_sb[c] + (int64_t)h * a.x_sh[c];
    if constexpr (VEC) {
      f16x8 lo = {0, 0, 0, 0, 0, 0, 0, 0}, hi = lo;
      if (id >= 0) {
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        const float s = *sp;
        lo = from_codes8(w.x, w.y, s);
        hi = from_codes8(w.z, w.w, s);
      }
      *reinterpret_cast<f16x8*>(o) = lo;
      *reinterpret_cast<f16x8*>(o + 8) = hi;
    } else {
      *o = id >= 0 ? from_codes<false>(*p, *sp)[0] : (f16)0.f;
    }
  }
}

// ---- argument checks and the C entry points ----

static bool multiple(const void* p, size_t n) { return (uintptr_t)p % n == 0; }

// The description of rows and positions; a PA_* status with the message set.
static int rows_args(Rows& r, const int32_t* block_tables, const int64_t* bt_strides,
                     const int32_t* seq_lens, const int32_t* query_start_loc, int num_seqs,
                     int num_tokens, int num_kv_heads, int head_dim, int block_size,
                     int num_blocks, int max_blocks_per_seq) {
  if (num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || num_blocks <= 0 ||
      max_blocks_per_seq <= 0) {
    set_error("num_kv_heads, head_dim, block_size, num_blocks and the table width must be "
              "positive");
    return PA_ERR_ARG;
  }
  if (!block_tables || !bt_strides || !seq_lens) {
    set_error("null pointer argument");
    return PA_ERR_ARG;
  }
  r = Rows{block_tables, bt_strides[0], bt_strides[1], seq_lens,   query_start_loc,
           num_seqs,     num_tokens,    block_size,    num_blocks, max_blocks_per_seq};
  return PA_OK;
}

static int launched() {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return PA_OK;
  set_error("HIP launch failed: %s", hipGetErrorString(e));
  return PA_ERR_HIP;
}

}  // namespace fp8
}  // namespace pa

using namespace pa;
using namespace pa::fp8;

extern "C" {

int pa_kv_write_fp8(const void* key, const int64_t key_strides[3], const void* value,
                    const int64_t value_strides[3], void* k_cache, const int64_t k_strides[4],
                    void* v_cache, const int64_t v_strides[4], float* k_scale,
                    const int64_t k_scale_strides[2], float* v_scale,
                    const int64_t v_scale_strides[2], const int32_t* block_tables,
                    const int64_t bt_strides[2], const int32_t* seq_lens,
                    const int32_t* query_start_loc, int num_seqs, int num_tokens,
                    int num_kv_heads, int head_dim, int block_size, int num_blocks,
                    int max_blocks_per_seq, void* stream) {
  clear_error();
  if (num_seqs < 0 || num_tokens < 0 || (!query_start_loc && num_seqs != num_tokens)) {
    set_error("num_seqs (%d) and num_tokens (%d) must be >= 0, and equal without "
              "query_start_loc", num_seqs, num_tokens);
    return PA_ERR_ARG;
  }
  if (num_seqs == 0 || num_tokens == 0) return PA_OK;
  if (!key || !value || !k_cache || !v_cache || !k_scale || !v_scale || !key_strides ||
      !value_strides || !k_strides || !v_strides || !k_scale_strides || !v_scale_strides) {
    set_error("null pointer argument");
    return PA_ERR_ARG;
  }
  WriteArgs a{};
  const int rc = rows_args(a.r, block_tables, bt_strides, seq_lens, query_start_loc, num_seqs,
                           num_tokens, num_kv_heads, head_dim, block_size, num_blocks,
                           max_blocks_per_seq);
  if (rc) return rc;
  if (k_strides[3] != 1 || v_strides[3] != 1) {
    set_error("cache head_dim stride must be 1");
    return PA_ERR_ARG;
  }
  const void* src[2] = {key, value};
  void* cache[2] = {k_cache, v_cache};
  float* scale[2] = {k_scale, v_scale};
  const int64_t* ss[2] = {key_strides, value_strides};
  const int64_t* cs[2] = {k_strides, v_strides};
  const int64_t* xs[2] = {k_scale_strides, v_scale_strides};
  bool vec = head_dim % 8 == 0;
  for (int i = 0; i < 2; ++i) {
    a.src[i] = (const uint16_t*)src[i];
    a.s_t[i] = ss[i][0];
    a.s_h[i] = ss[i][1];
    a.s_d[i] = ss[i][2];
    a.cache[i] = (uint8_t*)cache[i];
    a.c_sb[i] = cs[i][0];
    a.c_st[i] = cs[i][1];
    a.c_sh[i] = cs[i][2];
    a.scale[i] = scale[i];
    a.x_sb[i] = xs[i][0];
    a.x_sh[i] = xs[i][1];
    vec = vec && ss[i][2] == 1 && ss[i][0] % 8 == 0 && ss[i][1] % 8 == 0 && cs[i][0] % 8 == 0 &&
          cs[i][1] % 8 == 0 && cs[i][2] % 8 == 0 && multiple(src[i], 16) && multiple(cache[i], 8);
  }
  a.hkv = num_kv_heads;
  a.D = head_dim;
  const int64_t slots =
      query_start_loc ? (int64_t)num_tokens / block_size + 2 * (int64_t)num_seqs : num_seqs;
  // (Also in the kernel's 31-bit counts of units and of a block's values.)
  if (slots > 0x3ffffff0 || slots * num_kv_heads > 0x3ffffff0 || (int64_t)block_size * head_dim > 0x7fffff00) {
    set_error("%lld blocks of %d kv heads, %d rows of %d values each, exceed one launch",
              (long long)slots, num_kv_heads, block_size, head_dim);
    return PA_ERR_UNSUPPORTED;
  }
  const int64_t grid = (slots * num_kv_heads * 2 + 3) / 4;
  a.slots = (int)slots;
  if (vec)
    write_kernel<true><<<(unsigned)grid, 256, 0, (hipStream_t)stream>>>(a);
  else
    write_kernel<false><<<(unsigned)grid, 256, 0, (hipStream_t)stream>>>(a);
  return launched();
}

int pa_kv_read_fp8(const void* k_cache, const int64_t k_strides[4], const void* v_cache,
                   const int64_t v_strides[4], const float* k_scale,
                   const int64_t k_scale_strides[2], const float* v_scale,
                   const int64_t v_scale_strides[2], const int32_t* block_tables,
                   const int64_t bt_strides[2], const int32_t* seq_lens,
                   const int32_t* query_start_loc, void* key, const int64_t key_strides[3],
                   void* value, const int64_t value_strides[3], int num_seqs, int num_tokens,
                   int num_kv_heads, int head_dim, int block_size, int num_blocks,
                   int max_blocks_per_seq, void* stream) {
  clear_error();
  if (num_seqs < 0 || num_tokens < 0) {
    set_error("num_seqs (%d) and num_tokens (%d) must be >= 0", num_seqs, num_tokens);
    return PA_ERR_ARG;
  }
  // Rows of no sequence are zeros, without any sequence too; of the other arguments nothing
  // is then asked (tables of no rows have null pointers).
  const bool none = num_seqs == 0;
  if (num_tokens == 0 ||
      (none && (!key || !value || !key_strides || !value_strides || num_kv_heads <= 0 || head_dim <= 0)))
    return PA_OK;
  if (!none && (!key || !value || !k_cache || !v_cache || !k_scale || !v_scale || !key_strides ||
                !value_strides || !k_strides || !v_strides || !k_scale_strides ||
                !v_scale_strides || !query_start_loc)) {
    set_error("null pointer argument");
    return PA_ERR_ARG;
  }
  ReadArgs a{};
  if (none) {
    a.r.num_tokens = num_tokens;
  } else {
    const int rc = rows_args(a.r, block_tables, bt_strides, seq_lens, query_start_loc, num_seqs,
                             num_tokens, num_kv_heads, head_dim, block_size, num_blocks,
                             max_blocks_per_seq);
    if (rc) return rc;
  }
  if ((!none && (k_strides[3] != 1 || v_strides[3] != 1)) || key_strides[2] != 1 ||
      value_strides[2] != 1) {
    set_error("the head_dim stride of the caches, key and value must be 1");
    return PA_ERR_ARG;
  }
  if ((int64_t)num_kv_heads * head_dim > (1 << 24)) {
    set_error("%d kv heads x head_dim %d is not built", num_kv_heads, head_dim);
    return PA_ERR_UNSUPPORTED;
  }
  const int64_t no_strides[4] = {};
  const void* cache[2] = {none ? nullptr : k_cache, none ? nullptr : v_cache};
  const float* scale[2] = {none ? nullptr : k_scale, none ? nullptr : v_scale};
  void* out[2] = {key, value};
  const int64_t* os[2] = {key_strides, value_strides};
  const int64_t* cs[2] = {none ? no_strides : k_strides, none ? no_strides : v_strides};
  const int64_t* xs[2] = {none ? no_strides : k_scale_strides, none ? no_strides : v_scale_strides};
  bool vec = head_dim % 16 == 0;
  for (int i = 0; i < 2; ++i) {
    a.cache[i] = (const uint8_t*)cache[i];
    a.c_sb[i] = cs[i][0];
    a.c_st[i] = cs[i][1];
    a.c_sh[i] = cs[i][2];
    a.scale[i] = scale[i];
    a.x_sb[i] = xs[i][0];
    a.x_sh[i] = xs[i][1];
    a.out[i] = (f16*)out[i];
    a.o_t[i] = os[i][0];
    a.o_h[i] = os[i][1];
    vec = vec && cs[i][0] % 16 == 0 && cs[i][1] % 16 == 0 && cs[i][2] % 16 == 0 &&
          os[i][0] % 8 == 0 && os[i][1] % 8 == 0 && multiple(cache[i], 16) && multiple(out[i], 16);
  }
  a.hkv = num_kv_heads;
  a.D = head_dim;
  const unsigned grid = (unsigned)(((int64_t)num_tokens + kReadRows - 1) / kReadRows);
  if (vec)
    read_kernel<true><<<grid, 256, 0, (hipStream_t)stream>>>(a);
  else
    read_kernel<false><<<grid, 256, 0, (hipStream_t)stream>>>(a);
  return launched();
}

}  // extern "C"
