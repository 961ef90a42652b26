// Causal grouped-query attention over an 8-bit cache (cache8.h), for a step's few rows a sequence and for prompts, with an optional window.
//
// Row r of a sequence with n new rows and k_len keys stands at p = k_len - n + r and sees the keys lo..p, lo = 0 or p - window + 1.  q head h reads kv head
// h / (nq / nkv).  With c = scale * log2(e):  m = max of (q.k) c over the keys seen;  w = 2^((q.k) c - m);  out = sum w v / sum w (0 for a row that sees none).
//
// A wave computes S^T = K Q^T and O^T = V^T P^T with 16 columns a tile: the rows of an item times the q heads of a kv head, so that what is read of the cache
// serves all of them.  64 keys a tile.  Lane l (r = l % 16, g = l / 16) reads 16 bytes at a time of both: of K the entries 16 g .. 16 g + 15 (+ 64 j) of key
// 16 (r / 4) + 4 t + r % 4 for t = 0..3, of V the keys 16 g .. 16 g + 15 of entry 16 dt + r.  K's rows are taken in that order so that the scores that a lane ends with
// (rows 4 g + i of S^T's tile t) are those of the keys 16 g + 4 t + i: the lane's own 16 keys of V, and no weight has to change lanes between the products.
//
// Arithmetic.  A key's entry times its scale is exact in the element type, so the first product takes q as it is and 32-bit sums.  Where tiles are 128 or 256 entries wide (heads of 80 to 128 and of 208 to 256) it takes the keys as they are
// stored, and q as two e4m3 numbers of four digits each in units of the head's largest entry: they hold its eight digits where it is 2^-14 of the largest's power of two or more, and are off by
// 2^-22 of that power at most elsewhere; products of twice the rate make up for there being two, and no key has to be turned into an operand (a prompt of 4,096 rows 186 -> 163 us; of heads of 64 the
// product, 128 entries long, would be half empty).  Weights go into the
// second product in 16-bit floating point with eleven digits down to 2^-21 of the column's largest, and off by 2^-32 of that at most below (A8_LOW), against values without their scale, which
// they hold to the bit: bfloat16 weights, with eight, would double the squared error of the result.  Values' scales stand in the product's entries relative to a unit of the wave's sums
// that follows the tile's (A8_UNIT_DOWN); pages of scales 2^11 apart and more in one tile are multiplied one after the other.  So a row's values keep their digits whatever stands in other
// pages, up to scales 2^75 below the largest that the wave's columns see.  The 32-bit build takes everything in 32 bits.  The sum of the weights comes from the matrix
// unit too, a product with ones: it is that of the very weights that the values are multiplied by, and the vector unit has enough to do.
//
// Keys that a row does not see weigh 0, whatever is stored: their scores are never used, and values outside what the wave's rows see, or NaN, are
// taken out of the second product of a tile that not all rows see whole; a row that does see a NaN gets it back through a product of its own.
//
// What bounds it (MI355X, bfloat16, heads of 128, 8 kv heads; reading alone reaches 6.45 TB/s here, a large bfloat16 product 1.45 PFLOP/s): 64 rows with 8,192 keys each, 32 heads, 1.08 GB
// of cache: 188 us, 5.7 TB/s, and 5 us for the join: bytes.  13 sequences of 5 rows and up to 4,096 keys, 64 heads, 73 MB: 26 us and 5: 592 workgroups with keys, all of them on the card at
// once, each eight tiles one after the other.  A prompt of 4,096 rows over itself, 32 heads, 137 GFLOP: 159 us, 140 in a row of calls, 0.87 to 0.99 PFLOP/s: a wave's products
// and the exponentials behind them follow each other, and its registers leave room for two waves a unit.  Portions of 5 prompts, 2,625 rows in all, windows of 1,024, pages of 16, 49 GFLOP: 99 us, 92 in a row:
// 16 to 18 tiles each for 792 workgroups on 512 places, two rounds of them where one and a half are needed; pages of 64 take 3 us off it.  A single row with 333 keys: 10 us, loads that wait for each other.
#include <type_traits>

#include "cache8.h"
#include "lines.h"
#include "mma.h"
#include "vec.h"

#define A8_TILE 64
#define A8_SEG 512               // keys that are summed up apart where a row's keys are split over workgroups
// A column's reference, log2: A8_LOW below the maximum that set it, and it moves where a tile's maximum stands more than A8_STEP above it, 8 above the one that set it.  Weights of 16 bits are then 2^15 at
// most (and no more than 2^15.2 with the rounding of a maximum below 2^22); they hold eleven digits down to 2^-21 of the largest and are off by half of 2^-24, 2^-32 of the largest, below that.  With references that
// are the maximum itself it was 2^-25: 4,096 keys that stand that far behind one whose value is 0 gave a result off by 2 % and more.
#ifdef VK_BF16
#define A8_LOW 7.0f
#define A8_PART 0.0078125f        // 2^-A8_LOW: of sums that meet others, which may be 32-bit numbers of the values' own size
#define A8_STEP 15.0f
#define A8_FAR 4194304.0f         // 2^22
#else
#define A8_LOW 0.0f
#define A8_PART 1.0f
#define A8_STEP 8.0f
#define A8_FAR 67108864.0f        // 2^26
#endif
#define A8_NONE -3.0e38f          // the reference maximum of a column that has seen no key: finite, so that differences with it are numbers
// Values go into their product in 16-bit floating point, in units of 2^unit, and an e4m3 number is a whole multiple of 2^-9 of its scale, 448 of it at most: of scales from 2^-15 to 2^6 of the unit it
// is held to the bit (2^-24 is the least such number).  The unit stays while a tile's largest scale is from 2^-4 to 2^6 of it, so that scales 2^11 apart need no second pass; it falls by
// 2^60 at most, so that sums in larger units remain numbers in smaller ones.
#define A8_UNIT_UP 6
#define A8_UNIT_STAYS 4
#define A8_UNIT_DOWN 15
#define A8_UNIT_FALLS 60
#define A8_STAGES 2               // tiles in LDS: one is computed, the next is arriving.  A third changed nothing for prompts (155 us for 4,096 rows both ways) and keeps workgroups of split keys from
                                  // the CU (5 rows each, 32 heads of 128, 32 sequences of 4,000 keys: 79 us against 72; 13 of 4,096 43 against 36; of unequal lengths 52 against 50)
#define A8_ITEM_ROWS 128         // rows of an item, at most

struct A8Args {
  const elem_t* q;          // [T, nq, d]
  elem_t* out;
  const uint8_t *kc, *vc;
  const float* scales;
  const int32_t *table, *cu_q, *k_len, *items;
  float *part_ml, *part_acc;   // per (item, kv head, segment of the column's block from its first on, column): reference and sum; d sums
  int W, T, S, nq, nkv, d, P, lp, pages, group, item_rows, cols_max, window, nseg, n_items, max_keys;
  float scale_log2;
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// Over the lanes l, l ^ 16, l ^ 32, l ^ 48, in every one of them.
__device__ __forceinline__ float over_groups_max(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const unsigned a = r[0], b = r[1], w = __builtin_bit_cast(unsigned, fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));
  const auto q = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  const unsigned c = q[0], e = q[1];
  return fmaxf(__builtin_bit_cast(float, c), __builtin_bit_cast(float, e));
}

// ---- operands of the two products
#ifdef VK_BF16
#define A8_QJ 2                                   // q registers a 16-entry piece: 8 entries each
typedef bf16x8 q_part;
typedef f16x8 w_part;                             // weights of 8 keys
#define A8_WP 2
__device__ __forceinline__ bf16x8 keys_of(uint32_t a, uint32_t b, float scale) {
  const bf16x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, false), p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, true);
  const bf16x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, false), p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, true);
  return bf16x8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}
__device__ __forceinline__ f16x8 values_of(uint32_t a, uint32_t b, float scale) {
  const f16x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, scale, false), p1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, scale, true);
  const f16x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, scale, false), p3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, scale, true);
  return f16x8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}
template <int NT>
__device__ __forceinline__ void keys_times(u32x4 raw, float scale, const q_part (&q)[NT][A8_QJ], f32x4 (&s)[NT]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const bf16x8 k = keys_of(raw[2 * h], raw[2 * h + 1], scale);
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[n][h], s[n], 0, 0, 0);
  }
}
typedef __attribute__((ext_vector_type(8))) int i32x8;
__device__ __forceinline__ i32x8 two_pieces(u32x4 a, u32x4 b) { return i32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]}; }
template <int NT>
__device__ __forceinline__ void keys_times8(u32x4 a, u32x4 b, int k_exp, const q_part (&qa)[NT][A8_QJ], const q_part (&qb)[NT][A8_QJ], const int (&q_exp)[NT], f32x4 (&s)[NT]) {
  const i32x8 k = two_pieces(a, b);
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int n = 0; n < NT; ++n)
      s[n] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, two_pieces(__builtin_bit_cast(u32x4, qa[n][h]), __builtin_bit_cast(u32x4, qb[n][h])), s[n], 0, 0, 0, k_exp, 0,
                                                              q_exp[n] - 5 * h);
}
template <int NT>
__device__ __forceinline__ void values_times(u32x4 raw, float scale, const w_part (&w)[NT][A8_WP], f32x4 (&o)[NT]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f16x8 v = values_of(raw[2 * h], raw[2 * h + 1], scale);
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, w[n][h], o[n], 0, 0, 0);
  }
}
// The sum of the weights of a column, in every row of the result.
template <int NT>
__device__ __forceinline__ void ones_times(const w_part (&w)[NT][A8_WP], f32x4 (&o)[NT]) {
  const _Float16 one = (_Float16)1.f;
  const f16x8 ones = {one, one, one, one, one, one, one, one};
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, w[n][h], o[n], 0, 0, 0);
}
__device__ __forceinline__ void set_weights(const float (&p)[16], w_part (&w)[A8_WP]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 8; ++e) w[h][e] = (_Float16)p[8 * h + e];
}
#else
#define A8_QJ 16
typedef float q_part;
typedef float w_part;
#define A8_WP 16
template <int NT>
__device__ __forceinline__ void bytes_times(u32x4 raw, float scale, const float (&b)[NT][16], f32x4 (&c)[NT]) {
#pragma unroll
  for (int e = 0; e < 16; e += 4) {
    const f32x2 lo = from_fp8x2<false>(raw[e / 4], scale), hi = from_fp8x2<true>(raw[e / 4], scale);
    const float x[4] = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n) c[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], b[n][e + i], c[n], 0, 0, 0);
  }
}
template <int NT>
__device__ __forceinline__ void keys_times(u32x4 raw, float scale, const q_part (&q)[NT][A8_QJ], f32x4 (&s)[NT]) { bytes_times<NT>(raw, scale, q, s); }
template <int NT>
__device__ __forceinline__ void values_times(u32x4 raw, float scale, const w_part (&w)[NT][A8_WP], f32x4 (&o)[NT]) { bytes_times<NT>(raw, scale, w, o); }
template <int NT>
__device__ __forceinline__ void ones_times(const w_part (&w)[NT][A8_WP], f32x4 (&o)[NT]) {
#pragma unroll
  for (int e = 0; e < 16; ++e)
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(1.f, w[n][e], o[n], 0, 0, 0);
}
__device__ __forceinline__ void set_weights(const float (&p)[16], w_part (&w)[A8_WP]) {
#pragma unroll
  for (int e = 0; e < 16; ++e) w[e] = p[e];
}
#endif

// An item's columns as one wave sees them: column col0 + 16 n + r of its rows times the kv head's q heads.
template <int NT>
struct A8Rows {
  int seq, tok0, rows, cols, col0, pos0, kvh, r, g;
  int wave_lo, wave_pos, all_lo, all_pos;    // first and last key that some column sees; that all columns see
  int lo[NT], pos[NT];                       // this lane's columns see lo..pos (none: pos = -1)
};

// False: there is nothing to do.  item: which; head_cols: kv head and block of 16 NT * waves columns; col_wave: the wave's first column in the block.
template <int NT>
__device__ __forceinline__ bool a8_rows(const A8Args& a, int item, int kvh, int col0, A8Rows<NT>& c) {
  const int lane = threadIdx.x & 63;
  c.r = lane & 15;
  c.g = lane >> 4;
  c.kvh = kvh;
  // (Read first lane: the same for the wave, which the compiler cannot know of what is loaded.)
  c.seq = __builtin_amdgcn_readfirstlane(a.items[2 * item]);
  const int first = __builtin_amdgcn_readfirstlane(a.items[2 * item + 1]);
  if ((unsigned)c.seq >= (unsigned)a.S || first < 0) return false;
  const int t0 = __builtin_amdgcn_readfirstlane(a.cu_q[c.seq]), t1 = __builtin_amdgcn_readfirstlane(a.cu_q[c.seq + 1]);
  if (t0 < 0 || t1 > a.T || t1 <= t0 || first >= t1 - t0) return false;
  c.rows = min(a.item_rows, t1 - t0 - first);
  c.cols = c.rows * a.group;
  c.col0 = col0;
  if (col0 >= c.cols) return false;
  c.tok0 = t0 + first;
  c.pos0 = max(__builtin_amdgcn_readfirstlane(a.k_len[c.seq]), 0) - (t1 - t0) + first;
  // Keys from max_keys on are not looked for, whatever k_len says: neither the table nor the launch has a place for them.
  const int row_first = col0 / a.group, row_last = (min(c.cols, col0 + 16 * NT) - 1) / a.group, end = a.max_keys - 1;
  c.all_pos = min(c.pos0 + row_first, end);
  c.wave_pos = min(c.pos0 + row_last, end);
  c.wave_lo = a.window > 0 ? max(0, c.pos0 + row_first - a.window + 1) : 0;
  c.all_lo = a.window > 0 ? max(0, c.pos0 + row_last - a.window + 1) : 0;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = col0 + 16 * n + c.r;
    const int pos = c.pos0 + col / a.group;
    c.pos[n] = col < c.cols ? min(pos, end) : -1;
    c.lo[n] = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  }
  return true;
}

// q of the wave's columns: entries 64 j + 16 g + .. of each.  EIGHT: as two 8-bit numbers each, all first ones of the 16, then all second ones, with the exponent (+ 127) of what the first ones of a
// column stand in.
template <int DP, int NT>
struct A8Query {
#ifdef VK_BF16
  static constexpr bool EIGHT = DP % 128 == 0;
#else
  static constexpr bool EIGHT = false;
#endif
  q_part q[DP / 64][NT][A8_QJ];
  int exp[NT];
};
#ifdef VK_BF16
template <int DP, int NT>
__device__ __forceinline__ void a8_split_q(A8Query<DP, NT>& q) {
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < DP / 64; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf((float)q.q[j][n][e / 8][e % 8]));
    const int e7 = max(exponent_of(over_groups_max(top)), -100) - 7;
    q.exp[n] = e7 + 127;
    const float by = pow2f(-e7);
#pragma unroll
    for (int j = 0; j < DP / 64; ++j) {
      u32x4 hi, lo;
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = (float)q.q[j][n][p / 2][4 * (p & 1) + i] * by;
          x[i] = fabsf(v) < INFINITY ? v : NAN;
        }
        hi[p] = to_fp8x4(x[0], x[1], x[2], x[3]);
        const f32x2 a = from_fp8x2<false>(hi[p], 1.f), b = from_fp8x2<true>(hi[p], 1.f);
        lo[p] = to_fp8x4((x[0] - a.x) * 32.f, (x[1] - a.y) * 32.f, (x[2] - b.x) * 32.f, (x[3] - b.y) * 32.f);
      }
      q.q[j][n][0] = __builtin_bit_cast(bf16x8, hi);
      q.q[j][n][1] = __builtin_bit_cast(bf16x8, lo);
    }
  }
}
#endif
template <int DP, int NT>
__device__ __forceinline__ void a8_load_q(const A8Args& a, const A8Rows<NT>& c, A8Query<DP, NT>& to) {
  q_part (&q)[DP / 64][NT][A8_QJ] = to.q;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = c.col0 + 16 * n + c.r, row = min(col, c.cols - 1) / a.group, head = min(col, c.cols - 1) - row * a.group;
    const elem_t* p = a.q + ((int64_t)(c.tok0 + row) * a.nq + c.kvh * a.group + head) * a.d;
#pragma unroll
    for (int j = 0; j < DP / 64; ++j) {
      const int at = 64 * j + 16 * c.g;
      const bool ok = col < c.cols && at < a.d;
#ifdef VK_BF16
      q[j][n][0] = load_frag(p + at, ok);
      q[j][n][1] = load_frag(p + at + 8, ok);
#else
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const f32x4 v = load_frag(p + at + e, ok);
        q[j][n][e] = v.x; q[j][n][e + 1] = v.y; q[j][n][e + 2] = v.z; q[j][n][e + 3] = v.w;
      }
#endif
    }
  }
}

// q has arrived (and is split): waited for in front of a loop, so that no wait for it stands inside, where it would be one for all loads under way.
template <int DP, int NT>
__device__ __forceinline__ void a8_wait_q(A8Query<DP, NT>& to) {
#ifdef VK_BF16
  if constexpr (A8Query<DP, NT>::EIGHT) a8_split_q<DP, NT>(to);
#endif
  q_part (&q)[DP / 64][NT][A8_QJ] = to.q;
#pragma unroll
  for (int j = 0; j < DP / 64; ++j)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < A8_QJ; ++e) asm volatile("" : "+v"(q[j][n][e]));
}

// Bytes of four that hold a NaN, as 0x01 each.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u; }

// A column's sums: m its reference maximum, l the sum of its weights, acc those of weights times values in units of 2^unit (the same for the wave).
template <int DP, int NT>
struct A8Sums {
  float m[NT];
  f32x4 l[NT];                 // the same number in all four
  f32x4 acc[NT][DP / 16];
  typename std::conditional<(DP > 128), uint64_t, uint32_t>::type bad[NT];     // bit 4 dt + i: acc[n][dt][i] is NaN, by a value that is (where tiles are in registers; else it is set so)
  int unit, least_unit;
  __device__ __forceinline__ void clear() {
    unit = least_unit = -256;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n] = A8_NONE;
      bad[n] = 0;
      l[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int dt = 0; dt < DP / 16; ++dt) acc[n][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  // acc[n][dt] times a number.
  __device__ __forceinline__ f32x4 times(int n, int dt, float by) const {
    f32x4 x = acc[n][dt] * by;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (bad[n] >> (4 * dt + i) & 1) ? NAN : x[i];
    return x;
  }
  __device__ __forceinline__ float scale() const {
#ifdef VK_BF16
    return unit > -256 ? pow2f(unit) : 1.f;
#else
    return 1.f;
#endif
  }
  // For values whose largest scale is 2^top (-256: there are none): the unit that suits them, and the least exponent that goes with it.  What lies below it takes a pass of its own.
#ifdef VK_BF16
  __device__ __forceinline__ int next_unit(int top) const {
    const int to = unit == -256 || top > unit + A8_UNIT_UP ? top : top == -256 || top >= unit - A8_UNIT_STAYS ? unit : max(top, least_unit);
    return __builtin_amdgcn_readfirstlane(to);
  }
  __device__ __forceinline__ static int least_exponent(int next, int top) { return top < next - A8_UNIT_DOWN ? -255 : next - A8_UNIT_DOWN; }
#else
  __device__ __forceinline__ int next_unit(int) const { return 0; }
  __device__ __forceinline__ static int least_exponent(int, int) { return -255; }
#endif
};

// The scores of a tile: S^T's, unscaled.  src.k(i, j): the lane's 16 bytes of K's tile i; k_scale: of the keys that they belong to.
template <int DP, int NT, typename SRC>
__device__ __forceinline__ void a8_scores(const SRC& src, float k_scale, const A8Query<DP, NT>& q, f32x4 (&s)[4][NT]) {
  // What a product reads is asked for one product ahead, and not further: the scheduler would take all of a tile first, and spill.
  u32x4 next[DP / 64];
#pragma unroll
  for (int j = 0; j < DP / 64; ++j) next[j] = src.k(0, j);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    u32x4 k[DP / 64];
#pragma unroll
    for (int j = 0; j < DP / 64; ++j) {
      k[j] = next[j];
      if (i < 3) next[j] = src.k(i + 1, j);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) s[i][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < DP / 64; ++j) {
#ifdef VK_BF16
      if constexpr (A8Query<DP, NT>::EIGHT) {
        if (j % 2 == 0) keys_times8<NT>(k[j], k[j + 1], (int)(__builtin_bit_cast(uint32_t, k_scale) >> 23), q.q[j], q.q[j + 1], q.exp, s[i]);
        continue;
      }
#endif
      keys_times<NT>(k[j], k_scale, q.q[j], s[i]);
    }
    asm volatile("" ::: "memory");
  }
}

// A tile's scores and values onto the wave's sums.  src.v(dt): the lane's 16 bytes of V's entries 16 dt + r; v_exp: of the 16 keys that they belong to, -256: none of them is there;
// unit: next_unit() of the wave's largest.
//
// A column's reference follows its maximum only where that is more than 2^8 above the one that set it (A8_STEP): the sums are scaled in few tiles.  Which columns move is each column's own business; whether any does is the wave's.
// WHOLE: 1: every column that stands for a row sees every key; 0: not so; 2: unknown, and found out for the values.  (What is only done under a condition must not touch scores and sums:
// where the ways meet again they would be copied, and held twice.  A loop for each kind of tile in place of a condition: 225 -> 196 us for a prompt of 4,096 rows.)
template <int WHOLE, int DP, int NT, typename SRC>
__device__ __forceinline__ void a8_weigh(const A8Args& a, const A8Rows<NT>& c, int kb, const SRC& src, f32x4 (&s)[4][NT], int v_exp, int unit, A8Sums<DP, NT>& o) {
  const bool there = v_exp > -256;
  const bool full = WHOLE == 1 || (WHOLE == 2 && kb >= c.all_lo && kb + A8_TILE - 1 <= c.all_pos && __all(there));
  const int first = kb + 16 * c.g;
  float m_tile[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float top = -INFINITY;
    const int lo = c.lo[n] - first, pos = there ? c.pos[n] - first : -1;
    if (WHOLE == 1) {
#pragma unroll
      for (int x = 0; x < 16; ++x) top = fmaxf(top, s[x / 4][n][x % 4]);
    } else {
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const float v = x >= lo && x <= pos ? s[x / 4][n][x % 4] : -INFINITY;
        s[x / 4][n][x % 4] = v;
        top = fmaxf(top, v);
      }
    }
    m_tile[n] = over_groups_max(top) * a.scale_log2;
  }
  auto is_far = [&](int n) { return fabsf(m_tile[n]) >= A8_FAR && (WHOLE == 1 || m_tile[n] != -INFINITY); };      // -inf: no key
  bool moves = false, far = false;
  float by[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const bool move = m_tile[n] - o.m[n] > A8_STEP;      // (the difference of neighbours is exact, a sum with the step is not)
    const float to = move ? m_tile[n] - A8_LOW : o.m[n];
    by[n] = exp2_fast(o.m[n] - to);
    o.m[n] = to;
    moves = moves || move;
    far = far || is_far(n);
  }
#ifdef VK_BF16
  const float to_unit = o.unit - unit < -126 ? 0.f : pow2f(o.unit - unit), v_scale = pow2f(max(-126, v_exp - unit));
  moves = moves || unit != o.unit;
  o.unit = unit;
  o.least_unit = max(o.least_unit, unit - A8_UNIT_FALLS);
#else
  const float to_unit = 1.f, v_scale = there ? pow2f(v_exp) : 1.f;
#endif
  float from[NT];                                       // what is taken from the scores
#pragma unroll
  for (int n = 0; n < NT; ++n) from[n] = o.m[n];
  if (__any(moves || far)) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      o.l[n] = o.l[n] * by[n];
#pragma unroll
      for (int dt = 0; dt < DP / 16; ++dt) o.acc[n][dt] = o.acc[n][dt] * (by[n] * to_unit);
    }
    // The reference maximum was rounded and a score times the scale is not, before it is taken away: half a step of the maximum is a factor of all weights of the column.  From A8_FAR on it could take
    // a weight beyond sixteen bits, and then to 2^64 and more: there the score is rounded as the maximum was.
    if (__any(far)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int x = 0; x < 16; ++x) s[x / 4][n][x % 4] = is_far(n) ? (s[x / 4][n][x % 4] * a.scale_log2 - from[n]) / a.scale_log2 : s[x / 4][n][x % 4];
        from[n] = is_far(n) ? 0.f : from[n];
      }
    }
  }
  w_part w[NT][A8_WP];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float p[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) p[x] = exp2_fast(__builtin_fmaf(s[x / 4][n][x % 4], a.scale_log2, -from[n]));
    set_weights(p, w[n]);
  }
  // Where two waves meet on a unit the one in front of these products goes first: they leave most cycles for the other's arithmetic (179 -> 161 us for a prompt of
  // 4,096 rows; 165 with the scores' products too).
  __builtin_amdgcn_s_setprio(1);
  ones_times<NT>(w, o.l);
  // Values that no column sees are taken out; so are NaN, which some may not see: those that do get it back through a product of ones.
  uint32_t keep[4] = {0, 0, 0, 0}, nans = 0;
  if (!full) {
    const int from = c.wave_lo - first, to = c.wave_pos - first;
#pragma unroll
    for (int b = 0; b < 16; ++b) keep[b / 4] |= there && b >= from && b <= to ? 0xffu << 8 * (b & 3) : 0u;
  }
  u32x4 ahead = src.v(0);
#pragma unroll
  for (int dt = 0; dt < DP / 16; ++dt) {
    u32x4 v = ahead;
    if (dt + 1 < DP / 16) ahead = src.v(dt + 1);
    if (!full) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const uint32_t x = v[b] & keep[b], where = nan_bytes(x);
        nans |= where;
        v[b] = x & ~(where * 0xffu);
      }
    }
    f32x4 x[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) x[n] = o.acc[n][dt];
    values_times<NT>(v, v_scale, w, x);
#pragma unroll
    for (int n = 0; n < NT; ++n) o.acc[n][dt] = x[n];
    asm volatile("" ::: "memory");
  }
  __builtin_amdgcn_s_setprio(0);
  if (__any(nans != 0)) {
    // Made anew from here on, not kept for this: what follows happens next to never.
#pragma unroll
    for (int b = 0; b < 4; ++b) asm volatile("" : "+v"(keep[b]));
    w_part seen[NT][A8_WP];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float one[16];
#pragma unroll
      for (int y = 0; y < 16; ++y) one[y] = there && first + y >= c.lo[n] && first + y <= c.pos[n] ? 1.f : 0.f;
      set_weights(one, seen[n]);
    }
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt) {
      u32x4 v = src.v(dt);
      f32x4 count[NT];
#pragma unroll
      for (int b = 0; b < 4; ++b) v[b] = nan_bytes(v[b] & keep[b]) * 0x38u;     // 1 in e4m3
#pragma unroll
      for (int n = 0; n < NT; ++n) count[n] = f32x4{0.f, 0.f, 0.f, 0.f};
      values_times<NT>(v, 1.f, seen, count);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (SRC::HELD) o.bad[n] |= (decltype(o.bad[n] + 0))(count[n][i] > 0.f) << (4 * dt + i);
          else o.acc[n][dt][i] = o.acc[n][dt][i] + (count[n][i] > 0.f ? NAN : 0.f);
        }
      asm volatile("" ::: "memory");
    }
  }
}

// Where a column's result goes, from its first entry 4 g on.
template <int NT>
__device__ __forceinline__ elem_t* a8_out(const A8Args& a, const A8Rows<NT>& c, int col) {
  const int row = col / a.group;
  return a.out + ((int64_t)(c.tok0 + row) * a.nq + c.kvh * a.group + col - row * a.group) * a.d + 4 * c.g;
}

// Segments: what is summed up apart where a row's keys are split over workgroups.  Those in which the columns of a block have keys; a block that has none at all
// counts the first.
__device__ __forceinline__ void a8_segments(int lo, int pos, int& first, int& last) {
  last = max(pos, 0) / A8_SEG;
  first = min(lo / A8_SEG, last);
}

// The pages that a workgroup walks, 64 at a time: lane l has number `base + l` of the sequence's.
struct A8Pages {
  int base;
  uint64_t at;               // where its block of the kv head begins, in keys and in values alike (the first page's, for a page that is none)
  float k_scale;
  int v_exp;
  bool clean;                // all of them that hold keys up to the last one are there
  template <int NT>
  __device__ __forceinline__ void fill(const A8Args& a, const A8Rows<NT>& c, int first, int pos) {
    base = first;
    const int i = first + (threadIdx.x & 63);
    const int page = i < a.W && i <= pos >> a.lp ? a.table[(int64_t)c.seq * a.W + i] : -1;
    const bool there = (unsigned)page < (unsigned)a.pages;
    const int64_t block = (int64_t)(there ? page : 0) * a.nkv + c.kvh;
    const float ks = a.scales[2 * block], vs = a.scales[2 * block + 1];
    unsigned lo = (unsigned)(block * a.P * a.d), hi = (unsigned)((uint64_t)(block * a.P * a.d) >> 32);
    k_scale = there ? ks : 1.f;
    v_exp = there ? exponent_of(vs) : -256;
    clean = __ballot(i <= pos >> a.lp && !there) == 0;
    // Waited for here: a wait where they are used would be one for every load that is under way there.
    asm volatile("" : "+v"(lo), "+v"(hi), "+v"(k_scale), "+v"(v_exp));
    at = (uint64_t)hi << 32 | lo;
  }
  __device__ __forceinline__ uint64_t of_lane(int lane) const {                  // the same lane for the wave
    return (uint64_t)(unsigned)__builtin_amdgcn_readlane((int)(at >> 32), lane) << 32 | (unsigned)__builtin_amdgcn_readlane((int)at, lane);
  }
  __device__ __forceinline__ uint64_t of_any(int lane) const { return (uint64_t)(unsigned)__shfl((int)(at >> 32), lane) << 32 | (unsigned)__shfl((int)at, lane); }
};

// ---- few columns (decoded tokens, small groups' drafted ones): a workgroup takes segments of 512 keys one after the other, a wave two of a segment's tiles, every fourth, for up to 16 NT
// columns.
// Tiles come straight into registers: a tile's keys are asked for when the last tile's have been multiplied, its values when those have, so that there is something under way at any
// time and no load waits for another (page numbers and scales are read 64 pages ahead; a page number read in turn would wait for all loads before it).  The waves' sums meet in LDS, the
// segments' in a8_join_kernel.
// A tile in registers.  Of heads of 128 a load takes eight rows of K in whole lines of the cache, 128 bytes, and not half of each of sixteen: the load of the other halves
// would wait in the first cache for the lines that are under way, and what stands behind it too (200 -> 188 us for 64 rows of 8,192 keys).  So kr[i][0] has in lane rows 0..7 the first
// half of rows 0..7, in lane rows 8..15 their second half, kr[i][1] the same of rows 8..15, and a lane's own row comes together when it is used.
template <int DP>
struct A8Held {
  static constexpr bool HELD = true, LINES = DP % 128 == 0;
  u32x4 kr[4][DP / 64], vr[DP / 16];
  __device__ __forceinline__ u32x4 k(int i, int j) const {
    if (!LINES) return kr[i][j];
    u32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int a = (int)kr[i][j & ~1][e], b = (int)kr[i][j | 1][e];
      // Lane rows 8 apart change places (row_ror:8), in those lanes that have another row's half.
      x[e] = (j & 1) ? (uint32_t)__builtin_amdgcn_update_dpp(b, a, 0x128, 0xF, 0x3, false) : (uint32_t)__builtin_amdgcn_update_dpp(a, b, 0x128, 0xF, 0xC, false);
    }
    return x;
  }
  __device__ __forceinline__ u32x4 v(int dt) const { return vr[dt]; }
};

template <int DP, int NT>
__global__ __launch_bounds__(256, DP <= 128 && NT == 1 ? 2 : 1) void a8_few_kernel(A8Args a, int segs_each) {
  __shared__ float sums[4][DP / 16][64][4];
  __shared__ float maxima[4][16 * NT], totals[4][16 * NT];
  A8Rows<NT> c;
  const int kvh = blockIdx.x % a.nkv, item = blockIdx.x / a.nkv, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (!a8_rows<NT>(a, item, kvh, 0, c)) return;
  int seg_first, seg_last;
  a8_segments(c.wave_lo, c.wave_pos, seg_first, seg_last);
  const int seg0 = seg_first + (int)blockIdx.y * segs_each, seg1 = min(seg_last, seg0 + segs_each - 1);
  if (seg0 > seg1) return;
  const int kb0 = seg0 * A8_SEG + wave * A8_TILE, pos = min(c.wave_pos, seg1 * A8_SEG + A8_SEG - 1);
  A8Query<DP, NT> q;
  a8_load_q<DP, NT>(a, c, q);
  A8Pages pages;
  pages.fill(a, c, seg0 * A8_SEG >> a.lp, pos);

  A8Held<DP> t;
  // Loads that stand under a condition are waited for where the ways meet again: every tile asks for the next one, the last for itself once more (from the cache).
  const int tile_lo = max(c.wave_lo, seg0 * A8_SEG) & ~(A8_TILE - 1), tile_hi = max(pos, 0) & ~(A8_TILE - 1);
  float k_scale;
  int v_exp, v_key;
  auto ask_k = [&](int kb) {
    const int at = min(max(kb, tile_lo), tile_hi);
    if (((at + A8_TILE - 1) >> a.lp) - pages.base >= 64) pages.fill(a, c, at >> a.lp, pos);
    v_key = at + 16 * c.g;
    k_scale = __shfl(pages.k_scale, ((at + 16 * (c.r >> 2)) >> a.lp) - pages.base);
    v_exp = __shfl(pages.v_exp, (v_key >> a.lp) - pages.base);
    v_exp = v_key <= c.wave_pos && v_key + 15 >= c.wave_lo ? v_exp : -256;
    constexpr bool LINES = A8Held<DP>::LINES;
    constexpr int HALVES = LINES ? 2 : 1;
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
      const int r = LINES ? (c.r & 7) + 8 * h : c.r, key = at + 16 * (r >> 2);
      const uint8_t* kp = a.kc + pages.of_any((key >> a.lp) - pages.base) + ((key & (a.P - 1)) + (r & 3)) * a.d;
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int j = 0; j < DP / 64 / HALVES; ++j) {
          const int piece = LINES ? 128 * j + 64 * (c.r >> 3) + 16 * c.g : 64 * j + 16 * c.g;
          t.kr[s][HALVES * j + h] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kp + 4 * s * a.d + min(piece, a.d - 16)));     // beyond d: the last again, times q's zeros
        }
    }
  };
  auto ask_v = [&]() {
    const uint8_t* vp = a.vc + pages.of_any((v_key >> a.lp) - pages.base) + c.r * a.P + (v_key & (a.P - 1));
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt) t.vr[dt] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(vp + min(16 * dt, a.d - 16) * a.P));     // and here for nothing
  };
  ask_k(kb0);
  ask_v();
  a8_wait_q<DP, NT>(q);
  A8Sums<DP, NT> o;
  o.clear();
  int below = 256;                                      // scales of this and more have been taken, in the tile's passes before this one
  for (int kb = kb0; (kb & ~(A8_SEG - 1)) <= seg1 * A8_SEG;) {
    const bool mine = kb <= pos && kb + A8_TILE > c.wave_lo;
    const int exp_now = v_exp < below ? v_exp : -256, top = __builtin_amdgcn_readfirstlane((int)over_groups_max((float)exp_now));
    const int unit = o.next_unit(top), least = o.least_exponent(unit, top);
    const bool more = mine && __any(exp_now > -256 && exp_now < least);
    f32x4 s[4][NT];
    if (mine) a8_scores<DP, NT>(t, k_scale, q, s);
    ask_k(more ? kb : kb + A8_SEG / 2);
    if (mine) a8_weigh<2, DP, NT>(a, c, kb, t, s, exp_now >= least ? exp_now : -256, unit, o);
    ask_v();
    below = more ? least : 256;
    if (more) continue;
    const bool second = (kb & (A8_SEG / 2)) != 0;
    const int seg = kb / A8_SEG;
    kb += A8_SEG / 2;
    if (!second) continue;
    // Both tiles of the segment.
#pragma unroll
    for (int n = 0; n < NT; ++n)
      if (c.g == 0) {
        maxima[wave][16 * n + c.r] = o.m[n];
        totals[wave][16 * n + c.r] = o.l[n][0];
      }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      __syncthreads();                                  // the maxima are there; the sums of the columns before have been read
      const int x0 = 16 * n + c.r, col = c.col0 + x0;
      const float top = fmaxf(fmaxf(maxima[0][x0], maxima[1][x0]), fmaxf(maxima[2][x0], maxima[3][x0])), by = exp2_fast(o.m[n] - top) * (o.scale() * A8_PART);
      float total = 0.f;
#pragma unroll
      for (int x = 0; x < 4; ++x) total = __builtin_fmaf(totals[x][x0] * A8_PART, exp2_fast(maxima[x][x0] - top), total);
#pragma unroll
      for (int dt = 0; dt < DP / 16; ++dt) *reinterpret_cast<f32x4*>(sums[wave][dt][lane]) = o.times(n, dt, by);
      __syncthreads();
      if (col < c.cols) {
        const int64_t part = (((int64_t)item * a.nkv + kvh) * a.nseg + seg - seg_first) * a.cols_max + col;
#pragma unroll
        for (int x = 0; x < DP / 64; ++x) {
          const int dt = 4 * x + wave;
          if (16 * dt >= a.d) continue;
          f32x4 v = *reinterpret_cast<const f32x4*>(sums[0][dt][lane]);
#pragma unroll
          for (int y = 1; y < 4; ++y) v = v + *reinterpret_cast<const f32x4*>(sums[y][dt][lane]);
          if (seg_first == seg_last) store_elems4(a8_out<NT>(a, c, col) + 16 * dt, total == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : v * (1.f / total));
          else *reinterpret_cast<f32x4*>(a.part_acc + part * a.d + 16 * dt + 4 * c.g) = v;
        }
        if (seg_first != seg_last && wave == 0 && c.g == 0) *reinterpret_cast<f32x2*>(a.part_ml + 2 * part) = f32x2{top, total};
      }
    }
    o.clear();
    __syncthreads();                                    // all have read the maxima: the next segment's may be written
  }
}

// ---- more columns (prompts, drafted tokens): tiles pass through LDS once for all waves, each of which has 16 NT columns.  SPLIT: a workgroup takes one segment.
//
// A tile in LDS: K's row 16 i + r (the key that lane row r reads for tile i) in DP bytes, V's entry in 64; the 16-byte piece p of K's row r lies at p ^ turn(r), of V's entry
// e at p ^ (e / 4 % 4), so that the 16 lanes that read a piece of 16 rows read 16 different quads of banks.  Pieces come by loads that go to LDS without passing registers: a load
// brings a kilobyte, lane l's 16 bytes to place l, and the order is made by what each lane asks for.
template <int DP, int WAVES>
struct A8Stage {
  static constexpr int BYTES = 2 * A8_TILE * DP, LOADS = DP / 16 / WAVES;      // of a tile; of K, and of V, that a wave asks for
  static_assert(DP / 16 % WAVES == 0, "every wave asks for the same number of loads");
  static constexpr int PIECES = DP / 16;                                       // of a row of K
  __device__ static __forceinline__ int turn(int r) { return DP == 128 ? r >> 1 & 7 : DP == 256 ? r : r >> 2 & 3; }
};

#ifdef VK_BF16
constexpr bool EXPONENTS = true;         // values' scales go into a unit of the sums
#else
constexpr bool EXPONENTS = false;
#endif

// What stands in scalar registers for an instruction written out, said to the compiler next to it: it may have moved the arithmetic to vector registers.
__device__ __forceinline__ const uint8_t* a8_scalar(const uint8_t* p) {
  const uint64_t u = (uint64_t)p;
  return (const uint8_t*)((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(u >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)u));
}
__device__ __forceinline__ void a8_load_to_lds(const uint8_t* p, unsigned lds_addr) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(p), "s"(__builtin_amdgcn_readfirstlane(lds_addr)) : "memory");
}

// What a lane asks for lies at the same distance from the start of the page (of pages smaller than a tile: of the one of its 16 keys) in every tile, but for the tile's own place in a
// larger page.
template <int DP, int WAVES>
struct A8Offsets {
  unsigned k[A8Stage<DP, WAVES>::LOADS], v[A8Stage<DP, WAVES>::LOADS];
  int k_page[A8Stage<DP, WAVES>::LOADS], v_page[A8Stage<DP, WAVES>::LOADS];      // which of the tile's pages
  __device__ __forceinline__ void set(const A8Args& a, int wave, int lane) {
    typedef A8Stage<DP, WAVES> ST;
    const int within = min(a.P, A8_TILE) - 1;
#pragma unroll
    for (int i = 0; i < ST::LOADS; ++i) {
      const int at = (i * WAVES + wave) * 64 + lane;           // piece of K's tile
      const int row = at / ST::PIECES, r = row & 15, piece = min((at % ST::PIECES) ^ ST::turn(r), a.d / 16 - 1);
      const int k_key = 16 * (r >> 2) + 4 * (row >> 4) + (r & 3), v_key = 16 * ((at & 3) ^ (at >> 4 & 3));
      k[i] = (k_key & within) * a.d + 16 * piece;
      v[i] = min(at >> 2, a.d - 1) * a.P + (v_key & within);
      k_page[i] = k_key >> a.lp;
      v_page[i] = v_key >> a.lp;
    }
  }
};

// Asks for a tile, whose first page is the wave's lane `first` of pg and whose first key stands at `within` of it.  WIDE: a tile lies in one page.
template <bool WIDE, int DP, int WAVES>
__device__ __forceinline__ void a8_ask(const A8Args& a, const A8Pages& pg, const A8Offsets<DP, WAVES>& off, int first, int within, unsigned lds) {
  typedef A8Stage<DP, WAVES> ST;
  const unsigned to = __builtin_amdgcn_readfirstlane(lds);
  if (WIDE) {
    const uint64_t at = pg.of_lane(first);
    const uint8_t *kp = a8_scalar(a.kc + at + within * a.d), *vp = a8_scalar(a.vc + at + within);
#pragma unroll
    for (int i = 0; i < ST::LOADS; ++i) pipe_load_to_lds16_sv(kp, off.k[i], to + i * WAVES * 1024);
#pragma unroll
    for (int i = 0; i < ST::LOADS; ++i) pipe_load_to_lds16_sv(vp, off.v[i], to + A8_TILE * DP + i * WAVES * 1024);
  } else {
#pragma unroll
    for (int i = 0; i < ST::LOADS; ++i) a8_load_to_lds(a.kc + pg.of_any(first + off.k_page[i]) + off.k[i], to + i * WAVES * 1024);
#pragma unroll
    for (int i = 0; i < ST::LOADS; ++i) a8_load_to_lds(a.vc + pg.of_any(first + off.v_page[i]) + off.v[i], to + A8_TILE * DP + i * WAVES * 1024);
  }
}

template <int DP, int WAVES>
struct A8Shared {
  static constexpr bool HELD = false;
  const uint8_t* tile;
  int r, g;
  __device__ __forceinline__ u32x4 k(int i, int j) const {
    return *reinterpret_cast<const u32x4*>(tile + (16 * i + r) * DP + (((4 * j + g) ^ A8Stage<DP, WAVES>::turn(r)) << 4));
  }
  __device__ __forceinline__ u32x4 v(int dt) const { return *reinterpret_cast<const u32x4*>(tile + A8_TILE * DP + (16 * dt + r) * 64 + ((g ^ (r >> 2)) << 4)); }
};

template <int DP, int NT, int WAVES, bool SPLIT, bool WIDE>
__global__ __launch_bounds__(64 * WAVES, DP <= 128 ? 2 : 1) void a8_shared_kernel(A8Args a, int blocks) {
  typedef A8Stage<DP, WAVES> ST;
  extern __shared__ __attribute__((aligned(1024))) uint8_t stages[];      // A8_STAGES tiles
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Which wave has which columns turns with the workgroup: where there are none for the last one it is not always the same unit of the CU that has nothing to do.
  const unsigned turn = SPLIT ? blockIdx.x ^ blockIdx.x >> 3 ^ blockIdx.x >> 8 : 0;
  // The kv head first: the workgroups of one, which read the same pages, then fall to as few of the eight caches as there are.
  int unit = blockIdx.x;
  const int kvh = unit % a.nkv;
  unit /= a.nkv;
  const int seg_at = SPLIT ? unit % a.nseg : 0;
  if (SPLIT) unit /= a.nseg;
  const int block = unit % blocks, item = SPLIT ? unit / blocks : a.n_items - 1 - unit / blocks;     // a prompt's last rows, which see most keys, first
  A8Rows<NT> c;
  A8Rows<NT * WAVES> all;                                                 // the workgroup's columns
  if (!a8_rows<NT * WAVES>(a, item, kvh, block * 16 * NT * WAVES, all)) return;
  const bool mine = a8_rows<NT>(a, item, kvh, (block * WAVES + (wave + turn) % WAVES) * 16 * NT, c);
  int lo = all.wave_lo, pos = all.wave_pos, seg_first = 0, seg_last = 0;
  if (SPLIT) {
    a8_segments(lo, pos, seg_first, seg_last);
    const int seg = seg_first + seg_at;
    if (seg > seg_last) return;
    lo = max(lo, seg * A8_SEG);
    pos = min(pos, seg * A8_SEG + A8_SEG - 1);
  }
  if (!mine) {
    c.seq = all.seq;
    c.kvh = kvh;
  }
  A8Query<DP, NT> q;
  if (mine) a8_load_q<DP, NT>(a, c, q);
  A8Sums<DP, NT> o;
  o.clear();
  a8_wait_q<DP, NT>(q);
  lo &= ~(A8_TILE - 1);
  const int tiles = pos < lo ? 0 : ((pos - lo) >> 6) + 1;
  const unsigned lds = (unsigned)(unsigned long)((__attribute__((address_space(3))) const void*)stages);
  A8Pages ahead, now;                                                     // of the tiles that are asked for, of those that are computed
  A8Offsets<DP, WAVES> off;
  off.set(a, wave, threadIdx.x & 63);
  // Tiles from which on the 64 pages that were read are used up.
  int ahead_end = 0, now_end = 0;
  auto fill = [&](A8Pages& pages, int& end, int i) {
    const int kb = lo + i * A8_TILE;
    pages.fill(a, c, kb >> a.lp, pos);
    // and their values' scales are within 2^5 of the first one's, so that no tile of several pages needs a second pass (the whole spread, by two reductions: portions in pages of 16 keys 93 us for 90).
    if (!WIDE && EXPONENTS) {
      const int off = pages.v_exp - __builtin_amdgcn_readfirstlane(pages.v_exp);
      pages.clean = pages.clean && __ballot(pages.v_exp > -256 && abs(off) > (A8_UNIT_DOWN - A8_UNIT_STAYS) / 2) == 0;
    }
    end = __builtin_amdgcn_readfirstlane(i + (((64 << a.lp) - (kb & (a.P - 1))) >> 6));
  };
  if (tiles > 0) {
    fill(ahead, ahead_end, 0);
    now = ahead;
    now_end = ahead_end;
  }
  unsigned stage = 0;                                   // of the tile that is asked for, in bytes
  auto ask = [&](int tile) {
    const int i = __builtin_amdgcn_readfirstlane(tile), kb = lo + i * A8_TILE;
    if (i >= ahead_end) fill(ahead, ahead_end, i);
    a8_ask<WIDE, DP, WAVES>(a, ahead, off, (kb >> a.lp) - ahead.base, kb & (a.P - 1), lds + wave * 1024 + stage);
    stage ^= ST::BYTES;
  };
  if (tiles > 0) ask(0);
  // Tiles that all of the wave's rows see whole, where no page is missing.
  const int whole0 = mine ? (max(c.all_lo - lo, 0) + A8_TILE - 1) >> 6 : 0, whole1 = mine ? min(tiles, (c.all_pos + 1 - lo) >> 6) : 0;
  auto step = [&](int tile, auto all_see) {
    const int i = __builtin_amdgcn_readfirstlane(tile), kb = lo + i * A8_TILE;
    // Tile i has arrived, this wave has what it read of tile i - 1; behind the barrier that holds for all.
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const A8Shared<DP, WAVES> src{stages + (stage ^ ST::BYTES), c.r, c.g};
    if (i + 1 < tiles) ask(i + 1);
    if (!all_see.value && (!mine || kb > c.wave_pos || kb + A8_TILE <= c.wave_lo)) return;
    if (i >= now_end) fill(now, now_end, i);
    const int key = kb + 16 * c.g;
    float k_scale;
    int v_exp;
    if (WIDE) {
      const int l = (kb >> a.lp) - now.base;
      k_scale = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, now.k_scale), l));
      const int exp = __builtin_amdgcn_readlane(now.v_exp, l), unit = o.next_unit(exp);
      v_exp = all_see.value || (key <= c.wave_pos && key + 15 >= c.wave_lo) ? exp : -256;
      f32x4 s[4][NT];
      a8_scores<DP, NT>(src, k_scale, q, s);
      a8_weigh<all_see.value, DP, NT>(a, c, kb, src, s, v_exp, unit, o);
      return;
    }
    k_scale = __shfl(now.k_scale, ((kb + 16 * (c.r >> 2)) >> a.lp) - now.base);
    v_exp = __shfl(now.v_exp, (key >> a.lp) - now.base);
    if (!all_see.value) v_exp = key <= c.wave_pos && key + 15 >= c.wave_lo ? v_exp : -256;
    if (all_see.value) {
      const int unit = o.next_unit(__builtin_amdgcn_readfirstlane((int)over_groups_max((float)v_exp)));
      f32x4 s[4][NT];
      a8_scores<DP, NT>(src, k_scale, q, s);
      a8_weigh<all_see.value, DP, NT>(a, c, kb, src, s, v_exp, unit, o);
      return;
    }
    for (bool more = true; more;) {
      const int top = __builtin_amdgcn_readfirstlane((int)over_groups_max((float)v_exp)), unit = o.next_unit(top), least = o.least_exponent(unit, top);
      more = __any(v_exp > -256 && v_exp < least);
      int from = kb;
      asm volatile("" : "+s"(from));                    // or every comparison with it would be made before the loop and held in scalar registers that there are not
      f32x4 s[4][NT];
      a8_scores<DP, NT>(src, k_scale, q, s);
      a8_weigh<0, DP, NT>(a, c, from, src, s, v_exp >= least ? v_exp : -256, unit, o);
      v_exp = v_exp >= least ? -256 : v_exp;
    }
  };
  for (int i = 0; i < tiles;) {
    for (; i < tiles && !(i >= whole0 && i < whole1 && i < now_end && now.clean); ++i) step(i, std::integral_constant<int, 0>());
    for (; i < whole1 && i < now_end && now.clean; ++i) step(i, std::integral_constant<int, 1>());
  }
  if (!mine) return;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = c.col0 + 16 * n + c.r;
    const float l = o.l[n][0];
    if (col >= c.cols) continue;
    if (SPLIT && seg_first != seg_last) {
      const int64_t part = (((int64_t)item * a.nkv + kvh) * a.nseg + seg_at) * a.cols_max + col;
#pragma unroll
      for (int dt = 0; dt < DP / 16; ++dt)
        if (16 * dt < a.d) *reinterpret_cast<f32x4*>(a.part_acc + part * a.d + 16 * dt + 4 * c.g) = o.times(n, dt, o.scale() * A8_PART);
      if (c.g == 0) *reinterpret_cast<f32x2*>(a.part_ml + 2 * part) = f32x2{o.m[n], l * A8_PART};
    } else {
      elem_t* to = a8_out<NT>(a, c, col);
      const float by = l == 0.f ? 0.f : o.scale() / l;
#pragma unroll
      for (int dt = 0; dt < DP / 16; ++dt)
        if (16 * dt < a.d) store_elems4(to + 16 * dt, l == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : o.times(n, dt, by));
    }
  }
}

// ---- the segments of a column, by a wave: weights relative to their largest maximum, sums in ascending order.  cols: of a block in the kernel that wrote them.
__global__ __launch_bounds__(256) void a8_join_kernel(A8Args a, int cols) {
  A8Rows<1> c;
  const int kvh = blockIdx.x % a.nkv, item = blockIdx.x / a.nkv, lane = threadIdx.x & 63, col = blockIdx.y * 4 + (threadIdx.x >> 6);
  if (!a8_rows<1>(a, item, kvh, col, c)) return;
  const int block0 = col / cols * cols, row_first = block0 / a.group, row_last = (min(c.cols, block0 + cols) - 1) / a.group;
  int seg_first, seg_last;
  a8_segments(a.window > 0 ? max(0, c.pos0 + row_first - a.window + 1) : 0, min(c.pos0 + row_last, a.max_keys - 1), seg_first, seg_last);
  if (seg_first == seg_last) return;                    // the other kernel wrote the result
  const int64_t part0 = ((int64_t)item * a.nkv + kvh) * a.nseg * a.cols_max + col;
  const int segs = seg_last - seg_first + 1;
  float top = A8_NONE;
  for (int s = lane; s < segs; s += 64) top = fmaxf(top, a.part_ml[2 * (part0 + (int64_t)s * a.cols_max)]);
  top = wave_max_xor(top);
  float total = 0.f;
  f32x2 o[2] = {{0.f, 0.f}, {0.f, 0.f}};
  for (int s0 = 0; s0 < segs; s0 += 64) {
    float by = 0.f;
    if (s0 + lane < segs) {
      const f32x2 ml = *reinterpret_cast<const f32x2*>(a.part_ml + 2 * (part0 + (int64_t)(s0 + lane) * a.cols_max));
      by = exp2_fast(ml.x - top);
      total = __builtin_fmaf(ml.y, by, total);
    }
    const int n = min(64, segs - s0);
    const float* p = a.part_acc + (part0 + (int64_t)s0 * a.cols_max) * a.d + 2 * lane;
    for (int s = 0; s < n; s += 8) {
      f32x2 v[8][2];
#pragma unroll
      for (int x = 0; x < 8; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          v[x][h] = f32x2{0.f, 0.f};
          if (s + x < n && 2 * lane + 128 * h < a.d) v[x][h] = *reinterpret_cast<const f32x2*>(p + (int64_t)(s + x) * a.cols_max * a.d + 128 * h);
        }
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const float b = __shfl(by, min(s + x, 63));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          o[h].x = s + x < n ? __builtin_fmaf(v[x][h].x, b, o[h].x) : o[h].x;
          o[h].y = s + x < n ? __builtin_fmaf(v[x][h].y, b, o[h].y) : o[h].y;
        }
      }
    }
  }
  total = wave_sum_xor(total);
  const int row = col / a.group;
  elem_t* to = a.out + ((int64_t)(c.tok0 + row) * a.nq + kvh * a.group + col - row * a.group) * a.d + 2 * lane;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (2 * lane + 128 * h < a.d) {
      to[128 * h] = from_f32<elem_t>(total == 0.f ? 0.f : o[h].x / total);
      to[128 * h + 1] = from_f32<elem_t>(total == 0.f ? 0.f : o[h].y / total);
    }
}

template <int DP, int NT, int WAVES, bool SPLIT, bool WIDE>
static int a8_shared_as(const A8Args& a, hipStream_t st) {
  const int blocks = (a.cols_max + 16 * NT * WAVES - 1) / (16 * NT * WAVES);
  const int64_t units = (int64_t)a.n_items * a.nkv * blocks * (SPLIT ? a.nseg : 1);
  VK_REQUIRE(units < (1ll << 31), "attention8: %d items of %d rows, %d heads: too many for one launch", a.n_items, a.item_rows, a.nq);
  const int lds = A8_STAGES * A8Stage<DP, WAVES>::BYTES;
  static_assert(A8_STAGES * A8Stage<DP, WAVES>::BYTES <= 64 * 1024, "what a launch may ask for");
  a8_shared_kernel<DP, NT, WAVES, SPLIT, WIDE><<<(unsigned)units, 64 * WAVES, lds, st>>>(a, blocks);
  return vk_check_launch("attention8");
}
template <int DP, int NT, int WAVES, bool SPLIT>
static int a8_shared(const A8Args& a, hipStream_t st) {
  // Tiles of one page in kernels of their own: what is the same for a wave stays in scalar registers, and the loop has no branch (2,048 rows of heads of 64 over themselves 49 -> 44 us, 4,096 of 128
  // 161 -> 157).
  return a.P >= A8_TILE ? a8_shared_as<DP, NT, WAVES, SPLIT, true>(a, st) : a8_shared_as<DP, NT, WAVES, SPLIT, false>(a, st);
}

extern "C" {

// Segments that the rows of an item may have keys in: those of the bound, and of a window no more than its keys and the rows' other places touch.
static int64_t a8_most_segments(int item_rows, int max_k_len, int window) {
  const int64_t all = ((int64_t)max_k_len + A8_SEG - 1) / A8_SEG, keys = (int64_t)window + item_rows - 1;
  return window > 0 && window < max_k_len ? min(all, (keys + A8_SEG - 2) / A8_SEG + 1) : all;
}

// 32-bit words of scratch for `items` items of up to item_rows <= 16 rows: 0 for more rows, whose keys are not split, and for few keys.  window: 0, or that of the call.
int64_t vk_attn8_scratch_floats(int items, int item_rows, int nq, int d, int max_k_len, int window) {
  const int64_t nseg = a8_most_segments(item_rows, max_k_len, window);
  if (item_rows > 16 || nseg <= 1) return 0;
  return (int64_t)items * item_rows * nq * nseg * (d + 2);
}

// Attention of the rows named by items [n_items, 2] = (sequence, first row of the item within its rows): each up to item_rows rows.  Up to 16 rows: the keys
// are split over workgroups, whose sums meet in scratch; more: whole rows by a workgroup.  Sequences and rows that the arrays do not have are left out, a page
// number outside the cache is a page without keys, and keys are looked for up to max_k_len (k_len's bound; the table covers it).  scratch: 16-byte aligned.
int vk_paged_attention8(elem_t* out, const elem_t* q, const uint8_t* kc, const uint8_t* vc, const float* scales, const int32_t* table, int W,
                        const int32_t* cu_q, const int32_t* k_len, const int32_t* items, int n_items, int item_rows, float* scratch, int64_t scratch_floats,
                        int T, int S, int nq, int nkv, int d, int P, int pages, int max_k_len, int window, float scale, hipStream_t st) {
  VK_REQUIRE(T >= 0 && S >= 0 && n_items >= 0 && nq > 0 && nkv > 0 && nq % nkv == 0, "attention8: bad sizes T=%d S=%d items=%d nq=%d nkv=%d", T, S, n_items, nq, nkv);
  VK_REQUIRE(d >= 16 && d <= 256 && d % 16 == 0, "attention8: head size %d is no multiple of 16 from 16 to 256", d);
  VK_REQUIRE(P >= CACHE8_MIN_PAGE && P <= CACHE8_MAX_PAGE && (P & (P - 1)) == 0, "attention8: page size %d is no power of two from %d to %d", P, CACHE8_MIN_PAGE,
             CACHE8_MAX_PAGE);
  VK_REQUIRE(item_rows >= 1 && item_rows <= A8_ITEM_ROWS, "attention8: items of %d rows; at most %d", item_rows, A8_ITEM_ROWS);
  VK_REQUIRE(pages > 0 && W > 0 && max_k_len >= 0 && (int64_t)W * P >= max_k_len && (int64_t)W * P < (1ll << 31), "attention8: a table of %d pages of %d does not cover %d keys", W, P, max_k_len);
  VK_REQUIRE(window >= 0, "attention8: window %d", window);
  VK_REQUIRE(scale > 0.f && scale < INFINITY, "attention8: scale %g is no positive number", (double)scale);
  if (n_items == 0 || T == 0 || S == 0) return 0;
  VK_REQUIRE(((uintptr_t)q | (uintptr_t)out | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)scratch) % 16 == 0, "attention8: rows, cache and scratch have to lie on 16 bytes");
  const int group = nq / nkv, nseg = max(1, (int)a8_most_segments(item_rows, max_k_len, window));
  // A window as long as the keys hides none; as none it takes part in no difference that could pass 32 bits.
  A8Args a{q, out, kc, vc, scales, table, cu_q, k_len, items, nullptr, nullptr, W, T, S, nq, nkv, d, P, 0, pages, group, item_rows, item_rows * group,
           window >= max_k_len ? 0 : window, nseg, n_items, max_k_len, scale * 1.4426950408889634f};
  while (1 << a.lp < P) ++a.lp;
  constexpr bool F32 = sizeof(elem_t) == 4;
  if (item_rows > 16) {
    constexpr int NT = F32 ? 1 : 2;
    return d <= 64 ? a8_shared<64, NT, 4, false>(a, st) : d <= 128 ? a8_shared<128, NT, 4, false>(a, st) : d <= 192 ? a8_shared<192, NT, 4, false>(a, st)
                                                                                                                   : a8_shared<256, NT, 4, false>(a, st);
  }
  const int64_t need = vk_attn8_scratch_floats(n_items, item_rows, nq, d, max_k_len, window);
  VK_REQUIRE(need == 0 || (scratch != nullptr && scratch_floats >= need), "attention8: scratch of %lld floats needed", (long long)need);
  a.part_acc = scratch;
  a.part_ml = scratch + need / (d + 2) * d;
  const int64_t joins = (int64_t)n_items * nkv;
  VK_REQUIRE(joins < (1ll << 31) && nseg <= 65535, "attention8: %d items, %d keys: too many for one launch", n_items, max_k_len);
  // Few columns go by tiles in registers, which each wave reads and converts for itself: in bfloat16 for one tile of columns, as with more the conversion is done once for all waves'
  // tiles in LDS and not once a wave's tile (64 sequences of 4,000 keys, 8 kv heads of 64: 70 us for 32 columns and 100 for 64, in registers 113 and 182; a single sequence of 1,000
  // keys, which waits for its loads only, takes 16 us and took 13).  In 32 bits the products bound it, and two tiles of columns stay in registers while the cache's fit beside
  // them, to heads of 64: 21 us against 31 for one sequence of 4,000 keys, 39 against 51 for 8, 242 against 192 for 64.  The choice is made by what a row's own item is, not by how many there are: a row's
  // result doesn't depend on its company.
  const int most = F32 && d <= 64 ? 2 : 1, nt = (a.cols_max + 15) / 16;
  int cols;                                             // of a block
  if (nt <= most) {
    cols = 16 * nt;
    // Workgroups of several segments where there are more than the card holds at once: what stands in front of a workgroup's first loads is then paid once (64 rows of 8,192 keys,
    // calls in a row: 203 us, with a segment each 230; up to 4 or 16 instead of 8 change it by 2 %).
    const int64_t held = (nt == 1 ? 2 : 1) * vk_device_cus();
    const int each = (int)max((int64_t)1, min((int64_t)8, joins * nseg / (2 * held)));
    const dim3 grid((unsigned)joins, (nseg + each - 1) / each);
#define FEW(D, N) a8_few_kernel<D, N><<<grid, 256, 0, st>>>(a, each)
#ifndef VK_BF16
    if (nt == 2) FEW(64, 2);
    else
#endif
    if (d <= 64) FEW(64, 1);
    else if (d <= 128) FEW(128, 1);
    else if (d <= 192) FEW(192, 1);
    else FEW(256, 1);
#undef FEW
    if (vk_check_launch("attention8")) return 1;
  } else {
    // Two waves where they have a tile of columns each (32 columns, 64 sequences of 4,000 keys, heads of 64: 70 us against 81 with four waves; in 32 bits, heads of 128, 497 against
    // 592); of the largest heads' tiles half would be too many loads for a wave's registers.  Two tiles of columns a wave and half the waves were no faster for 64 columns (97 us
    // against 99 for heads of 64, 181 against 177 for 128) and slower for one sequence (19 against 16).
    const bool two = a.cols_max <= 32 && d <= 192;
    constexpr int SMALL = F32 ? 128 : 64;               // two tiles of columns of heads of 64 are in registers in 32 bits
    cols = two ? 32 : 64;
    const int bad = two ? (d <= SMALL ? a8_shared<SMALL, 1, 2, true>(a, st) : d <= 128 ? a8_shared<128, 1, 2, true>(a, st) : a8_shared<192, 1, 2, true>(a, st))
                        : (d <= 64 ? a8_shared<64, 1, 4, true>(a, st) : d <= 128 ? a8_shared<128, 1, 4, true>(a, st) : d <= 192 ? a8_shared<192, 1, 4, true>(a, st)
                                                                                                                               : a8_shared<256, 1, 4, true>(a, st));
    if (bad) return 1;
  }
  if (nseg == 1) return 0;
  a8_join_kernel<<<dim3((unsigned)joins, (a.cols_max + 3) / 4), 256, 0, st>>>(a, cols);
  return vk_check_launch("attention8 (join)");
}

}  // extern "C"
