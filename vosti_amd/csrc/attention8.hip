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
// Arithmetic.  A key's entry times its scale is exact in the element type, so the first product takes q as it is and 32-bit sums.  Weights are at most 1 (2^8
// where a reference maximum is kept) and go into the second product in 16-bit floating point with eleven digits, against values without their scale, which
// they hold to the bit: bfloat16 weights, with eight, doubled the squared error of the result.  Values' scales that differ within a product stand in its
// entries relative to the largest of them.  The 32-bit build takes everything in 32 bits.  Sums of weights are of the unrounded ones.
//
// Keys that a row does not see weigh 0, whatever is stored: their scores are never used, and values outside what the wave's rows see, or NaN, are
// taken out of the second product of a tile that not all rows see whole; a row that does see a NaN gets it back through a product of its own.
#include "cache8.h"
#include "mma.h"
#include "vec.h"

#define A8_TILE 64
#define A8_SEG_TILES 4           // tiles of a segment: what a workgroup of the few rows' kernel takes, a tile a wave
#define A8_SEG (A8_TILE * A8_SEG_TILES)
#define A8_ITEM_ROWS 128         // rows of an item, at most

struct A8Args {
  const elem_t* q;          // [T, nq, d]
  elem_t* out;
  const uint8_t *kc, *vc;
  const float* scales;
  const int32_t *table, *cu_q, *k_len, *items;
  float *part_ml, *part_acc;   // per (item, kv head, segment, column): maximum and sum; d sums
  int W, T, S, nq, nkv, d, P, lp, pages, group, item_rows, cols_max, window, nseg;
  float scale_log2;
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float over_groups_max(float v) {
  v = fmaxf(v, lane_xor16(v));
  return fmaxf(v, lane_xor32(v));
}
__device__ __forceinline__ float over_groups_sum(float v) {
  v = v + lane_xor16(v);
  return v + lane_xor32(v);
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
template <int NT>
__device__ __forceinline__ void values_times(u32x4 raw, float scale, const w_part (&w)[NT][A8_WP], f32x4 (&o)[NT]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f16x8 v = values_of(raw[2 * h], raw[2 * h + 1], scale);
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, w[n][h], o[n], 0, 0, 0);
  }
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
  c.seq = a.items[2 * item];
  const int first = a.items[2 * item + 1];
  if ((unsigned)c.seq >= (unsigned)a.S || first < 0) return false;
  const int t0 = a.cu_q[c.seq], t1 = a.cu_q[c.seq + 1];
  if (t0 < 0 || t1 > a.T) return false;
  c.rows = min(a.item_rows, t1 - t0 - first);
  c.cols = c.rows * a.group;
  c.col0 = col0;
  if (c.rows <= 0 || col0 >= c.cols) return false;
  c.tok0 = t0 + first;
  c.pos0 = a.k_len[c.seq] - (t1 - t0) + first;
  const int row_first = col0 / a.group, row_last = (min(c.cols, col0 + 16 * NT) - 1) / a.group;
  c.all_pos = c.pos0 + row_first;
  c.wave_pos = c.pos0 + row_last;
  c.wave_lo = a.window > 0 ? max(0, c.all_pos - a.window + 1) : 0;
  c.all_lo = a.window > 0 ? max(0, c.wave_pos - a.window + 1) : 0;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = col0 + 16 * n + c.r;
    c.pos[n] = col < c.cols ? c.pos0 + col / a.group : -1;
    c.lo[n] = a.window > 0 ? max(0, c.pos[n] - a.window + 1) : 0;
  }
  return true;
}

// q of the wave's columns: entries 64 j + 16 g + .. of each.
template <int DP, int NT>
__device__ __forceinline__ void a8_load_q(const A8Args& a, const A8Rows<NT>& c, q_part (&q)[DP / 64][NT][A8_QJ]) {
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

// The page of the 16 keys from `key` on, and whether any of them is there for the wave; a page number outside the cache is no page.
template <int NT>
__device__ __forceinline__ int a8_page(const A8Args& a, const A8Rows<NT>& c, int key, bool& there) {
  there = key <= c.wave_pos && key + 15 >= c.wave_lo && key < a.W << a.lp;
  const int page = there ? a.table[(int64_t)c.seq * a.W + (key >> a.lp)] : 0;
  there = there && (unsigned)page < (unsigned)a.pages;
  return there ? page : 0;
}

// What a wave reads of a tile, and the scales that go with it.
template <int DP>
struct A8Tile {
  u32x4 k[4][DP / 64], v[DP / 16];
  float k_scale;             // of the keys that the lane reads
  int v_exp;                 // of the 16 keys whose values it reads, -256: none of them is there
};

template <int DP, int NT>
__device__ __forceinline__ void a8_load(const A8Args& a, const A8Rows<NT>& c, int kb, A8Tile<DP>& t) {
  bool k_there, v_there;
  const int kkey = kb + 16 * (c.r >> 2), vkey = kb + 16 * c.g;
  const int64_t kblock = (int64_t)a8_page(a, c, kkey, k_there) * a.nkv + c.kvh, vblock = (int64_t)a8_page(a, c, vkey, v_there) * a.nkv + c.kvh;
  const float ks = a.scales[2 * kblock], vs = a.scales[2 * vblock + 1];
  t.k_scale = k_there ? ks : 1.f;
  t.v_exp = v_there ? exponent_of(vs) : -256;
  const uint8_t* kp = a.kc + (kblock * a.P + (kkey & (a.P - 1)) + (c.r & 3)) * a.d + 16 * c.g;
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int j = 0; j < DP / 64; ++j)
      t.k[s][j] = 64 * j + 16 * c.g < a.d ? *reinterpret_cast<const u32x4*>(kp + 4 * s * a.d + 64 * j) : u32x4{0, 0, 0, 0};
  const uint8_t* vp = a.vc + (vblock * a.d + c.r) * a.P + (vkey & (a.P - 1));
#pragma unroll
  for (int dt = 0; dt < DP / 16; ++dt)
    if (16 * dt < a.d) t.v[dt] = *reinterpret_cast<const u32x4*>(vp + (int64_t)16 * dt * a.P);
}

// Bytes of four that hold a NaN, as 0x01 each.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u; }

// One tile onto the wave's sums: m, l and acc of a column, acc in units of 2^unit (the same for the wave).  full: every column that stands for a row sees every key.
template <int DP, int NT>
__device__ __forceinline__ void a8_tile(const A8Args& a, const A8Rows<NT>& c, int kb, A8Tile<DP>& t, const q_part (&q)[DP / 64][NT][A8_QJ], float (&m)[NT],
                                        float (&l)[NT], f32x4 (&acc)[NT][DP / 16], int& unit) {
  const bool full = kb >= c.all_lo && kb + A8_TILE - 1 <= c.all_pos && __all(t.v_exp > -256);
  f32x4 s[4][NT];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int n = 0; n < NT; ++n) s[i][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < DP / 64; ++j) keys_times<NT>(t.k[i][j], t.k_scale, q[j], s[i]);
  }
#ifdef VK_BF16
  // The unit never falls, so that sums are scaled down only: what a smaller page adds is then in units of a larger one's.
  float top = over_groups_max((float)t.v_exp);
  const int unit_now = max(unit, (int)top);
  const float to_unit = unit_now == unit ? 1.f : unit - unit_now < -126 ? 0.f : pow2f(unit - unit_now);
  unit = unit_now;
  const float v_scale = pow2f(max(-126, t.v_exp - unit));
#else
  const float to_unit = 1.f, v_scale = t.v_exp > -256 ? pow2f(t.v_exp) : 1.f;
#endif
  const bool there = t.v_exp > -256;
  w_part w[NT][A8_WP], seen[NT][A8_WP];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float p[16], top_s = -INFINITY;
    const int first = kb + 16 * c.g;
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const bool vis = full || (there && first + x >= c.lo[n] && first + x <= c.pos[n]);
      p[x] = vis ? s[x / 4][n][x % 4] : -INFINITY;
      top_s = fmaxf(top_s, p[x]);
    }
    const float m_new = fmaxf(m[n], over_groups_max(top_s) * a.scale_log2), ref = m_new > -INFINITY ? m_new : 0.f;
    const float by = exp2_fast(m[n] - ref);
    float sum = 0.f, ones[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const bool vis = full || (there && first + x >= c.lo[n] && first + x <= c.pos[n]);
      ones[x] = vis ? 1.f : 0.f;
      p[x] = vis ? exp2_fast(__builtin_fmaf(p[x], a.scale_log2, -ref)) : 0.f;
      sum = sum + p[x];
    }
    l[n] = __builtin_fmaf(l[n], by, over_groups_sum(sum));
    m[n] = m_new;
    set_weights(p, w[n]);
    set_weights(ones, seen[n]);
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt) acc[n][dt] = acc[n][dt] * (by * to_unit);
  }
  bool nan = false;
  if (!full) {
    // Values that no column sees are taken out; so are NaN, which some may not see.
    uint32_t keep[4];
    const int from = c.wave_lo - (kb + 16 * c.g), to = c.wave_pos - (kb + 16 * c.g);
#pragma unroll
    for (int b = 0; b < 16; ++b) {
      const uint32_t one = there && b >= from && b <= to ? 0xffu << 8 * (b & 3) : 0u;
      keep[b / 4] = b % 4 == 0 ? one : keep[b / 4] | one;
    }
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt)
      if (16 * dt < a.d) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          t.v[dt][b] &= keep[b];
          nan = nan || nan_bytes(t.v[dt][b]) != 0;
        }
      }
    nan = __any(nan);
  }
#pragma unroll
  for (int dt = 0; dt < DP / 16; ++dt) {
    if (16 * dt >= a.d) continue;
    f32x4 o[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n] = acc[n][dt];
    if (nan) {
      u32x4 where, clean;
      f32x4 count[NT];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const uint32_t x = nan_bytes(t.v[dt][b]);
        where[b] = x * 0x38u;                         // 1 in e4m3
        clean[b] = t.v[dt][b] & ~(x * 0xffu);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) count[n] = f32x4{0.f, 0.f, 0.f, 0.f};
      values_times<NT>(where, 1.f, seen, count);
      values_times<NT>(clean, v_scale, w, o);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = count[n][i] > 0.f ? NAN : o[n][i];
    } else {
      values_times<NT>(t.v[dt], v_scale, w, o);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][dt] = o[n];
  }
}

__device__ __forceinline__ float unit_of(int unit) {
#ifdef VK_BF16
  return unit > -256 ? pow2f(unit) : 1.f;
#else
  return 1.f;
#endif
}

// ---- prompts: a wave takes 16 NT columns of an item through all their keys.
template <int DP, int NT>
__global__ __launch_bounds__(256) void a8_prompt_kernel(A8Args a, int blocks_y) {
  A8Rows<NT> c;
  const int kvh = blockIdx.y % a.nkv, block = blockIdx.y / a.nkv, wave = threadIdx.x >> 6;
  if (!a8_rows<NT>(a, blockIdx.x, kvh, (block * 4 + wave) * 16 * NT, c)) return;
  q_part q[DP / 64][NT][A8_QJ];
  a8_load_q<DP, NT>(a, c, q);
  float m[NT], l[NT];
  f32x4 acc[NT][DP / 16];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt) acc[n][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  int unit = -256;
  A8Tile<DP> t;
  for (int kb = c.wave_lo & ~(A8_TILE - 1); kb <= c.wave_pos; kb += A8_TILE) {
    a8_load<DP, NT>(a, c, kb, t);
    a8_tile<DP, NT>(a, c, kb, t, q, m, l, acc, unit);
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = c.col0 + 16 * n + c.r;
    if (col >= c.cols) continue;
    const int row = col / a.group;
    elem_t* o = a.out + ((int64_t)(c.tok0 + row) * a.nq + kvh * a.group + col - row * a.group) * a.d + 4 * c.g;
    const float by = l[n] == 0.f ? 0.f : 1.f / l[n], u = unit_of(unit);
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt)
      if (16 * dt < a.d) store_elems4(o + 16 * dt, l[n] == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[n][dt] * by * u);
  }
}

// ---- few rows: a workgroup takes 16 NT columns through a segment of 256 keys, a wave a tile; segments are joined by a8_join_kernel.
// The segments that columns col0 .. have keys in; one that has none at all counts the first.
__device__ __forceinline__ void a8_segments(int lo, int pos, int& first, int& last) {
  last = max(pos, 0) / A8_SEG;
  first = min(lo / A8_SEG, last);
}

template <int DP, int NT>
__global__ __launch_bounds__(256) void a8_few_kernel(A8Args a) {
  extern __shared__ float sums[];                       // [4 waves][DP / 16][64 lanes][4]
  __shared__ float maxima[4][16 * NT], totals[4][16 * NT];
  A8Rows<NT> c;
  const int kvh = blockIdx.y % a.nkv, block = blockIdx.y / a.nkv, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, seg = blockIdx.z;
  if (!a8_rows<NT>(a, blockIdx.x, kvh, block * 16 * NT, c)) return;
  int seg_first, seg_last;
  a8_segments(c.wave_lo, c.wave_pos, seg_first, seg_last);
  if (seg < seg_first || seg > seg_last) return;
  const int kb = seg * A8_SEG + wave * A8_TILE;
  float m[NT], l[NT];
  f32x4 acc[NT][DP / 16];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt) acc[n][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  int unit = -256;
  if (kb <= c.wave_pos && kb + A8_TILE > c.wave_lo) {
    q_part q[DP / 64][NT][A8_QJ];
    A8Tile<DP> t;
    a8_load<DP, NT>(a, c, kb, t);
    a8_load_q<DP, NT>(a, c, q);
    a8_tile<DP, NT>(a, c, kb, t, q, m, l, acc, unit);
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
    if (c.g == 0) {
      maxima[wave][16 * n + c.r] = m[n];
      totals[wave][16 * n + c.r] = l[n];
    }
  __syncthreads();
  const int mine = DP / 64;                             // entries' tiles that a wave sums up: wave, wave + 4, ...
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = c.col0 + 16 * n + c.r;
    float top = maxima[0][16 * n + c.r];
#pragma unroll
    for (int x = 1; x < 4; ++x) top = fmaxf(top, maxima[x][16 * n + c.r]);
    const float ref = top > -INFINITY ? top : 0.f, by = exp2_fast(m[n] - ref) * unit_of(unit);
    float total = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) total = __builtin_fmaf(totals[x][16 * n + c.r], exp2_fast(maxima[x][16 * n + c.r] - ref), total);
    if (n > 0) __syncthreads();
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt) *reinterpret_cast<f32x4*>(sums + ((wave * (DP / 16) + dt) * 64 + lane) * 4) = acc[n][dt] * by;
    __syncthreads();
    if (col >= c.cols) continue;
    const int row = col / a.group;
    const int64_t part = (((int64_t)blockIdx.x * a.nkv + kvh) * a.nseg + seg) * a.cols_max + col;
#pragma unroll
    for (int x = 0; x < mine; ++x) {
      const int dt = 4 * x + wave;
      if (16 * dt >= a.d) continue;
      f32x4 o = *reinterpret_cast<const f32x4*>(sums + (dt * 64 + lane) * 4);
#pragma unroll
      for (int y = 1; y < 4; ++y) o = o + *reinterpret_cast<const f32x4*>(sums + ((y * (DP / 16) + dt) * 64 + lane) * 4);
      if (seg_first == seg_last) {
        store_elems4(a.out + ((int64_t)(c.tok0 + row) * a.nq + kvh * a.group + col - row * a.group) * a.d + 16 * dt + 4 * c.g,
                     total == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : o * (1.f / total));
      } else {
        *reinterpret_cast<f32x4*>(a.part_acc + part * a.d + 16 * dt + 4 * c.g) = o;
      }
    }
    if (seg_first != seg_last && wave == 0 && c.g == 0) *reinterpret_cast<f32x2*>(a.part_ml + 2 * part) = f32x2{top, total};
  }
}

// A wave a column: its segments' sums, in ascending order.
template <int NT>
__global__ __launch_bounds__(256) void a8_join_kernel(A8Args a) {
  A8Rows<NT> c;
  const int kvh = blockIdx.y, lane = threadIdx.x & 63, col = blockIdx.z * 4 + (threadIdx.x >> 6);
  if (!a8_rows<NT>(a, blockIdx.x, kvh, col / (16 * NT) * (16 * NT), c) || col >= c.cols) return;
  int seg_first, seg_last;
  a8_segments(c.wave_lo, c.wave_pos, seg_first, seg_last);
  if (seg_first == seg_last) return;                    // the other kernel wrote the result
  const int64_t part0 = ((int64_t)blockIdx.x * a.nkv + kvh) * a.nseg * a.cols_max + col;
  float top = -INFINITY;
  for (int s = seg_first + lane; s <= seg_last; s += 64) top = fmaxf(top, a.part_ml[2 * (part0 + (int64_t)s * a.cols_max)]);
  top = wave_max_xor(top);
  const float ref = top > -INFINITY ? top : 0.f;
  float total = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = seg_first; s <= seg_last; ++s) {
    const int64_t part = part0 + (int64_t)s * a.cols_max;
    const f32x2 ml = *reinterpret_cast<const f32x2*>(a.part_ml + 2 * part);
    const float by = exp2_fast(ml.x - ref);
    total = __builtin_fmaf(ml.y, by, total);
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (lane + 64 * x < a.d) o[x] = __builtin_fmaf(a.part_acc[part * a.d + lane + 64 * x], by, o[x]);
  }
  const int row = col / a.group;
  elem_t* to = a.out + ((int64_t)(c.tok0 + row) * a.nq + kvh * a.group + col - row * a.group) * a.d;
#pragma unroll
  for (int x = 0; x < 4; ++x)
    if (lane + 64 * x < a.d) to[lane + 64 * x] = from_f32<elem_t>(total == 0.f ? 0.f : o[x] / total);
}

// Column tiles a wave of the few rows' kernel takes at once: as many as there are columns, up to what its registers hold.
static int few_tiles(int cols, int d) { return cols <= 16 || d > 128 ? 1 : cols <= 32 || sizeof(elem_t) == 4 ? 2 : 4; }

extern "C" {

int vk_attn8_item_rows(void) { return A8_ITEM_ROWS; }

// 32-bit words of scratch for `items` items of up to item_rows <= 16 rows: 0 for more rows, whose keys are not split, and for few keys.
int64_t vk_attn8_scratch_floats(int items, int item_rows, int nq, int d, int max_k_len) {
  const int64_t nseg = ((int64_t)max_k_len + A8_SEG - 1) / A8_SEG;
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
  if (n_items == 0 || T == 0 || S == 0) return 0;
  VK_REQUIRE(((uintptr_t)q | (uintptr_t)out | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)scratch) % 16 == 0, "attention8: rows, cache and scratch have to lie on 16 bytes");
  const int group = nq / nkv, nseg = max(1, (int)(((int64_t)max_k_len + A8_SEG - 1) / A8_SEG));
  A8Args a{q, out, kc, vc, scales, table, cu_q, k_len, items, nullptr, nullptr, W, T, S, nq, nkv, d, P, 0, pages, group, item_rows, item_rows * group, window, nseg,
           scale * 1.4426950408889634f};
  while (1 << a.lp < P) ++a.lp;
  if (item_rows > 16) {
    constexpr int NT = sizeof(elem_t) == 4 ? 1 : 2;
    const int blocks = (a.cols_max + 64 * NT - 1) / (64 * NT);
    VK_REQUIRE((int64_t)blocks * nkv <= 65535, "attention8: %d heads of %d rows are too many for one launch", nq, item_rows);
#define PROMPT(D) a8_prompt_kernel<D, NT><<<dim3(n_items, nkv * blocks), 256, 0, st>>>(a, blocks)
    if (d <= 64) PROMPT(64);
    else if (d <= 128) PROMPT(128);
    else if (d <= 192) PROMPT(192);
    else PROMPT(256);
#undef PROMPT
    return vk_check_launch("attention8 (prompt)");
  }
  const int64_t need = vk_attn8_scratch_floats(n_items, item_rows, nq, d, max_k_len);
  VK_REQUIRE(need == 0 || (scratch != nullptr && scratch_floats >= need), "attention8: scratch of %lld floats needed", (long long)need);
  a.part_acc = scratch;
  a.part_ml = scratch + need / (d + 2) * d;
  const int nt = few_tiles(a.cols_max, d), blocks = (a.cols_max + 16 * nt - 1) / (16 * nt);
  VK_REQUIRE((int64_t)blocks * nkv <= 65535 && nseg <= 65535 && (a.cols_max + 3) / 4 <= 65535, "attention8: %d heads, %d keys: too many for one launch", nq, max_k_len);
  const dim3 grid(n_items, nkv * blocks, nseg), join(n_items, nkv, (a.cols_max + 3) / 4);
#define FEW(D, N) (a8_few_kernel<D, N><<<grid, 256, D * 256, st>>>(a))
#ifdef VK_BF16
#define FEW_D(D) (nt == 1 ? FEW(D, 1) : nt == 2 ? FEW(D, 2) : FEW(D, 4))
#else
#define FEW_D(D) (nt == 1 ? FEW(D, 1) : FEW(D, 2))
#endif
  if (d <= 64) FEW_D(64);
  else if (d <= 128) FEW_D(128);
  else if (d <= 192) FEW(192, 1);
  else FEW(256, 1);
#undef FEW_D
#undef FEW
  if (vk_check_launch("attention8")) return 1;
  if (nseg == 1) return 0;
  if (nt == 1) a8_join_kernel<1><<<join, 256, 0, st>>>(a);
  else if (nt == 2) a8_join_kernel<2><<<join, 256, 0, st>>>(a);
  else a8_join_kernel<4><<<join, 256, 0, st>>>(a);
  return vk_check_launch("attention8 (join)");
}

}  // extern "C"
