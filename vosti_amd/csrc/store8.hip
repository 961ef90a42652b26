// What stands between the projections and attention over an 8-bit cache (cache8.h), in one launch: norm of q's and k's heads, rotation by
// tables, and the append of k and v to their pages, whose scales grow where the new entries ask for it.
//
//   norm    y = x / sqrt(mean(x^2) + eps) * w            q and k, a weight [d] for all heads
//   turn    (y_c, y_c+h) by the angle of the row's place: y_c cos - y_c+h sin, y_c+h cos + y_c sin, c < h = rot_half
//   scale   of (page, head, k or v): 2^e, e the least with which no entry given to the page so far exceeds 448 of it; a page that begins with
//           this call starts anew
//   entry   x / 2^e to the nearest e4m3, half to even; the page's other entries are rounded once more where e has grown
//
// q is computed in 32-bit and rounded to the element type once.  k is computed in 64-bit: its entries keep four digits, and which ones they keep is decided by
// the formula and not by the last bits of its evaluation; in between they are rounded to odd, to 32 and to 16 bits, which changes no rounding to four digits (the vector unit's 64-bit additions and products are as fast as its 32-bit ones).
//
// A row of the step stands at place k_len - (rows of its sequence) + its number, in page table[sequence][place / P].  A workgroup takes
// one (page, head, k or v) that the step writes to, so that the scale, the new entries and the old ones are one workgroup's
// business; rows come to it by their sequence, not by slots.  The other workgroups take a token's q heads each.
//
// Measured (MI355X, bfloat16, 32 q and 8 kv heads of 128, pages of 64; a copy reaches 4.75 TB/s here): a prompt of 4,096 tokens, 93 MB: 31 us, 28.6 in a row of calls, 3.0 to 3.3 TB/s: four
// workgroups a CU is what the 64-bit norm's registers leave (five or six spill: 38 -> 50 us with nothing in the caches), and a page's rows wait for their maximum.  Rows and angles that are read one row ahead, as
// they are stored, took 3 us off it and 2 off a step of 64 tokens.  A token each of 64 sequences, 1.5 MB: 8.8 us where no page's scale grows: the sequence's lengths, then the page's number and
// its scale, one load behind the other; 16.7 where a third of them do: a page's entries behind that.  The 32-bit build, 2,300 tokens of 7 sequences, 16 and 8 heads of 64: 13 us, whether scales grow or not.
#include "cache8.h"
#include "vec.h"

#define STORE8_THREADS 256

struct Store8Args {
  const elem_t* qkv;        // [T, row_stride]: nq q heads, nkv k heads, nkv v heads, d each
  int64_t row_stride;
  elem_t* q_out;            // [T, nq, d]
  uint8_t* kc;
  uint8_t* vc;
  float* scales;
  const void *q_w, *k_w;    // [d] or null
  int w_is_f32;
  const elem_t *cos_t, *sin_t;   // [at least max_k_len, rot_half] or null
  int rot_half;
  int whole;                // weights and tables lie on 16 bytes, and rot_half is a whole number of vectors: a lane's entries of them are read at once
  const int32_t *table, *cu_q, *k_len;
  int W, T, S, nq, nkv, d, P, lp, pages, kv_blocks, held, max_k_len;
  double eps, per_d;        // per_d: 1 / d
};

// Sum over the LPH neighbouring lanes of a head; the order is fixed by LPH.
template <int LPH>
__device__ __forceinline__ float head_sum(float v) { return group_sum<LPH>(v); }
template <int LPH>
__device__ __forceinline__ double head_sum(double v) {
  if (LPH >= 2) v = v + dpp_d<0xB1>(v);               // quad_perm [1, 0, 3, 2]
  if (LPH >= 4) v = v + dpp_d<0x4E>(v);               // quad_perm [2, 3, 0, 1]
  if (LPH >= 8) v = v + dpp_d<0x141>(v);              // row_half_mirror
  if (LPH >= 16) v = v + dpp_d<0x140>(v);             // row_mirror
  if (LPH >= 32) v = add_xor16(v);
  if (LPH >= 64) v = add_xor32(v);
  return v;
}
__device__ __forceinline__ float one_over_root(float v) { return rsqrtf(v); }
__device__ __forceinline__ double one_over_root(double v) { return rsqrt(v); }

// Sixteen bytes of elements, as they are read; element e of them.
__device__ __forceinline__ u32x4 read_raw(const elem_t* p, bool aligned) {
  if (aligned) return *reinterpret_cast<const u32x4*>(p);
  u32x4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
#ifdef VK_BF16
    r[e] = (uint32_t)__builtin_bit_cast(uint16_t, p[2 * e]) | (uint32_t)__builtin_bit_cast(uint16_t, p[2 * e + 1]) << 16;
#else
    r[e] = __builtin_bit_cast(uint32_t, p[e]);
#endif
  }
  return r;
}
__device__ __forceinline__ float element(u32x4 r, int e) {
#ifdef VK_BF16
  return __builtin_bit_cast(float, (e & 1) ? r[e / 2] & 0xffff0000u : r[e / 2] << 16);
#else
  return __builtin_bit_cast(float, (uint32_t)r[e]);
#endif
}

// The norm's weights of a lane's VK_VEC entries of a head, from entry c0 on.
__device__ __forceinline__ void read_weights(const Store8Args& a, const void* w, int c0, float (&to)[VK_VEC]) {
  const int at = min(c0, a.d - VK_VEC);                 // lanes behind the head have nothing to multiply
  if (a.whole && !a.w_is_f32) {
    load_elems(static_cast<const elem_t*>(w) + at, to);
  } else {
#pragma unroll
    for (int e = 0; e < VK_VEC; ++e) to[e] = load_weight(w, a.w_is_f32, at + e);
  }
}
// The cosines and sines that they turn by.  Entry c turns with entry c + h, c < h, and c - h, c < 2 h; others stand.
struct Angles {
  u32x4 cs, sn;
};
__device__ __forceinline__ void read_angles(const Store8Args& a, int c0, int place, Angles& t) {
  const int h = a.rot_half;
  const elem_t *cs = a.cos_t + (int64_t)place * h, *sn = a.sin_t + (int64_t)place * h;
  if (a.whole) {
    const int at = c0 < h ? c0 : c0 < 2 * h ? c0 - h : 0;
    t.cs = read_raw(cs + at, true);
    t.sn = read_raw(sn + at, true);
  } else {
    elem_t c_of[VK_VEC], s_of[VK_VEC];
#pragma unroll
    for (int e = 0; e < VK_VEC; ++e) {
      const int c = c0 + e, at = c < h ? c : c < 2 * h ? c - h : 0;
      c_of[e] = cs[at];
      s_of[e] = sn[at];
    }
    t.cs = read_raw(c_of, false);
    t.sn = read_raw(s_of, false);
  }
}

// Norm and turn of a lane's entries.  y: the head's own LPH * VK_VEC numbers of LDS, for rotations that are no whole vectors.
template <int LPH, typename F>
__device__ __forceinline__ void norm_and_turn(F (&v)[VK_VEC], const Store8Args& a, bool norm, const float (&w)[VK_VEC], const Angles& t, int c0, F* y) {
  if (norm) {
    F part = 0;
#pragma unroll
    for (int e = 0; e < VK_VEC; ++e) part = part + v[e] * v[e];
    const F r = one_over_root(head_sum<LPH>(part) * (F)a.per_d + (F)a.eps);
#pragma unroll
    for (int e = 0; e < VK_VEC; ++e) v[e] = v[e] * r * (F)w[e];
  }
  if (a.cos_t != nullptr) {
    const int h = a.rot_half;
    F other[VK_VEC];
    if (a.whole) {                                      // another lane's vector
      const int lane = threadIdx.x & 63, from = c0 < h ? lane + h / VK_VEC : c0 < 2 * h ? lane - h / VK_VEC : lane;
#pragma unroll
      for (int e = 0; e < VK_VEC; ++e) other[e] = __shfl(v[e], from);
    } else {
#pragma unroll
      for (int e = 0; e < VK_VEC; ++e) y[c0 + e] = v[e];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int e = 0; e < VK_VEC; ++e) other[e] = y[c0 + e < h ? c0 + e + h : c0 + e < 2 * h ? c0 + e - h : c0 + e];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int e = 0; e < VK_VEC; ++e) {
      const int c = c0 + e;
      const float cs = c < 2 * h ? element(t.cs, e) : 1.f, sn = c < h ? -element(t.sn, e) : c < 2 * h ? element(t.sn, e) : 0.f;
      v[e] = v[e] * (F)cs + other[e] * (F)sn;
    }
  }
}

// The rows of sequence i: how many, from which one on, and its keys; none where the arrays do not make sense.
__device__ __forceinline__ int rows_of(const Store8Args& a, int i, int& first, int& keys) {
  first = keys = 0;
  if (i >= a.S) return 0;
  first = a.cu_q[i];
  keys = a.k_len[i];
  const int end = a.cu_q[i + 1];
  return first >= 0 && first < end && end <= a.T && end - first <= keys && keys <= a.max_k_len ? end - first : 0;
}

// A number between its maximum and its rounding to four digits: the first eight of them, the last one set where more were lost, so that it is rounded, and compared with 448 of a scale, as it was.
__device__ __forceinline__ uint32_t held_of(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  return u >> 16 | ((u & 0xffffu) != 0 ? 1u : 0u);
}
__device__ __forceinline__ float number_of(uint32_t held) { return __builtin_bit_cast(float, held << 16); }

// LDS of a workgroup: each wave's heads while they turn, and the new entries of a page, `held` rows of d numbers, between their maximum and their rounding.
constexpr int STORE8_TURN = 4 * 64 * VK_VEC;

template <int LPH>
__global__ __launch_bounds__(STORE8_THREADS, 4) void store8_kernel(Store8Args a) {
  constexpr int HPW = 64 / LPH, ROWS = 4 * HPW;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ int wave_need[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane / LPH, c0 = lane % LPH * VK_VEC, d = a.d, P = a.P, block = blockIdx.x;
  const bool inside = c0 < d;

  if (block >= a.kv_blocks) {
    // ---- a token's q heads
    const int tok = block - a.kv_blocks;
    const elem_t* row = a.qkv + (int64_t)tok * a.row_stride + c0;
    float* y = reinterpret_cast<float*>(lds) + (wave * HPW + sub) * LPH * VK_VEC;
    u32x4 next;
    auto ask = [&](int h) {
      next = u32x4{0, 0, 0, 0};
      if (h + sub < a.nq && inside) next = read_raw(row + (h + sub) * d, true);
    };
    ask(wave * HPW);
    float w[VK_VEC];
    Angles t;
    if (a.q_w != nullptr) read_weights(a, a.q_w, c0, w);
    int place = -1;
    for (int base = 0; base < a.S && place < 0; base += 64) {
      int first, keys;
      const int n = rows_of(a, base + lane, first, keys);
      const uint64_t mine = __ballot(tok >= first && tok < first + n);
      if (mine != 0) place = __builtin_amdgcn_readlane(keys - n + tok - first, __builtin_ctzll(mine));
    }
    if (place < 0) return;                            // behind the last sequence's rows
    if (a.cos_t != nullptr) read_angles(a, c0, place, t);
    for (int h = wave * HPW; h < a.nq; h += ROWS) {
      float v[VK_VEC];
#pragma unroll
      for (int e = 0; e < VK_VEC; ++e) v[e] = element(next, e);
      ask(h + ROWS);
      norm_and_turn<LPH>(v, a, a.q_w != nullptr, w, t, c0, y);
      if (h + sub < a.nq && inside) store_elems(a.q_out + ((int64_t)tok * a.nq + h + sub) * d + c0, v);
    }
    return;
  }

  // ---- a page's new keys or values of one head
  const int job = block / (a.nkv * 2), head = (block >> 1) % a.nkv;
  const bool is_v = block & 1;
  float w[VK_VEC];
  if (!is_v && a.k_w != nullptr) read_weights(a, a.k_w, c0, w);
  int seq = -1, tok0 = 0, off0 = 0, m = 0, pidx = 0;
  for (int base = 0, run = 0; base < a.S; base += 64) {
    int first, keys;
    const int n = rows_of(a, base + lane, first, keys), from = keys - n;
    const int mine = n > 0 ? ((keys - 1) >> a.lp) - (from >> a.lp) + 1 : 0;
    int upto = mine;                                  // pages of the sequences up to this lane's
    upto += __builtin_amdgcn_update_dpp(0, upto, 0x111, 0xF, 0xF, true);      // row_shr 1, 2, 4, 8: within 16 lanes
    upto += __builtin_amdgcn_update_dpp(0, upto, 0x112, 0xF, 0xF, true);
    upto += __builtin_amdgcn_update_dpp(0, upto, 0x114, 0xF, 0xF, true);
    upto += __builtin_amdgcn_update_dpp(0, upto, 0x118, 0xF, 0xF, true);
    const int r0 = __builtin_amdgcn_readlane(upto, 15), r1 = r0 + __builtin_amdgcn_readlane(upto, 31), r2 = r1 + __builtin_amdgcn_readlane(upto, 47);
    upto += lane < 16 ? 0 : lane < 32 ? r0 : lane < 48 ? r1 : r2;
    const uint64_t hit = __ballot(job < run + upto);
    if (hit != 0) {
      const int l = __builtin_ctzll(hit);
      const int before = run + __builtin_amdgcn_readlane(upto - mine, l), k = __builtin_amdgcn_readlane(keys, l), f = __builtin_amdgcn_readlane(from, l);
      seq = base + l;
      pidx = (f >> a.lp) + job - before;
      const int lo = max(pidx << a.lp, f), hi = min((pidx + 1) << a.lp, k);
      off0 = lo - (pidx << a.lp);
      m = hi - lo;
      tok0 = __builtin_amdgcn_readlane(first, l) + lo - f;
      break;
    }
    run += __builtin_amdgcn_readlane(upto, 63);
  }
  if (seq < 0 || pidx >= a.W) return;
  const elem_t* rows = a.qkv + (int64_t)tok0 * a.row_stride + (a.nq + head + (is_v ? a.nkv : 0)) * d + c0;
  const int place0 = (pidx << a.lp) + off0;
  // A row's entries and its angles, asked for one row of the lane's ahead.
  const bool turns = !is_v && a.cos_t != nullptr;
  u32x4 next;
  Angles next_t;
  auto ask = [&](int i) {
    next = u32x4{0, 0, 0, 0};
    if (i < m && inside) next = read_raw(rows + (int64_t)i * a.row_stride, true);
    if (turns) read_angles(a, c0, place0 + min(i, m - 1), next_t);
  };
  ask(wave * HPW + sub);
  const int page = a.table[(int64_t)seq * a.W + pidx];
  if ((unsigned)page >= (unsigned)a.pages) return;    // a sequence whose rows are not to be kept
  const int64_t head_page = (int64_t)page * a.nkv + head;
  float* scale = a.scales + head_page * 2 + (is_v ? 1 : 0);
  const int stood = exponent_of(*scale), old = off0 > 0 ? stood : CACHE8_LOWEST;

  double* y = reinterpret_cast<double*>(lds) + (wave * HPW + sub) * LPH * VK_VEC;
  uint16_t* held = reinterpret_cast<uint16_t*>(lds + (a.whole ? 0 : STORE8_TURN * sizeof(double)));
  // Rows i0 .. i0 + a.held - 1 into LDS: values as they are, keys normed and turned.  Returns the exponent that this lane's need.
  auto entries = [&](int i0) {
    int need = CACHE8_LOWEST;
    const int end = min(m, i0 + a.held);
    for (int r0 = i0; r0 < end; r0 += ROWS) {
      const int i = r0 + wave * HPW + sub;
      float v[VK_VEC];
#pragma unroll
      for (int e = 0; e < VK_VEC; ++e) v[e] = element(next, e);
      const Angles t = next_t;
      ask(i + ROWS);
      if (!is_v) {
        double k[VK_VEC];
#pragma unroll
        for (int e = 0; e < VK_VEC; ++e) k[e] = (double)v[e];
        norm_and_turn<LPH>(k, a, a.k_w != nullptr, w, t, c0, y);
#pragma unroll
        for (int e = 0; e < VK_VEC; ++e) v[e] = round_to_odd(k[e]);
      }
      if (i < end && inside) {
        uint32_t pair[VK_VEC / 2];
#pragma unroll
        for (int e = 0; e < VK_VEC; ++e) need = max(need, least_exponent(v[e]));
#pragma unroll
        for (int e = 0; e < VK_VEC; e += 2) pair[e / 2] = held_of(v[e]) | held_of(v[e + 1]) << 16;
        uint32_t* to = reinterpret_cast<uint32_t*>(held + (i - i0) * d + c0);
#pragma unroll
        for (int e = 0; e < VK_VEC / 2; ++e) to[e] = pair[e];
      }
    }
    return need;
  };
  int need = entries(0);
  for (int i0 = a.held; i0 < m; i0 += a.held) {       // more rows than LDS holds: their maximum first, and once more for their entries
    __syncthreads();
    ask(i0 + wave * HPW + sub);
    need = max(need, entries(i0));
  }
  need = (int)wave_max_xor((float)need);
  if (lane == 0) wave_need[wave] = need;
  __syncthreads();
  const int now = max(max(old, max(wave_need[0], wave_need[1])), max(wave_need[2], wave_need[3]));

  uint8_t* kp = a.kc + head_page * P * d;
  uint8_t* vp = a.vc + head_page * P * d;
  for (int i0 = 0; i0 < m; i0 += a.held) {
    const int n = min(a.held, m - i0), at = off0 + i0;           // rows in LDS, and the place in the page of the first
    if (m > a.held) {
      __syncthreads();
      ask(i0 + wave * HPW + sub);
      (void)entries(i0);
      __syncthreads();
    }
    if (!is_v) {
      for (int x = threadIdx.x; x < n * d / 16; x += STORE8_THREADS) {
        const u32x4 lo = *reinterpret_cast<const u32x4*>(held + x * 16), hi = *reinterpret_cast<const u32x4*>(held + x * 16 + 8);
        const uint32_t from[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        u32x4 b;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          b[e] = to_fp8x4(entry_of(number_of(from[2 * e]), now), entry_of(number_of(from[2 * e] >> 16), now), entry_of(number_of(from[2 * e + 1]), now), entry_of(number_of(from[2 * e + 1] >> 16), now));
        *reinterpret_cast<u32x4*>(kp + at * d + x * 16) = b;
      }
    } else {
      // Sixteen places of an entry: neighbouring threads take neighbouring entries, which lie side by side in LDS.
      const int o0 = at & ~15, chunks = (at + n - o0 + 15) >> 4;
      constexpr int WIDE = LPH * VK_VEC;              // d, filled up to a power of two
      const int c = threadIdx.x % WIDE;
      for (int x = threadIdx.x / WIDE; x < (c < d ? chunks : 0); x += STORE8_THREADS / WIDE) {
        const int o = o0 + (x << 4);
        if (o >= at && o + 16 <= at + n) {
          const uint16_t* from = held + (o - at) * d + c;
          u32x4 b;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            b[e] = to_fp8x4(entry_of(number_of(from[4 * e * d]), now), entry_of(number_of(from[(4 * e + 1) * d]), now), entry_of(number_of(from[(4 * e + 2) * d]), now),
                            entry_of(number_of(from[(4 * e + 3) * d]), now));
          *reinterpret_cast<u32x4*>(vp + c * P + o) = b;
        } else {
          for (int b = max(at, o); b < min(at + n, o + 16); ++b) vp[c * P + b] = (uint8_t)to_fp8x4(entry_of(number_of(held[(b - at) * d + c]), now), 0.f, 0.f, 0.f);
        }
      }
    }
  }
  if (now > stood) {                                  // the page's other entries in the new scale
    const float by = now - stood > 126 ? 0.f : pow2f(stood - now);
    auto again = [&](uint32_t x) {
      const f32x2 lo = from_fp8x2<false>(x, 1.f), hi = from_fp8x2<true>(x, 1.f);
      return to_fp8x4(lo.x * by, lo.y * by, hi.x * by, hi.y * by);
    };
    if (!is_v) {
      uint32_t* p = reinterpret_cast<uint32_t*>(kp);
      const int row = d / 4, end = off0 * row;
      for (int x = threadIdx.x; x < (P - m) * row; x += STORE8_THREADS) {
        const int at = x < end ? x : x + m * row;
        p[at] = again(p[at]);
      }
    } else {
      for (int x = threadIdx.x; x < d * (P >> 4); x += STORE8_THREADS) {
        const int c = x / (P >> 4), o = (x % (P >> 4)) << 4;
        uint8_t* p = vp + c * P + o;
        if (o + 16 <= off0 || o >= off0 + m) {
          u32x4 v = *reinterpret_cast<u32x4*>(p);
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = again(v[i]);
          *reinterpret_cast<u32x4*>(p) = v;
        } else {                                      // the new ones beside them are other threads'
          for (int b = 0; b < 16; ++b)
            if (o + b < off0 || o + b >= off0 + m) p[b] = (uint8_t)again(p[b]);
        }
      }
    }
  }
  if (threadIdx.x == 0 && now != stood) *scale = pow2f(now);
}

extern "C" {

// Norm, rotation and append of a step's rows.  qkv [T, row_stride], q_out [T, nq, d] (nq may be 0: keys and values alone; nkv may be 0: q alone); the pages'
// tensors as in cache8.h; q_w / k_w null: no norm; cos_t null: no rotation, else tables of at least max_k_len rows; table [S, W], cu_q [S + 1], k_len [S]
// (keys with the step's rows).  max_k_len: the host's bound on k_len.  A sequence whose arrays exceed the bounds, and rows behind the last sequence's, leave
// everything as it was; rows whose page number is not in the cache are not kept.
int vk_qkv_post8(const elem_t* qkv, int64_t row_stride, elem_t* q_out, uint8_t* kc, uint8_t* vc, float* scales, const void* q_w, const void* k_w, int w_is_f32,
                 const elem_t* cos_t, const elem_t* sin_t, int rot_half, const int32_t* table, int W, const int32_t* cu_q, const int32_t* k_len, int T, int S,
                 int nq, int nkv, int d, int P, int pages, int max_k_len, double eps, hipStream_t st) {
  VK_REQUIRE(T >= 0 && S >= 0 && nq >= 0 && nkv >= 0 && nq + nkv > 0, "qkv_post8: bad sizes T=%d S=%d nq=%d nkv=%d", T, S, nq, nkv);
  VK_REQUIRE(d >= 16 && d <= 256 && d % 16 == 0, "qkv_post8: head size %d is no multiple of 16 from 16 to 256", d);
  VK_REQUIRE(nkv == 0 || (P >= CACHE8_MIN_PAGE && P <= CACHE8_MAX_PAGE && (P & (P - 1)) == 0), "qkv_post8: page size %d is no power of two from %d to %d", P,
             CACHE8_MIN_PAGE, CACHE8_MAX_PAGE);
  VK_REQUIRE(row_stride >= (int64_t)(nq + 2 * nkv) * d && row_stride % VK_VEC == 0, "qkv_post8: row stride %lld does not hold %d heads, or not in whole vectors",
             (long long)row_stride, nq + 2 * nkv);
  VK_REQUIRE(cos_t == nullptr || (sin_t != nullptr && rot_half > 0 && 2 * rot_half <= d), "qkv_post8: rotation of %d pairs in heads of %d", rot_half, d);
  VK_REQUIRE(nkv == 0 || (kc != nullptr && vc != nullptr && scales != nullptr && pages > 0 && W > 0), "qkv_post8: the cache is missing");
  VK_REQUIRE(nq == 0 || q_out != nullptr, "qkv_post8: q_out is missing");
  VK_REQUIRE(max_k_len >= 0 && (nkv == 0 || (int64_t)W * P >= max_k_len), "qkv_post8: a table of %d pages of %d does not cover %d keys", W, P, max_k_len);
  if (T == 0 || S == 0) return 0;
  VK_REQUIRE(((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)kc | (uintptr_t)vc) % 16 == 0, "qkv_post8: rows and cache have to lie on 16 bytes");
  Store8Args a{qkv, row_stride, q_out, kc, vc, scales, q_w, k_w, w_is_f32, cos_t, sin_t, rot_half, 0, table, cu_q, k_len, W, T, S, nq, nkv, d, P, 0, pages, 0, 0,
               max_k_len, eps, 1.0 / d};
  while (1 << a.lp < P) ++a.lp;
  a.whole = rot_half % VK_VEC == 0 && ((uintptr_t)q_w | (uintptr_t)k_w | (uintptr_t)cos_t | (uintptr_t)sin_t) % 16 == 0;
  // Pages that n rows of a sequence touch: n at most, and (n - 1) / P + 2.
  const int64_t jobs = nkv > 0 ? min((int64_t)T, (int64_t)T / P + 2 * (int64_t)S) : 0, kv_blocks = jobs * nkv * 2, q_blocks = nq > 0 ? T : 0;
  VK_REQUIRE(kv_blocks + q_blocks < (1ll << 31), "qkv_post8: %d rows of %d heads are too many for one launch", T, nq + 2 * nkv);
  a.kv_blocks = (int)kv_blocks;
  // Rows that a workgroup holds in LDS: a page's, up to 32 KB (four workgroups a CU), and one where every sequence has one.
  a.held = T <= S ? 1 : min(P, 32 * 1024 / 2 / d);
  const int lds_q = a.whole ? 0 : STORE8_TURN * (int)sizeof(float), lds_kv = a.held * d * 2 + (a.whole ? 0 : STORE8_TURN * (int)sizeof(double));
  const int vecs = d / VK_VEC;
#define STORE8(L) store8_kernel<L><<<(unsigned)(kv_blocks + q_blocks), STORE8_THREADS, kv_blocks > 0 ? lds_kv : lds_q, st>>>(a);
#ifdef VK_BF16
  if (vecs <= 2) STORE8(2)
  else if (vecs <= 4) STORE8(4)
  else if (vecs <= 8) STORE8(8)
  else if (vecs <= 16) STORE8(16)
  else STORE8(32)
#else
  if (vecs <= 4) STORE8(4)
  else if (vecs <= 8) STORE8(8)
  else if (vecs <= 16) STORE8(16)
  else if (vecs <= 32) STORE8(32)
  else STORE8(64)
#endif
#undef STORE8
  return vk_check_launch("qkv_post8");
}

}  // extern "C"
