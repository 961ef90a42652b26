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
// the formula and not by the last bits of its evaluation (the vector unit's 64-bit additions and products are as fast as its 32-bit ones).
//
// A row of the step stands at place k_len - (rows of its sequence) + its number, in page table[sequence][place / P].  A workgroup takes
// one (page, head, k or v) that the step writes to, so that the scale, the new entries and the old ones are one workgroup's
// business; rows come to it by their sequence, not by slots.  The other workgroups take a token's q heads each.
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
  const int32_t *table, *cu_q, *k_len;
  int W, T, S, nq, nkv, d, P, lp, pages, kv_jobs, max_k_len;
  double eps;
};

// Sum over the LPH neighbouring lanes of a head; the order is fixed by LPH.
template <int LPH>
__device__ __forceinline__ float head_sum(float v) { return group_sum<LPH>(v); }
template <int LPH>
__device__ __forceinline__ double head_sum(double v) {
#pragma unroll
  for (int off = 1; off < LPH; off <<= 1) v = v + __shfl_xor(v, off);
  return v;
}
__device__ __forceinline__ float root_of(float v) { return sqrtf(v); }
__device__ __forceinline__ double root_of(double v) { return sqrt(v); }

// A lane's VK_VEC entries of a head, from entry c0 on: norm and turn.  y: the head's own LPH * VK_VEC numbers of LDS.
template <int LPH, typename F>
__device__ __forceinline__ void norm_and_turn(F (&v)[VK_VEC], const Store8Args& a, const void* w, int c0, int place, F* y) {
  if (w != nullptr) {
    F part = 0;
#pragma unroll
    for (int e = 0; e < VK_VEC; ++e) part = part + v[e] * v[e];
    const F r = (F)1 / root_of(head_sum<LPH>(part) / (F)a.d + (F)a.eps);
#pragma unroll
    for (int e = 0; e < VK_VEC; ++e) v[e] = c0 + e < a.d ? v[e] * r * (F)load_weight(w, a.w_is_f32, c0 + e) : (F)0;
  }
  if (a.cos_t != nullptr) {
    const int h = a.rot_half;
    const elem_t *cs = a.cos_t + (int64_t)place * h, *sn = a.sin_t + (int64_t)place * h;
#pragma unroll
    for (int e = 0; e < VK_VEC; ++e) y[c0 + e] = v[e];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int e = 0; e < VK_VEC; ++e) {
      const int c = c0 + e;
      if (c < h) v[e] = v[e] * (F)to_f32(cs[c]) - y[c + h] * (F)to_f32(sn[c]);
      else if (c < 2 * h) v[e] = v[e] * (F)to_f32(cs[c - h]) + y[c - h] * (F)to_f32(sn[c - h]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// The rows of sequence i: how many, from which one on, and its keys; none where the arrays do not make sense.
__device__ __forceinline__ int rows_of(const Store8Args& a, int i, int& first, int& keys) {
  first = keys = 0;
  if (i >= a.S) return 0;
  first = a.cu_q[i];
  keys = a.k_len[i];
  const int end = a.cu_q[i + 1], n = end - first;
  return first >= 0 && end <= a.T && n > 0 && n <= keys && keys <= a.max_k_len ? n : 0;
}

template <int LPH>
__global__ __launch_bounds__(STORE8_THREADS) void store8_kernel(Store8Args a) {
  constexpr int HPW = 64 / LPH;
  __shared__ double turn_rows[4][64 * VK_VEC];
  __shared__ int wave_need[4];
  extern __shared__ uint8_t turned[];                // v's new entries, [d][P + 4]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane % LPH, sub = lane / LPH, c0 = j * VK_VEC, d = a.d, P = a.P;
  const bool inside = c0 < d;

  if ((int)blockIdx.x >= a.kv_jobs * a.nkv * 2) {
    // ---- a token's q heads
    const int tok = blockIdx.x - a.kv_jobs * a.nkv * 2;
    int place = -1;
    for (int base = 0; base < a.S && place < 0; base += 64) {
      int first, keys;
      const int n = rows_of(a, base + lane, first, keys);
      const uint64_t mine = __ballot(tok >= first && tok < first + n);
      if (mine != 0) place = __shfl(keys - n + tok - first, __builtin_ctzll(mine));
    }
    if (place < 0) return;                            // behind the last sequence's rows
    float* y = reinterpret_cast<float*>(turn_rows[wave]) + sub * LPH * VK_VEC;
    for (int h = wave * HPW; h < a.nq; h += 4 * HPW) {
      const bool live = h + sub < a.nq && inside;
      float v[VK_VEC];
#pragma unroll
      for (int e = 0; e < VK_VEC; ++e) v[e] = 0.f;
      if (live) load_elems(a.qkv + (int64_t)tok * a.row_stride + (h + sub) * d + c0, v);
      norm_and_turn<LPH>(v, a, a.q_w, c0, place, y);
      if (live) store_elems(a.q_out + ((int64_t)tok * a.nq + h + sub) * d + c0, v);
    }
    return;
  }

  // ---- a page's new keys or values of one head
  const int job = blockIdx.x / (a.nkv * 2), head = (blockIdx.x >> 1) % a.nkv;
  const bool is_v = blockIdx.x & 1;
  int seq = -1, tok0 = 0, off0 = 0, m = 0, pidx = 0;
  for (int base = 0, run = 0; base < a.S; base += 64) {
    int first, keys;
    const int n = rows_of(a, base + lane, first, keys), from = keys - n;
    const int mine = n > 0 ? ((keys - 1) >> a.lp) - (from >> a.lp) + 1 : 0;
    int upto = mine;                                  // pages of the sequences up to this lane's
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int t = __shfl_up(upto, off);
      if (lane >= off) upto += t;
    }
    const uint64_t hit = __ballot(job < run + upto);
    if (hit != 0) {
      const int l = __builtin_ctzll(hit);
      const int before = run + __shfl(upto - mine, l), k = __shfl(keys, l), f = __shfl(from, l), t = __shfl(first, l);
      seq = base + l;
      pidx = (f >> a.lp) + job - before;
      const int lo = max(pidx << a.lp, f), hi = min((pidx + 1) << a.lp, k);
      off0 = lo - (pidx << a.lp);
      m = hi - lo;
      tok0 = t + lo - f;
      break;
    }
    run += __shfl(upto, 63);
  }
  if (seq < 0 || pidx >= a.W) return;
  const int page = a.table[(int64_t)seq * a.W + pidx];
  if ((unsigned)page >= (unsigned)a.pages) return;    // a sequence whose rows are not to be kept
  const int64_t block = (int64_t)page * a.nkv + head;
  const int place0 = (pidx << a.lp) + off0;

  double* y = turn_rows[wave] + sub * LPH * VK_VEC;
  const elem_t* rows = a.qkv + (int64_t)tok0 * a.row_stride + (a.nq + head + (is_v ? a.nkv : 0)) * d + c0;
  double k[VK_VEC];
  float v[VK_VEC];
  auto entries = [&](int i) {                         // this lane's entries of new row i
#pragma unroll
    for (int e = 0; e < VK_VEC; ++e) v[e] = 0.f;
    if (i < m && inside) load_elems(rows + (int64_t)i * a.row_stride, v);
    if (is_v) return;
#pragma unroll
    for (int e = 0; e < VK_VEC; ++e) k[e] = (double)v[e];
    norm_and_turn<LPH>(k, a, a.k_w, c0, place0 + min(i, m - 1), y);
  };
  int need = CACHE8_LOWEST;
  for (int i0 = 0; i0 < m; i0 += 4 * HPW) {
    entries(i0 + wave * HPW + sub);
    if (i0 + wave * HPW + sub < m) {
#pragma unroll
      for (int e = 0; e < VK_VEC; ++e) need = max(need, is_v ? least_exponent(v[e]) : least_exponent(k[e]));
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) need = max(need, __shfl_xor(need, off));
  if (lane == 0) wave_need[wave] = need;
  float* scale = a.scales + block * 2 + (is_v ? 1 : 0);
  const int stood = exponent_of(*scale), old = off0 > 0 ? stood : CACHE8_LOWEST;
  __syncthreads();
  const int now = max(max(old, max(wave_need[0], wave_need[1])), max(wave_need[2], wave_need[3]));

  uint8_t* kp = a.kc + block * P * d;
  uint8_t* vp = a.vc + block * P * d;
  const int ts = P + 4;
  for (int i0 = 0; i0 < m; i0 += 4 * HPW) {
    const int i = i0 + wave * HPW + sub;
    if (m > 4 * HPW) entries(i);                      // else they are still there
    if (i >= m || !inside) continue;
    uint32_t b[VK_VEC / 4];
#pragma unroll
    for (int e = 0; e < VK_VEC; e += 4)
      b[e / 4] = is_v ? to_fp8x4(entry_of(v[e], now), entry_of(v[e + 1], now), entry_of(v[e + 2], now), entry_of(v[e + 3], now))
                      : to_fp8x4(entry_of(k[e], now), entry_of(k[e + 1], now), entry_of(k[e + 2], now), entry_of(k[e + 3], now));
    if (!is_v) {
      uint32_t* to = reinterpret_cast<uint32_t*>(kp + (off0 + i) * d + c0);
#pragma unroll
      for (int e = 0; e < VK_VEC / 4; ++e) to[e] = b[e];
    } else {
#pragma unroll
      for (int e = 0; e < VK_VEC; ++e) {
        const uint8_t one = b[e / 4] >> (8 * (e & 3));
        if (m == 1) vp[(c0 + e) * P + off0] = one;
        else turned[(c0 + e) * ts + off0 + i] = one;
      }
    }
  }
  if (is_v && m > 1) {
    __syncthreads();
    for (int x = threadIdx.x; x < d * (P >> 4); x += STORE8_THREADS) {
      const int c = x / (P >> 4), o = (x % (P >> 4)) << 4;
      if (o + 16 <= off0 || o >= off0 + m) continue;
      const uint8_t* from = turned + c * ts + o;
      if (o >= off0 && o + 16 <= off0 + m) {
        const uint32_t* f = reinterpret_cast<const uint32_t*>(from);
        *reinterpret_cast<u32x4*>(vp + c * P + o) = u32x4{f[0], f[1], f[2], f[3]};
      } else {
        for (int b = max(0, off0 - o); b < min(16, off0 + m - o); ++b) vp[c * P + o + b] = from[b];
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
  Store8Args a{qkv, row_stride, q_out, kc, vc, scales, q_w, k_w, w_is_f32, cos_t, sin_t, rot_half, table, cu_q, k_len, W, T, S, nq, nkv, d, P, 0, pages, 0,
               max_k_len, eps};
  while (1 << a.lp < P) ++a.lp;
  // Pages that n rows of a sequence touch: n at most, and (n - 1) / P + 2.
  a.kv_jobs = nkv > 0 ? (int)min((int64_t)T, (int64_t)T / P + 2 * (int64_t)S) : 0;
  const int64_t blocks = (int64_t)a.kv_jobs * nkv * 2 + (nq > 0 ? T : 0);
  VK_REQUIRE(blocks < (1ll << 31), "qkv_post8: %d rows of %d heads are too many for one launch", T, nq + 2 * nkv);
  const size_t lds = nkv > 0 ? (size_t)d * (P + 4) : 0;
  const int vecs = d / VK_VEC;
#define STORE8(L)                                                                                                                         \
  {                                                                                                                                       \
    if (lds > 48 * 1024) (void)hipFuncSetAttribute((const void*)store8_kernel<L>, hipFuncAttributeMaxDynamicSharedMemorySize, 80 * 1024); \
    store8_kernel<L><<<(unsigned)blocks, STORE8_THREADS, lds, st>>>(a);                                                                   \
  }
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
