// Drafted tokens against the target model's logits, from given random numbers.
//
// Sequence s brings n drafted tokens d_0 .. d_{n-1} and n + 1 rows of the target's logits, row i the one that token i was drafted for, row n the one behind
// them.  With the temperature T of the sequence p_i = softmax(row i / T), and q_i the same of the draft model's row (without such rows the draft is certain: q_i = 1
// at d_i).  A distribution is 1 at the row's maximum (the first of equal ones; a NaN counts as the maximum) where T <= 0 or the maximum is not finite.
//
//   token i stands while u_i q_i(d_i) < p_i(d_i); the first that does not, at a, ends it (a = n: all stand);
//   the token behind the standing ones is drawn from max(p_a - q_a, 0), from p_n if a = n, and from p_a if nothing is left of that: the first j at which the
//   running sum over 0..j exceeds (the sequence's random number) * (the sum over all).
//
// Everything behind the logits is 64-bit.  The drawn token is the one in whose share of the line the number lies, and 150,000 shares stand
// in the line: sums of 32-bit terms would move its borders by some 1e-9 of it each, and one token in some thousand draws would be another one.  The vector unit's
// 64-bit fused multiply-adds are as fast as its 32-bit ones.
//
// Three launches: maximum and sum of pieces of every row; which tokens stand, and what each piece of the row behind them weighs; the piece and the token in it.  Pieces
// have the same borders and their sums the same order whatever else is in the call.
#include "common.h"
#include "sampling.h"

#define VERIFY_THREADS 256
#define VERIFY_PIECE 8192                    // logits a workgroup takes of a row
#define VERIFY_VEC (16 / (int)sizeof(elem_t))
#define VERIFY_ITER (VERIFY_PIECE / VERIFY_VEC / VERIFY_THREADS)

typedef u32x4 __attribute__((aligned(sizeof(elem_t)))) u32x4_any;      // rows of odd length begin anywhere

struct VerifyPart {                          // of a piece of a row: its maximum, where that is first, the sum of exp((x - maximum) / T)
  float top;
  int at;
  double sum;
};
struct VerifyRow {                           // of a row: p(x) = exp((x - top) / T) * scale, or 1 at `at` alone
  double scale;
  float top;
  int at;                                    // -1: no such place
};
struct VerifySeq {                           // what the last launch needs of a sequence
  VerifyRow p, q;
  int row, draft;                            // rows of logits and draft logits (-1: nothing to take away)
  double per_t;
};
struct VerifySums { double left, whole; };   // of a piece: what max(p - q, 0) and p sum to

struct VerifyArgs {
  int32_t *tokens, *counts;
  float* accept;
  const elem_t *logits, *drafts;
  const int32_t *ids, *cu;
  const float *temps, *accept_u, *draw_u;
  VerifyPart* parts;                         // [R + D rows][pieces]
  VerifySums* sums;                          // [S][pieces]
  VerifySeq* seqs;
  int R, D, S, V, pieces;
};

// e^x for x <= 0, 0 below -700 and for NaN: 2^k times the Taylor polynomial of degree 10 on |r| <= ln 2 / 2, which is off by 3e-13 of it.
__device__ __forceinline__ double exp_down(double x) {
  const double k = __builtin_rint(x * 1.4426950408889634);
  const double r = __builtin_fma(-k, 0.6931471805599453, x);
  double p = 1.0 / 3628800;
  p = __builtin_fma(p, r, 1.0 / 362880);
  p = __builtin_fma(p, r, 1.0 / 40320);
  p = __builtin_fma(p, r, 1.0 / 5040);
  p = __builtin_fma(p, r, 1.0 / 720);
  p = __builtin_fma(p, r, 1.0 / 120);
  p = __builtin_fma(p, r, 1.0 / 24);
  p = __builtin_fma(p, r, 1.0 / 6);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  const uint64_t two = (uint64_t)((int)k + 1023) << 52;
  return x > -700.0 ? p * __builtin_bit_cast(double, two) : 0.0;
}

// VERIFY_VEC logits from x[i] on as numbers; those that the row does not have are -infinity.
__device__ __forceinline__ void load_logits(const elem_t* x, int i, int V, float (&out)[VERIFY_VEC]) {
  if (i + VERIFY_VEC <= V) {
    const u32x4 raw = *reinterpret_cast<const u32x4_any*>(x + i);
#pragma unroll
    for (int e = 0; e < VERIFY_VEC; ++e) {
#ifdef VK_BF16
      out[e] = __builtin_bit_cast(float, (e & 1) ? raw[e / 2] & 0xffff0000u : raw[e / 2] << 16);
#else
      out[e] = __builtin_bit_cast(float, (uint32_t)raw[e]);
#endif
    }
  } else {
#pragma unroll
    for (int e = 0; e < VERIFY_VEC; ++e) out[e] = i + e < V ? to_f32(x[i + e]) : -INFINITY;
  }
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = v + __shfl_xor(v, off);
  return v;
}
__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = min(v, __shfl_xor(v, off));
  return v;
}

// Of sequence `base + lane`: its first row, its first drafted token (the sequences before it, without their last rows) and how many it has; -1: no
// sequence, one without rows, or one that the arrays do not hold.  `seen`: sequences with rows before `base`, and then before base + 64.
__device__ __forceinline__ int drafts_of(const VerifyArgs& a, int base, int& first, int& draft, int& seen) {
  const int i = base + (threadIdx.x & 63);
  first = i < a.S ? a.cu[i] : 0;
  const int rows = i < a.S ? a.cu[i + 1] - first : 0;
  const uint64_t some = __ballot(rows > 0);
  draft = first - seen - __builtin_popcountll(some & ((1ull << (threadIdx.x & 63)) - 1));
  seen += __builtin_popcountll(some);
  return rows > 0 && first >= 0 && first + rows <= a.R && draft >= 0 && draft + rows - 1 <= a.D ? rows - 1 : -1;
}
__device__ __forceinline__ double per_temperature(const VerifyArgs& a, int seq) {        // 0: the maximum alone
  const float t = a.temps != nullptr ? a.temps[seq] : 0.f;
  return t > 0.f ? fmax(1.0 / (double)t, 1e-300) : 0.0;                                // an infinite one: every finite logit weighs the same
}
__device__ __forceinline__ bool is_finite(float x) { return (__builtin_bit_cast(uint32_t, x) >> 23 & 255) != 255; }

__global__ __launch_bounds__(VERIFY_THREADS) void verify_parts_kernel(VerifyArgs a) {
  __shared__ float s_top[4];
  __shared__ int s_at[4], s_nan[4];
  __shared__ double s_sum[4];
  const int row = blockIdx.x, piece = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool drafted = row >= a.R;
  int seq = -1;
  for (int base = 0, seen = 0; base < a.S && seq < 0; base += 64) {
    int first, draft;
    const int n = drafts_of(a, base, first, draft, seen), from = drafted ? a.R + draft : first;
    const uint64_t mine = __ballot(n >= 0 && row >= from && row < from + n + (drafted ? 0 : 1));
    if (mine != 0) seq = base + __builtin_ctzll(mine);
  }
  if (seq < 0) return;
  const double per_t = per_temperature(a, seq);
  const elem_t* x = drafted ? a.drafts + (int64_t)(row - a.R) * a.V : a.logits + (int64_t)row * a.V;
  float v[VERIFY_ITER][VERIFY_VEC];
  float top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < VERIFY_ITER; ++i) load_logits(x, piece * VERIFY_PIECE + (i * VERIFY_THREADS + tid) * VERIFY_VEC, a.V, v[i]);
#pragma unroll
  for (int i = 0; i < VERIFY_ITER; ++i)
#pragma unroll
    for (int e = 0; e < VERIFY_VEC; ++e) {
      top = fmaxf(top, v[i][e]);
      nan = nan || v[i][e] != v[i][e];
    }
  top = wave_max_xor(top);
  if (lane == 0) s_top[wave] = top;
  if (lane == 0) s_nan[wave] = 0;
  if (__any(nan) && lane == 0) s_nan[wave] = 1;
  __syncthreads();
  top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
  nan = (s_nan[0] | s_nan[1] | s_nan[2] | s_nan[3]) != 0;
  int at = 0x7fffffff;
  double sum = 0.0;
  const bool sums = per_t > 0.0 && !nan && is_finite(top);
#pragma unroll
  for (int i = 0; i < VERIFY_ITER; ++i)
#pragma unroll
    for (int e = 0; e < VERIFY_VEC; ++e) {
      const int j = piece * VERIFY_PIECE + (i * VERIFY_THREADS + tid) * VERIFY_VEC + e;
      if (j < a.V && (nan ? v[i][e] != v[i][e] : v[i][e] == top)) at = min(at, j);
      if (sums) sum = sum + exp_down(((double)v[i][e] - (double)top) * per_t);
    }
  at = wave_min_i(at);
  sum = wave_sum_d(sum);
  if (lane == 0) {
    s_at[wave] = at;
    s_sum[wave] = sum;
  }
  __syncthreads();
  if (tid == 0)
    a.parts[(int64_t)row * a.pieces + piece] =
        VerifyPart{nan ? NAN : top, min(min(s_at[0], s_at[1]), min(s_at[2], s_at[3])), (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3])};
}

// A row's distribution from its pieces, by a whole wave.
__device__ __forceinline__ VerifyRow join_row(const VerifyArgs& a, int row, double per_t) {
  const int lane = threadIdx.x & 63;
  const VerifyPart* parts = a.parts + (int64_t)row * a.pieces;
  float top = -INFINITY;
  bool nan = false;
  for (int c = lane; c < a.pieces; c += 64) {
    top = fmaxf(top, parts[c].top);
    nan = nan || parts[c].top != parts[c].top;
  }
  top = wave_max_xor(top);
  nan = __any(nan);
  if (per_t > 0.0 && !nan && is_finite(top)) {
    double sum = 0.0;
    for (int c = lane; c < a.pieces; c += 64) sum = sum + parts[c].sum * exp_down(((double)parts[c].top - (double)top) * per_t);
    return VerifyRow{1.0 / wave_sum_d(sum), top, -1};
  }
  int at = 0x7fffffff;
  for (int c = lane; c < a.pieces; c += 64)
    if (nan ? parts[c].top != parts[c].top : parts[c].top == top) at = min(at, parts[c].at);
  return VerifyRow{0.0, top, wave_min_i(at)};
}
__device__ __forceinline__ double chance(const VerifyRow& r, int j, float x, double per_t) {
  return r.at >= 0 ? (j == r.at ? 1.0 : 0.0) : exp_down(((double)x - (double)r.top) * per_t) * r.scale;
}

// p and max(p - q, 0) of the logits from j on.
__device__ __forceinline__ void weights_of(const VerifyArgs& a, const VerifySeq& s, int j, double (&whole)[VERIFY_VEC], double (&left)[VERIFY_VEC]) {
  float x[VERIFY_VEC], y[VERIFY_VEC];
  load_logits(a.logits + (int64_t)s.row * a.V, j, a.V, x);
  if (s.draft >= 0 && s.q.at < 0) load_logits(a.drafts + (int64_t)s.draft * a.V, j, a.V, y);
#pragma unroll
  for (int e = 0; e < VERIFY_VEC; ++e) {
    const double p = exp_down(((double)x[e] - (double)s.p.top) * s.per_t) * s.p.scale;
    const double q = s.draft < 0 ? 0.0 : s.q.at >= 0 ? (j + e == s.q.at ? 1.0 : 0.0) : exp_down(((double)y[e] - (double)s.q.top) * s.per_t) * s.q.scale;
    whole[e] = p;
    left[e] = fmax(p - q, 0.0);
  }
}

__global__ __launch_bounds__(VERIFY_THREADS) void verify_weigh_kernel(VerifyArgs a) {
  __shared__ int s_first;
  __shared__ double s_left[4], s_whole[4];
  const int seq = blockIdx.x, piece = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int n = -1, row0 = 0, draft0 = 0;
  for (int base = 0, seen = 0; base <= seq; base += 64) {
    const int mine = drafts_of(a, base, row0, draft0, seen);
    if (seq < base + 64) {
      n = __shfl(mine, seq - base);
      row0 = __shfl(row0, seq - base);
      draft0 = __shfl(draft0, seq - base);
    }
  }
  if (n < 0) {
    if (piece == 0 && tid == 0) {
      a.counts[seq] = 0;
      a.seqs[seq].row = -1;
    }
    return;
  }
  const double per_t = per_temperature(a, seq);
  if (tid == 0) s_first = n;
  __syncthreads();
  for (int i = wave; i < n; i += 4) {
    const int id = a.ids[draft0 + i];
    const bool known = (unsigned)id < (unsigned)a.V;
    const VerifyRow p = join_row(a, row0 + i, per_t);
    double pd = 0.0, qd = 0.0;
    if (known) pd = chance(p, id, to_f32(a.logits[(int64_t)(row0 + i) * a.V + id]), per_t);
    if (a.drafts != nullptr) {
      const VerifyRow q = join_row(a, a.R + draft0 + i, per_t);
      if (known) qd = chance(q, id, to_f32(a.drafts[(int64_t)(draft0 + i) * a.V + id]), per_t);
    } else if (known) {
      qd = 1.0;
    }
    const double u = a.accept_u != nullptr ? (double)a.accept_u[draft0 + i] : 0.0;
    if (lane == 0) {
      if (!(u * qd < pd)) atomicMin(&s_first, i);
      if (piece == 0) a.accept[draft0 + i] = (float)(qd > 0.0 ? fmin(1.0, pd / qd) : pd > 0.0 ? 1.0 : 0.0);
    }
  }
  __syncthreads();
  const int stand = s_first;
  VerifySeq s;
  s.row = row0 + stand;
  s.draft = stand < n ? draft0 + stand : -1;
  s.per_t = per_t;
  s.p = join_row(a, s.row, per_t);
  s.q = VerifyRow{0.0, 0.f, -1};
  if (stand < n) {
    if (a.drafts != nullptr) s.q = join_row(a, a.R + s.draft, per_t);
    else s.q.at = (unsigned)a.ids[s.draft] < (unsigned)a.V ? a.ids[s.draft] : 0x7fffffff;
  }
  if (piece == 0) {
    for (int i = tid; i <= n; i += VERIFY_THREADS)
      if (i != stand) a.tokens[row0 + i] = i < stand ? a.ids[draft0 + i] : -1;
    if (tid == 0) {
      a.counts[seq] = stand + 1;
      a.seqs[seq] = s;
      if (s.p.at >= 0) a.tokens[s.row] = s.p.at;         // 1 there: whatever is taken away, it is what is left, or nothing is
    }
  }
  if (s.p.at >= 0) return;
  double left = 0.0, whole = 0.0;
#pragma unroll
  for (int i = 0; i < VERIFY_ITER; ++i) {
    const int j = piece * VERIFY_PIECE + (i * VERIFY_THREADS + tid) * VERIFY_VEC;
    if (j >= a.V) break;
    double w[VERIFY_VEC], l[VERIFY_VEC];
    weights_of(a, s, j, w, l);
#pragma unroll
    for (int e = 0; e < VERIFY_VEC; ++e) {
      whole = whole + w[e];
      left = left + l[e];
    }
  }
  left = wave_sum_d(left);
  whole = wave_sum_d(whole);
  if (lane == 0) {
    s_left[wave] = left;
    s_whole[wave] = whole;
  }
  __syncthreads();
  if (tid == 0) a.sums[(int64_t)seq * a.pieces + piece] = VerifySums{(s_left[0] + s_left[1]) + (s_left[2] + s_left[3]), (s_whole[0] + s_whole[1]) + (s_whole[2] + s_whole[3])};
}

__global__ __launch_bounds__(VERIFY_THREADS) void verify_draw_kernel(VerifyArgs a) {
  __shared__ double s_wave[4];
  __shared__ int s_last[4], s_pick;
  const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const VerifySeq s = a.seqs[seq];
  if (s.row < 0 || s.p.at >= 0) return;
  const VerifySums* sums = a.sums + (int64_t)seq * a.pieces;
  double all = 0.0, all_whole = 0.0;
  for (int c = 0; c < a.pieces; ++c) {
    all = all + sums[c].left;
    all_whole = all_whole + sums[c].whole;
  }
  const bool use_left = all > 0.0;
  const double target = (double)a.draw_u[seq] * (use_left ? all : all_whole);
  // The piece: the first whose end lies beyond the target, else (the target is the end, by rounding) the last that weighs anything.
  int piece = -1, last = 0;
  double before = 0.0, run = 0.0, last_before = 0.0;
  for (int c = 0; c < a.pieces; ++c) {
    const double w = use_left ? sums[c].left : sums[c].whole;
    if (w > 0.0) {
      last = c;
      last_before = run;
    }
    if (piece < 0 && target < run + w) {
      piece = c;
      before = run;
    }
    run = run + w;
  }
  if (piece < 0) {
    piece = last;
    before = last_before;
  }
  // The token in it: a thread has as many neighbouring logits as it has vectors of them.
  double w[VERIFY_ITER][VERIFY_VEC];
  double sum = 0.0;
  const int j0 = piece * VERIFY_PIECE + tid * VERIFY_ITER * VERIFY_VEC;
  int my_last = -1;
#pragma unroll
  for (int i = 0; i < VERIFY_ITER; ++i) {
    double whole[VERIFY_VEC], left[VERIFY_VEC];
    weights_of(a, s, j0 + i * VERIFY_VEC, whole, left);
#pragma unroll
    for (int e = 0; e < VERIFY_VEC; ++e) {
      w[i][e] = use_left ? left[e] : whole[e];
      sum = sum + w[i][e];
      if (w[i][e] > 0.0) my_last = j0 + i * VERIFY_VEC + e;
    }
  }
  double upto = sum;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double t = __shfl_up(upto, off);
    if (lane >= off) upto = upto + t;
  }
  if (lane == 63) s_wave[wave] = upto;
  my_last = -wave_min_i(-my_last);
  if (lane == 0) s_last[wave] = my_last;
  if (tid == 0) s_pick = 0x7fffffff;
  __syncthreads();
  double start = before;
  for (int i = 0; i < wave; ++i) start = start + s_wave[i];
  start = start + (upto - sum);
  int pick = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < VERIFY_ITER; ++i)
#pragma unroll
    for (int e = 0; e < VERIFY_VEC; ++e) {
      start = start + w[i][e];
      if (w[i][e] > 0.0 && target < start) pick = min(pick, j0 + i * VERIFY_VEC + e);
    }
  if (pick != 0x7fffffff) atomicMin(&s_pick, pick);
  __syncthreads();
  if (tid == 0) a.tokens[s.row] = s_pick != 0x7fffffff ? s_pick : max(max(max(s_last[0], s_last[1]), max(s_last[2], s_last[3])), 0);
}

extern "C" {

static int64_t verify_pieces(int V) { return ((int64_t)V + VERIFY_PIECE - 1) / VERIFY_PIECE; }

int64_t vk_verify_scratch_bytes(int R, int D, int S, int V) {
  return verify_pieces(V) * (((int64_t)R + D) * (int64_t)sizeof(VerifyPart) + S * (int64_t)sizeof(VerifySums)) + S * (int64_t)sizeof(VerifySeq);
}

int vk_verify(int32_t* tokens, int32_t* counts, float* accept, const elem_t* logits, const int32_t* ids, const int32_t* cu, const elem_t* draft_logits,
              const float* temps, const float* accept_u, const float* draw_u, void* scratch, int64_t scratch_bytes, int R, int D, int S, int V, hipStream_t st) {
  VK_REQUIRE(R >= 0 && D >= 0 && S >= 0 && V > 0 && V < (1 << 30), "verify: bad sizes R=%d D=%d S=%d V=%d", R, D, S, V);
  VK_REQUIRE(temps == nullptr || (draw_u != nullptr && (accept_u != nullptr || D == 0)), "verify: temperatures need random numbers");
  if (S == 0) return 0;
  VK_REQUIRE(tokens != nullptr && counts != nullptr && logits != nullptr && cu != nullptr && (D == 0 || (ids != nullptr && accept != nullptr)), "verify: an array is missing");
  VK_REQUIRE(scratch != nullptr && (uintptr_t)scratch % 16 == 0 && scratch_bytes >= vk_verify_scratch_bytes(R, D, S, V), "verify: %lld bytes of scratch needed, on 16 bytes",
             (long long)vk_verify_scratch_bytes(R, D, S, V));
  const int pieces = (int)verify_pieces(V);
  VK_REQUIRE(pieces <= 65535, "verify: a vocabulary of %d is too large", V);
  VerifyArgs a{tokens, counts, accept, logits, draft_logits, ids, cu, temps, accept_u, draw_u, static_cast<VerifyPart*>(scratch), nullptr, nullptr, R, D, S, V, pieces};
  a.sums = reinterpret_cast<VerifySums*>(a.parts + ((int64_t)R + D) * pieces);
  a.seqs = reinterpret_cast<VerifySeq*>(a.sums + (int64_t)S * pieces);
  const int64_t rows = (int64_t)R + (draft_logits != nullptr ? D : 0);
  VK_REQUIRE(rows < (1ll << 31), "verify: %lld rows are too many", (long long)rows);
  if (rows > 0) {
    verify_parts_kernel<<<dim3((unsigned)rows, pieces), VERIFY_THREADS, 0, st>>>(a);
    if (vk_check_launch("verify (parts)")) return 1;
  }
  verify_weigh_kernel<<<dim3(S, pieces), VERIFY_THREADS, 0, st>>>(a);
  if (vk_check_launch("verify (weigh)")) return 1;
  verify_draw_kernel<<<S, VERIFY_THREADS, 0, st>>>(a);
  return vk_check_launch("verify (draw)");
}

}  // extern "C"
