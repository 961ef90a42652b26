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
// in the line: sums of 32-bit terms would move its borders by some 1e-9 of it each, and one token in some thousand draws would be another one; the exponentials' 1e-12 moves one in ten million.  The vector unit's
// 64-bit fused multiply-adds are as fast as its 32-bit ones.
//
// Measured (MI355X, bfloat16 logits of 151,936, four drafted tokens): 64 sequences, 175 MB: 67 us for maximum and sum (its bytes take 27; seventeen 64-bit operations an exponential 38, beside the
// search for the maximum), 8 to decide, 19 for the pieces, 8 to draw.  One sequence, its token drawn: 4.8, 7.3 and 6.6 us, launches and loads that wait for each other.
//
// Four launches: maximum and sum of pieces of every row, a wave each; which tokens stand, and the distributions behind them; what the pieces of those weigh; the piece and
// the token in it (the second and third as one where there are few pieces).  Pieces have the same borders and their sums the same order whatever else is in the call.
#include "common.h"
#include "sampling.h"

#define VERIFY_THREADS 256
#define VERIFY_PIECE 2048                    // logits a wave takes of a row
#define VERIFY_VEC (16 / (int)sizeof(elem_t))
#define VERIFY_ITER (VERIFY_PIECE / VERIFY_VEC / 64)

typedef u32x4 __attribute__((aligned(sizeof(elem_t)))) u32x4_any;      // rows of odd length begin anywhere

struct VerifyPart {                          // of a piece of a row: its maximum, the sum of exp((x - maximum) / T), or else where the maximum is first
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

// 2^t for t <= 0, and 0 for NaN: 2^k, k the nearest whole number, times the polynomial of degree 8 that meets 2^f at the nine Chebyshev points of |f| <= 1/2; it is off by
// 1.1e-12 of it.  k is what the addition of 1.5 * 2^52 leaves in the last bits.
#define VERIFY_LOG2E 1.4426950408889634
// The polynomial is written out: its constants stay in scalar registers, where the compiler's own form adds onto a copy that it makes for every addition, two moves of it (576 rows of 151,936
// logits: 103 -> 87 us, together with a row's loads all in front of its sums), and stands in one piece, where steps written out singly have a pause between them (one sequence 18.9 -> 18.0 us in all).
__device__ __forceinline__ double exp2_down(double t) {
  const double big = 6755399441055744.0, low = fmax(t, -2000.0), sum = low + big, f = low - (sum - big);
  double p;
  asm("v_fma_f64 %0, %1, %2, %3\n\tv_fma_f64 %0, %0, %1, %4\n\tv_fma_f64 %0, %0, %1, %5\n\tv_fma_f64 %0, %0, %1, %6\n\t"
      "v_fma_f64 %0, %0, %1, %7\n\tv_fma_f64 %0, %0, %1, %8\n\tv_fma_f64 %0, %0, %1, %9\n\tv_fma_f64 %0, %0, %1, 1.0"
      : "=&v"(p)
      : "v"(f), "v"(1.3255224887698904e-06), "s"(1.5310079402479794e-05), "s"(0.00015403455852411408), "s"(0.0013333450567999659), "s"(0.00961812915940262), "s"(0.05550410941205934),
        "s"(0.2402265069581299), "s"(0.6931471805459335));
  return __builtin_ldexp(p, (int)(uint32_t)__builtin_bit_cast(uint64_t, sum));
}

// The vector of logits from x[j] on; where the row ends inside it, its last whole vector (from `at` on, below j), so that a vector is one load anywhere.  Rows shorter than a vector are read one
// by one.
struct VerifyVec {
  u32x4 raw;
  int at;
};
__device__ __forceinline__ VerifyVec load_vec(const elem_t* x, int j, int V) {
  VerifyVec v;
  if (V >= VERIFY_VEC) {
    v.at = min(j, V - VERIFY_VEC);
    v.raw = *reinterpret_cast<const u32x4_any*>(x + v.at);
  } else {
    v.at = j;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#ifdef VK_BF16
      const uint32_t lo = j + 2 * e < V ? __builtin_bit_cast(uint16_t, x[j + 2 * e]) : 0xff80u, hi = j + 2 * e + 1 < V ? __builtin_bit_cast(uint16_t, x[j + 2 * e + 1]) : 0xff80u;
      v.raw[e] = lo | hi << 16;
#else
      v.raw[e] = j + e < V ? __builtin_bit_cast(uint32_t, x[j + e]) : 0xff800000u;
#endif
    }
  }
  return v;
}
// A row's last piece: elements of v that lie before j, in another vector, become -infinity.
__device__ __forceinline__ void only_own(VerifyVec& v, int j) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
#ifdef VK_BF16
    const uint32_t lo = v.at + 2 * e >= j ? v.raw[e] & 0xffffu : 0xff80u, hi = v.at + 2 * e + 1 >= j ? v.raw[e] & 0xffff0000u : 0xff800000u;
    v.raw[e] = lo | hi;
#else
    v.raw[e] = v.at + e >= j ? v.raw[e] : 0xff800000u;
#endif
  }
}
// Its numbers: element e is the logit v.at + e.
__device__ __forceinline__ float number_of(const VerifyVec& v, int e) {
#ifdef VK_BF16
  return __builtin_bit_cast(float, (e & 1) ? v.raw[e / 2] & 0xffff0000u : v.raw[e / 2] << 16);
#else
  return __builtin_bit_cast(float, (uint32_t)v.raw[e]);
#endif
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
  const int end = i < a.S ? a.cu[i + 1] : 0, rows = first >= 0 && first < end && end <= a.R ? end - first : 0;
  const uint64_t some = __ballot(rows > 0);
  draft = first - seen - __builtin_popcountll(some & ((1ull << (threadIdx.x & 63)) - 1));
  seen += __builtin_popcountll(some);
  return rows > 0 && draft >= 0 && draft + rows - 1 <= a.D ? rows - 1 : -1;
}
__device__ __forceinline__ double per_temperature(const VerifyArgs& a, int seq) {        // log2(e) / T; 0: the maximum alone
  const float t = a.temps != nullptr ? a.temps[seq] : 0.f;
  return t > 0.f ? fmax(VERIFY_LOG2E / (double)t, 1e-300) : 0.0;                       // an infinite one: every finite logit weighs the same
}
__device__ __forceinline__ bool is_finite(float x) { return (__builtin_bit_cast(uint32_t, x) >> 23 & 255) != 255; }

__global__ __launch_bounds__(VERIFY_THREADS) void verify_parts_kernel(VerifyArgs a) {
  const int row = blockIdx.x, lane = threadIdx.x & 63, piece = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (piece >= a.pieces) return;
  const bool drafted = row >= a.R;
  const elem_t* x = drafted ? a.drafts + (int64_t)(row - a.R) * a.V : a.logits + (int64_t)row * a.V;
  const int j0 = piece * VERIFY_PIECE + lane * VERIFY_VEC;
  VerifyVec raw[VERIFY_ITER];
#pragma unroll
  for (int i = 0; i < VERIFY_ITER; ++i) raw[i] = load_vec(x, j0 + i * 64 * VERIFY_VEC, a.V);
  int seq = -1;
  for (int base = 0, seen = 0; base < a.S && seq < 0; base += 64) {
    int first, draft;
    const int n = drafts_of(a, base, first, draft, seen), from = drafted ? a.R + draft : first;
    const uint64_t mine = __ballot(n >= 0 && row >= from && row < from + n + (drafted ? 0 : 1));
    if (mine != 0) seq = base + __builtin_ctzll(mine);
  }
  if (seq < 0) return;
  const double per_t = per_temperature(a, seq);
  if ((piece + 1) * VERIFY_PIECE > a.V) {
#pragma unroll
    for (int i = 0; i < VERIFY_ITER; ++i) only_own(raw[i], j0 + i * 64 * VERIFY_VEC);
  }
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < VERIFY_ITER; ++i)
#pragma unroll
    for (int e = 0; e < VERIFY_VEC; ++e) top = __builtin_elementwise_maximum(top, number_of(raw[i], e));       // NaN where there is one
  const bool nan = __any(top != top);
  top = wave_max_xor(top);
  int at = 0x7fffffff;
  double sum = 0.0;
  // Where a piece's maximum is not finite the row's is not, or comes from another piece.
  if (per_t > 0.0 && !nan && is_finite(top)) {
#pragma unroll
    for (int i = 0; i < VERIFY_ITER; ++i)
#pragma unroll
      for (int e = 0; e < VERIFY_VEC; ++e) sum = sum + exp2_down(((double)number_of(raw[i], e) - (double)top) * per_t);
    sum = wave_sum_xor(sum);
  } else {
#pragma unroll
    for (int i = 0; i < VERIFY_ITER; ++i)
#pragma unroll
      for (int e = 0; e < VERIFY_VEC; ++e) {
        const float v = number_of(raw[i], e);
        const int from = j0 + i * 64 * VERIFY_VEC, j = raw[i].at + e;
        if (j >= from && j < a.V && (nan ? v != v : v == top)) at = min(at, j);
      }
    at = wave_min_i(at);
  }
  if (lane == 0) a.parts[(int64_t)row * a.pieces + piece] = VerifyPart{nan ? NAN : top, at, sum};
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
    for (int c = lane; c < a.pieces; c += 64) sum = sum + parts[c].sum * exp2_down(((double)parts[c].top - (double)top) * per_t);
    return VerifyRow{1.0 / wave_sum_xor(sum), top, -1};
  }
  int at = 0x7fffffff;
  for (int c = lane; c < a.pieces; c += 64)
    if (nan ? parts[c].top != parts[c].top : parts[c].top == top) at = min(at, parts[c].at);
  return VerifyRow{0.0, top, wave_min_i(at)};
}
__device__ __forceinline__ double chance(const VerifyRow& r, int j, float x, double per_t) {
  return r.at >= 0 ? (j == r.at ? 1.0 : 0.0) : exp2_down(((double)x - (double)r.top) * per_t) * r.scale;
}

// p and max(p - q, 0) of N vectors of logits, the i-th from j[i] on; at[i]: the logit that its first element is (those before j[i] weigh nothing).  edge: the row's last piece.
template <int N>
__device__ __forceinline__ void weights_of(const VerifyArgs& a, const VerifySeq& s, bool edge, const int (&j)[N], int (&at)[N], double (&whole)[N][VERIFY_VEC], double (&left)[N][VERIFY_VEC]) {
  const bool drawn = s.draft >= 0 && s.q.at < 0;
  VerifyVec vx[N], vy[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    vx[i] = load_vec(a.logits + (int64_t)s.row * a.V, j[i], a.V);
    at[i] = vx[i].at;
  }
  if (drawn) {
#pragma unroll
    for (int i = 0; i < N; ++i) vy[i] = load_vec(a.drafts + (int64_t)s.draft * a.V, j[i], a.V);
  }
  if (edge) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      only_own(vx[i], j[i]);
      if (drawn) only_own(vy[i], j[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < VERIFY_VEC; ++e) whole[i][e] = exp2_down(((double)number_of(vx[i], e) - (double)s.p.top) * s.per_t) * s.p.scale;
  if (drawn) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < VERIFY_VEC; ++e) left[i][e] = fmax(whole[i][e] - exp2_down(((double)number_of(vy[i], e) - (double)s.q.top) * s.per_t) * s.q.scale, 0.0);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < VERIFY_VEC; ++e) left[i][e] = s.draft >= 0 && at[i] + e == s.q.at ? 0.0 : whole[i][e];        // q is 1 there, and p at most
  }
}

// Which of a sequence's tokens stand, and what stands behind them: by a workgroup, a wave every fourth row.  write: tokens, counts and chances too.
#define VERIFY_KEPT 16                       // rows whose distributions stay in LDS until it is known which one is needed
__device__ __forceinline__ VerifySeq decide(const VerifyArgs& a, int seq, bool write) {
  __shared__ int s_first;
  __shared__ VerifyRow s_p[VERIFY_KEPT], s_q[VERIFY_KEPT];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  VerifySeq s;
  s.row = -1;
  s.draft = -1;
  s.per_t = per_temperature(a, seq);
  s.p = s.q = VerifyRow{0.0, 0.f, -1};
  int n = -1, row0 = 0, draft0 = 0;
  for (int base = 0, seen = 0; base <= seq; base += 64) {
    const int mine = drafts_of(a, base, row0, draft0, seen);
    if (seq < base + 64) {
      n = __builtin_amdgcn_readlane(mine, seq - base);
      row0 = __builtin_amdgcn_readlane(row0, seq - base);
      draft0 = __builtin_amdgcn_readlane(draft0, seq - base);
    }
  }
  if (tid == 0) s_first = n;
  if (n < 0) {
    if (write && tid == 0) a.counts[seq] = 0;
    return s;
  }
  __syncthreads();
  for (int i = wave; i <= n; i += 4) {
    int id = -1;
    float x = 0.f, y = 0.f, u = 0.f;
    if (i < n) {
      id = a.ids[draft0 + i];
      if (a.accept_u != nullptr) u = a.accept_u[draft0 + i];
    }
    const bool known = (unsigned)id < (unsigned)a.V;
    if (known) {
      x = to_f32(a.logits[(int64_t)(row0 + i) * a.V + id]);
      if (a.drafts != nullptr) y = to_f32(a.drafts[(int64_t)(draft0 + i) * a.V + id]);
    }
    const VerifyRow p = join_row(a, row0 + i, s.per_t);
    VerifyRow q{0.0, 0.f, known ? id : 0x7fffffff};
    if (a.drafts != nullptr && i < n) q = join_row(a, a.R + draft0 + i, s.per_t);
    if (lane != 0) continue;
    if (i < VERIFY_KEPT) {
      s_p[i] = p;
      s_q[i] = q;
    }
    if (i == n) continue;
    const double pd = known ? chance(p, id, x, s.per_t) : 0.0, qd = known ? chance(q, id, y, s.per_t) : 0.0;
    if (!((double)u * qd < pd)) atomicMin(&s_first, i);
    if (write) a.accept[draft0 + i] = (float)(qd > 0.0 ? fmin(1.0, pd / qd) : pd > 0.0 ? 1.0 : 0.0);
  }
  __syncthreads();
  const int stand = s_first;
  s.row = row0 + stand;
  s.draft = stand < n ? draft0 + stand : -1;
  if (stand < VERIFY_KEPT) {
    s.p = s_p[stand];
    s.q = s_q[stand];
  } else {
    s.p = join_row(a, s.row, s.per_t);
    if (stand < n) {
      if (a.drafts != nullptr) s.q = join_row(a, a.R + s.draft, s.per_t);
      else s.q.at = (unsigned)a.ids[s.draft] < (unsigned)a.V ? a.ids[s.draft] : 0x7fffffff;
    }
  }
  if (write) {
    for (int i = tid; i <= n; i += VERIFY_THREADS)
      if (i != stand) a.tokens[row0 + i] = i < stand ? a.ids[draft0 + i] : -1;
    if (tid == 0) {
      a.counts[seq] = stand + 1;
      if (s.p.at >= 0) a.tokens[s.row] = s.p.at;         // 1 there: whatever is taken away, it is what is left, or nothing is
    }
  }
  return s;
}

__global__ __launch_bounds__(VERIFY_THREADS) void verify_decide_kernel(VerifyArgs a) {
  const VerifySeq s = decide(a, blockIdx.x, true);
  if (threadIdx.x == 0) a.seqs[blockIdx.x] = s;
}

// A piece is summed in four parts, (0 + 1) + (2 + 3).  DECIDE: every workgroup decides for itself, in place of a launch of its own, and has one piece, a part a wave; else a wave has a
// piece.
template <bool DECIDE>
__global__ __launch_bounds__(VERIFY_THREADS) void verify_weigh_kernel(VerifyArgs a) {
  __shared__ VerifySums s_part[4];
  const int seq = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), piece = DECIDE ? blockIdx.y : blockIdx.y * 4 + wave;
  VerifySeq s;
  if (DECIDE) {
    s = decide(a, seq, blockIdx.y == 0);
    if (blockIdx.y == 0 && threadIdx.x == 0) a.seqs[seq] = s;
  } else {
    s = a.seqs[seq];
  }
  if (piece >= a.pieces || s.row < 0 || s.p.at >= 0) return;
  constexpr int PART = VERIFY_ITER / 4;
  auto part = [&](int h) {
    double w[PART][VERIFY_VEC], l[PART][VERIFY_VEC], left = 0.0, whole = 0.0;
    int j[PART], at[PART];
#pragma unroll
    for (int i = 0; i < PART; ++i) j[i] = piece * VERIFY_PIECE + ((h * PART + i) * 64 + lane) * VERIFY_VEC;
    weights_of<PART>(a, s, (piece + 1) * VERIFY_PIECE > a.V, j, at, w, l);
#pragma unroll
    for (int i = 0; i < PART; ++i)
#pragma unroll
      for (int e = 0; e < VERIFY_VEC; ++e) {
        whole = whole + w[i][e];
        left = left + l[i][e];
      }
    return VerifySums{wave_sum_xor(left), wave_sum_xor(whole)};
  };
  VerifySums x[4];
  if (DECIDE) {
    const VerifySums mine = part(wave);
    if (lane == 0) s_part[wave] = mine;
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 4; ++h) x[h] = s_part[h];
  } else {
#pragma unroll
    for (int h = 0; h < 4; ++h) x[h] = part(h);
  }
  if (lane == 0 && (!DECIDE || wave == 0))
    a.sums[(int64_t)seq * a.pieces + piece] = VerifySums{(x[0].left + x[1].left) + (x[2].left + x[3].left), (x[0].whole + x[1].whole) + (x[2].whole + x[3].whole)};
}

__global__ __launch_bounds__(VERIFY_THREADS) void verify_draw_kernel(VerifyArgs a) {
  constexpr int PER = VERIFY_PIECE / VERIFY_VEC / VERIFY_THREADS;      // vectors a thread
  __shared__ double s_wave[4];
  __shared__ int s_last[4], s_pick;
  const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const VerifySeq s = a.seqs[seq];
  if (s.row < 0 || s.p.at >= 0) return;
  // A lane a piece, 64 at a time: running sums over them, the first that ends beyond the target, else (the target is the end, by rounding) the last that weighs
  // anything.  Every wave for itself.
  const VerifySums* sums = a.sums + (int64_t)seq * a.pieces;
  double all = 0.0, all_whole = 0.0;
  for (int c0 = 0; c0 < a.pieces; c0 += 64) {
    const VerifySums mine = c0 + lane < a.pieces ? sums[c0 + lane] : VerifySums{0.0, 0.0};
    all = all + wave_sum_xor(mine.left);
    all_whole = all_whole + wave_sum_xor(mine.whole);
  }
  const bool use_left = all > 0.0;
  const double target = (double)a.draw_u[seq] * (use_left ? all : all_whole);
  int piece = -1, last = 0;
  double before = 0.0, run = 0.0, last_before = 0.0;
  for (int c0 = 0; c0 < a.pieces && piece < 0; c0 += 64) {
    const VerifySums mine = c0 + lane < a.pieces ? sums[c0 + lane] : VerifySums{0.0, 0.0};
    const double w = use_left ? mine.left : mine.whole;
    double upto = w;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const double t = __shfl_up(upto, off);
      if (lane >= off) upto = upto + t;
    }
    const double begin = run + (upto - w);
    const uint64_t beyond = __ballot(w > 0.0 && target < run + upto), some = __ballot(w > 0.0);
    if (beyond != 0) {
      const int l = __builtin_ctzll(beyond);
      piece = c0 + l;
      before = __shfl(begin, l);
    }
    if (some != 0) {
      const int l = 63 - __builtin_clzll(some);
      last = c0 + l;
      last_before = __shfl(begin, l);
    }
    run = run + __shfl(upto, 63);
  }
  if (piece < 0) {
    piece = last;
    before = last_before;
  }
  // The token in it: a thread has as many neighbouring logits as it has vectors of them.
  double w[PER][VERIFY_VEC], l[PER][VERIFY_VEC], sum = 0.0;
  int j[PER], at[PER], my_last = -1;
#pragma unroll
  for (int i = 0; i < PER; ++i) j[i] = piece * VERIFY_PIECE + (tid * PER + i) * VERIFY_VEC;
  weights_of<PER>(a, s, (piece + 1) * VERIFY_PIECE > a.V, j, at, w, l);
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int e = 0; e < VERIFY_VEC; ++e) {
      w[i][e] = use_left ? l[i][e] : w[i][e];
      sum = sum + w[i][e];
      if (w[i][e] > 0.0) my_last = at[i] + e;
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
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int e = 0; e < VERIFY_VEC; ++e) {
      start = start + w[i][e];
      if (w[i][e] > 0.0 && target < start) pick = min(pick, at[i] + e);
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
  VK_REQUIRE(counts != nullptr && cu != nullptr && (R == 0 || (tokens != nullptr && logits != nullptr)) && (D == 0 || (ids != nullptr && accept != nullptr)), "verify: an array is missing");
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
    verify_parts_kernel<<<dim3((unsigned)rows, (pieces + 3) / 4), VERIFY_THREADS, 0, st>>>(a);
    if (vk_check_launch("verify (parts)")) return 1;
  }
  // Where the next launch's workgroups, a piece each, are not many rounds of the card they decide for themselves, in place of a launch of its own, and each reads its rows' parts again (four
  // drafted tokens over 151,936 logits, 75 pieces, all launches: one sequence 19 us against 24, 6 25 against 31, 16 40 against 44, 64 110 against 99).  The sums are the same.
  if ((int64_t)S * pieces <= 8 * vk_device_cus()) {
    verify_weigh_kernel<true><<<dim3(S, pieces), VERIFY_THREADS, 0, st>>>(a);
  } else {
    verify_decide_kernel<<<S, VERIFY_THREADS, 0, st>>>(a);
    if (vk_check_launch("verify (decide)")) return 1;
    verify_weigh_kernel<false><<<dim3(S, (pieces + 3) / 4), VERIFY_THREADS, 0, st>>>(a);
  }
  if (vk_check_launch("verify (weigh)")) return 1;
  verify_draw_kernel<<<S, VERIFY_THREADS, 0, st>>>(a);
  return vk_check_launch("verify (draw)");
}

}  // extern "C"
