// Verification of drafted tokens against the target model's logits.
//
// Per sequence with drafts x_0..x_{d-1} and target rows l_0..l_d:
//     p_j = softmax(l_j / T)          (T <= 0: 1 at the row's first maximum)
//     x_j is accepted while u_j q_j(x_j) < p_j(x_j)
//     the first rejected row is sampled from max(p_j - q_j, 0), or, after all
//     drafts, row d from p_d: the first token whose running mass exceeds
//     u * (whole mass); where max(p - q, 0) is nothing, from p.
//
// A token's weight is e = exp2((l - m) log2(e) / T) in fp32, at most 1; the
// factor is kept in two terms, since its rounding would shift every weight of
// a row alike. Sums of weights and everything compared with a random number
// are fp64: a border of the running mass is then off by about 1e-8, where an
// fp32 sum over 10^5 tokens moves it by 1e-5.
//
// A row is read in pieces of kPiece tokens, one wave each, so that one
// sequence's rows spread over the chip and no barrier is needed: first every
// target row's (max, sum, first maximum) per piece, then, per sequence, the
// decision, the rejected row's residual masses per piece, and the token.
#include "le_common.h"
#include "le_internal.h"

namespace le {
namespace {

constexpr int kLaneTokens = 8;                          // consecutive tokens a lane takes at a time
constexpr int kSteps = kVerifyPiece / (kWave * kLaneTokens);

struct PieceStat {  // 16 bytes
  float m;          // largest logit of the piece (-inf: none)
  int32_t arg;      // its first index, -1: none
  double s;         // sum of exp((l - m) / T)
};

// The row to sample from, as the decision leaves it for the later kernels.
struct Choice {
  int64_t row;      // target row; -1: the sequence's offsets are invalid
  int64_t q_row;    // its draft row, to be subtracted; -1: none
  int32_t draft;    // the rejected token (drafts without probabilities: its mass is taken out); -1: none
  int32_t column;   // where the token goes
  float m, c_hi, c_lo;
  int32_t only;     // >= 0: the token is this one (T <= 0, or no logit above -inf)
  double inv_s;     // 1 / sum of the row's weights
};

// Eight consecutive elements at i, of which n are in the row; the others come
// back as `fill`. Rows need no more than their element's alignment: the
// vector loads say so (memory takes them at any address).
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Eight { T v[8]; };
template <typename T>
__device__ __forceinline__ void load_tokens(const T* row, int64_t i, int64_t n, float fill, float* o) {
  if (n >= kLaneTokens) {
    const Eight<T> r = *reinterpret_cast<const Eight<T>*>(row + i);
#pragma unroll
    for (int e = 0; e < kLaneTokens; e++) o[e] = elem<T>::load1(&r.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < kLaneTokens; e++) o[e] = e < n ? elem<T>::load1(row + i + e) : fill;
  }
}

// weight of a logit under the row's maximum m > -inf; NaN and -inf weigh
// nothing (nor does a finite logit under +inf, or one too far below m: a
// comparison with a NaN or -inf fails)
__device__ __forceinline__ float weight(float l, float m, float c_hi, float c_lo) {
  const float d = l - m, x = d * c_hi;
  const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(d, c_hi, d * c_lo));
  return l == m ? 1.f : (x > -200.f ? e : 0.f);
}
__device__ __forceinline__ void factor(float t, float& c_hi, float& c_lo) {
  const double c = 1.4426950408889634 / static_cast<double>(t);
  c_hi = static_cast<float>(c);
  if (!(c_hi < 3.0e38f)) {  // a temperature so small that only the maximum is left
    c_hi = 3.0e38f;
    c_lo = 0.f;
  } else {
    c_lo = static_cast<float>(c - static_cast<double>(c_hi));
  }
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) v += __shfl_xor(v, d, kWave);
  return v;
}
__device__ __forceinline__ int wave_min_i32(int v) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) v = min(v, __shfl_xor(v, d, kWave));
  return v;
}

// A sequence's drafts [begin, begin + n); false where its offsets are not
// within the drafts or hold more than max_drafts.
__device__ __forceinline__ bool span_of(const VerifyParams& p, int seq, int& begin, int& n) {
  begin = p.cu_drafts[seq];
  const int end = p.cu_drafts[seq + 1];
  n = end - begin;
  return begin >= 0 && end >= begin && end <= p.n_drafts && n <= p.max_drafts;
}
__device__ __forceinline__ float temperature_of(const VerifyParams& p, int seq) {
  return p.temperature ? p.temperature[seq] : 1.f;
}

// ---- (max, sum, first maximum) of every piece of every target row ----
template <typename T>
__global__ __launch_bounds__(256) void stats_kernel(VerifyParams p) {
  const int lane = threadIdx.x & (kWave - 1);
  const int piece = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int seq = blockIdx.z, j = blockIdx.y;
  int begin, n;
  if (piece >= p.n_pieces || !span_of(p, seq, begin, n) || j > n) return;
  const int64_t row = static_cast<int64_t>(begin) + seq + j;
  const T* l = static_cast<const T*>(p.logits) + row * p.logits_stride;
  const float t = temperature_of(p, seq);
  float x[kSteps][kLaneTokens];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kSteps; k++) {
    const int64_t i = static_cast<int64_t>(piece) * kVerifyPiece + (k * kWave + lane) * kLaneTokens;
    load_tokens(l, i, p.vocab - i, -INFINITY, x[k]);
  }
#pragma unroll
  for (int k = 0; k < kSteps; k++)
#pragma unroll
    for (int e = 0; e < kLaneTokens; e++) m = fmaxf(m, x[k][e]);  // NaN is passed over
  m = wave_max(m);
  int arg = INT32_MAX;
#pragma unroll
  for (int k = kSteps - 1; k >= 0; k--)
#pragma unroll
    for (int e = kLaneTokens - 1; e >= 0; e--)
      if (x[k][e] == m) arg = piece * kVerifyPiece + (k * kWave + lane) * kLaneTokens + e;
  arg = wave_min_i32(arg);
  double s = 0.0;
  if (t > 0.f && m > -INFINITY) {
    float c_hi, c_lo;
    factor(t, c_hi, c_lo);
#pragma unroll
    for (int k = 0; k < kSteps; k++)
#pragma unroll
      for (int e = 0; e < kLaneTokens; e++) s += weight(x[k][e], m, c_hi, c_lo);
    s = wave_sum_f64(s);
  }
  if (lane == 0) {
    PieceStat* st = static_cast<PieceStat*>(p.stats) + row * p.n_pieces + piece;
    *st = PieceStat{m, m > -INFINITY ? arg : -1, s};
  }
}

// A row's (max, sum, first maximum) from its pieces, by one wave.
struct RowStat {
  float m;
  int32_t arg;
  double s;
};
__device__ __forceinline__ RowStat row_stat(const VerifyParams& p, int64_t row, float c_hi, float c_lo) {
  const int lane = threadIdx.x & (kWave - 1);
  const PieceStat* st = static_cast<const PieceStat*>(p.stats) + row * p.n_pieces;
  float m = -INFINITY;
  for (int i = lane; i < p.n_pieces; i += kWave) m = fmaxf(m, st[i].m);
  m = wave_max(m);
  int arg = INT32_MAX;
  double s = 0.0;
  for (int i = lane; i < p.n_pieces; i += kWave) {
    const PieceStat a = st[i];
    if (a.m == m && a.arg >= 0) arg = min(arg, a.arg);
    s += a.s * static_cast<double>(weight(a.m, m, c_hi, c_lo));
  }
  return RowStat{m, wave_min_i32(arg), wave_sum_f64(s)};
}

// exp((l - m) / T) in fp64, for the one token that is compared with a random number
__device__ __forceinline__ double weight_f64(float l, float m, float t) {
  if (l == m) return 1.0;
  if (!(l < m) || l == -INFINITY || m == INFINITY) return 0.0;
  return exp((static_cast<double>(l) - static_cast<double>(m)) / static_cast<double>(t));
}

// ---- a sequence's accepted drafts, and the row its next token comes from ----
template <typename T, typename Q>
__global__ __launch_bounds__(256) void decide_kernel(VerifyParams p) {
  __shared__ int first;  // the first row that is not accepted
  const int seq = blockIdx.x;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  Choice* choice = static_cast<Choice*>(p.choices) + seq;
  int32_t* out = p.out + static_cast<int64_t>(seq) * (p.max_drafts + 1);
  for (int i = threadIdx.x; i <= p.max_drafts; i += 256) out[i] = -1;
  int begin, n;
  if (!span_of(p, seq, begin, n)) {
    if (threadIdx.x == 0) {
      p.n_accepted[seq] = -1;
      choice->row = -1;
    }
    return;
  }
  if (threadIdx.x == 0) first = n;
  __syncthreads();
  const float t = temperature_of(p, seq);
  float c_hi = 0.f, c_lo = 0.f;
  if (t > 0.f) factor(t, c_hi, c_lo);
  const T* logits = static_cast<const T*>(p.logits);
  const Q* probs = static_cast<const Q*>(p.draft_probs);
  for (int j = wave; j < n; j += 4) {
    const int64_t row = static_cast<int64_t>(begin) + seq + j;
    const RowStat r = row_stat(p, row, c_hi, c_lo);
    if (lane == 0) {
      const int x = p.draft_tokens[begin + j];
      bool ok = false;
      if (x >= 0 && x < p.vocab) {
        const double q = probs ? static_cast<double>(elem<Q>::load1(probs + (begin + j) * p.probs_stride + x)) : 1.0;
        const double u = static_cast<double>(p.accept_u[begin + j]);
        double w, s = 1.0;
        if (t > 0.f && r.m > -INFINITY) {
          w = weight_f64(elem<T>::load1(logits + row * p.logits_stride + x), r.m, t);
          s = r.s;
        } else {
          w = x == (r.m > -INFINITY ? r.arg : 0) ? 1.0 : 0.0;
        }
        ok = u * q * s < w;
      }
      if (!ok) atomicMin(&first, j);
    }
  }
  __syncthreads();
  const int acc = first;
  for (int j = threadIdx.x; j < acc; j += 256) out[j] = p.draft_tokens[begin + j];
  if (wave != 0) return;
  const int64_t row = static_cast<int64_t>(begin) + seq + acc;
  const RowStat r = row_stat(p, row, c_hi, c_lo);
  if (lane == 0) {
    p.n_accepted[seq] = acc;
    Choice c;
    c.row = row;
    c.q_row = acc < n && probs ? begin + acc : -1;
    c.draft = acc < n && !probs ? p.draft_tokens[begin + acc] : -1;
    c.column = acc;
    c.m = r.m;
    c.c_hi = c_hi;
    c.c_lo = c_lo;
    c.only = !(r.m > -INFINITY) ? 0 : (t > 0.f ? -1 : r.arg);
    c.inv_s = 1.0 / r.s;
    *choice = c;
  }
}

// The masses of a lane's eight tokens from i on; residual: less the draft's.
template <typename T, typename Q>
__device__ __forceinline__ void masses(const VerifyParams& p, const Choice& c, int64_t i, bool residual, double* w) {
  float l[kLaneTokens], q[kLaneTokens];
  load_tokens(static_cast<const T*>(p.logits) + c.row * p.logits_stride, i, p.vocab - i, -INFINITY, l);
  const bool less = residual && c.q_row >= 0;
  if (less)
    load_tokens(static_cast<const Q*>(p.draft_probs) + c.q_row * p.probs_stride, i, p.vocab - i, 0.f, q);
#pragma unroll
  for (int e = 0; e < kLaneTokens; e++) {
    w[e] = static_cast<double>(weight(l[e], c.m, c.c_hi, c.c_lo)) * c.inv_s;
    if (less) w[e] = fmax(w[e] - static_cast<double>(q[e]), 0.0);  // a NaN leaves nothing
    if (residual && i + e == c.draft) w[e] = 0.0;
  }
}

// ---- masses of every piece of the row to sample from ----
template <typename T, typename Q>
__global__ __launch_bounds__(256) void mass_kernel(VerifyParams p) {
  const int lane = threadIdx.x & (kWave - 1);
  const int piece = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int seq = blockIdx.y;
  if (piece >= p.n_pieces) return;
  const Choice c = static_cast<const Choice*>(p.choices)[seq];
  if (c.row < 0 || c.only >= 0) return;
  double s = 0.0;
#pragma unroll
  for (int k = 0; k < kSteps; k++) {
    const int64_t i = static_cast<int64_t>(piece) * kVerifyPiece + (k * kWave + lane) * kLaneTokens;
    double w[kLaneTokens];
    masses<T, Q>(p, c, i, true, w);
#pragma unroll
    for (int e = 0; e < kLaneTokens; e++) s += w[e];
  }
  s = wave_sum_f64(s);
  if (lane == 0) p.mass[static_cast<int64_t>(seq) * p.n_pieces + piece] = s;
}

__device__ __forceinline__ double wave_scan_f64(double v) {  // inclusive
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const double o = __shfl_up(v, d, kWave);
    if (lane >= d) v += o;
  }
  return v;
}

// ---- the token: the piece that the border falls into, then the place in it ----
template <typename T, typename Q>
__global__ __launch_bounds__(kWave) void pick_kernel(VerifyParams p) {
  const int lane = threadIdx.x, seq = blockIdx.x;
  const Choice c = static_cast<const Choice*>(p.choices)[seq];
  if (c.row < 0) return;
  int32_t* out = p.out + static_cast<int64_t>(seq) * (p.max_drafts + 1) + c.column;
  if (c.only >= 0) {
    if (lane == 0) *out = c.only;
    return;
  }
  const double u = static_cast<double>(p.sample_u[seq]);
  const double* mass = p.mass + static_cast<int64_t>(seq) * p.n_pieces;
  const PieceStat* st = static_cast<const PieceStat*>(p.stats) + c.row * p.n_pieces;
  bool residual = true;
  auto piece_mass = [&](int i) {
    if (i >= p.n_pieces) return 0.0;
    return residual ? mass[i] : st[i].s * static_cast<double>(weight(st[i].m, c.m, c.c_hi, c.c_lo)) * c.inv_s;
  };
  auto total_of = [&]() {
    double s = 0.0;
    for (int i = lane; i < p.n_pieces; i += kWave) s += piece_mass(i);
    return wave_sum_f64(s);
  };
  double total = total_of();
  if (!(total > 0.0)) {
    residual = false;
    total = total_of();
  }
  const double border = u * total;
  // the first piece whose running mass exceeds the border; the last one with
  // any mass where none does (u of 1 or more, NaN, or the sums' last bits)
  int piece = -1, last = -1;
  double before = 0.0, run = 0.0, last_before = 0.0;
  for (int i0 = 0; i0 < p.n_pieces && piece < 0; i0 += kWave) {
    const double w = piece_mass(i0 + lane);
    const double sum = run + wave_scan_f64(w);
    const uint64_t over = __builtin_amdgcn_ballot_w64(w > 0.0 && sum > border);
    const uint64_t any = __builtin_amdgcn_ballot_w64(w > 0.0);
    if (over) {
      const int at = __builtin_ctzll(over);
      piece = i0 + at;
      before = __shfl(sum, at, kWave) - __shfl(w, at, kWave);
    } else if (any) {
      const int at = 63 - __builtin_clzll(any);
      last = i0 + at;
      last_before = __shfl(sum, at, kWave) - __shfl(w, at, kWave);
    }
    run = __shfl(sum, kWave - 1, kWave);
  }
  if (piece < 0) {
    piece = last;
    before = last_before;
  }
  int token = -1, tail = 0;  // tail: the last token of the piece with any mass
  run = before;
  for (int k = 0; k < kSteps && piece >= 0 && token < 0; k++) {
    const int64_t i = static_cast<int64_t>(piece) * kVerifyPiece + (k * kWave + lane) * kLaneTokens;
    double w[kLaneTokens], own = 0.0;
    masses<T, Q>(p, c, i, residual, w);
#pragma unroll
    for (int e = 0; e < kLaneTokens; e++) own += w[e];
    const double upto = run + wave_scan_f64(own);
    double at = upto - own;
    int mine = INT32_MAX, final_mine = -1;
#pragma unroll
    for (int e = 0; e < kLaneTokens; e++) {
      at += w[e];
      if (w[e] > 0.0) {
        if (at > border) mine = min(mine, static_cast<int>(i) + e);
        final_mine = static_cast<int>(i) + e;
      }
    }
    const int got = wave_min_i32(mine);
    if (got != INT32_MAX) token = got;
    const int fin = -wave_min_i32(-final_mine);
    if (fin >= 0) tail = fin;
    run = __shfl(upto, kWave - 1, kWave);
  }
  if (lane == 0) *out = token >= 0 ? token : tail;
}

}  // namespace

size_t verify_workspace(int64_t n_seqs, int64_t n_drafts, int vocab) {
  const size_t pieces = (static_cast<size_t>(vocab) + kVerifyPiece - 1) / kVerifyPiece;
  return static_cast<size_t>(n_seqs) * sizeof(Choice) + static_cast<size_t>(n_seqs + n_drafts) * pieces * sizeof(PieceStat) +
         static_cast<size_t>(n_seqs) * pieces * sizeof(double);
}

hipError_t verify_drafts(const VerifyParams& in, int logits_dtype, int probs_dtype, void* workspace,
                         hipStream_t stream) {
  VerifyParams p = in;
  p.n_pieces = (p.vocab - 1) / kVerifyPiece + 1;
  char* ws = static_cast<char*>(workspace);
  p.choices = ws;
  ws += static_cast<size_t>(p.n_seqs) * sizeof(Choice);
  p.stats = ws;
  ws += static_cast<size_t>(p.n_seqs + p.n_drafts) * p.n_pieces * sizeof(PieceStat);
  p.mass = reinterpret_cast<double*>(ws);
  const unsigned groups = static_cast<unsigned>((p.n_pieces + 3) / 4), seqs = static_cast<unsigned>(p.n_seqs);
  return with_dtype(logits_dtype, [&](auto a) {
    return with_dtype(probs_dtype, [&](auto b) {
      using T = decltype(a);
      using Q = decltype(b);
      stats_kernel<T><<<dim3(groups, static_cast<unsigned>(p.max_drafts + 1), seqs), 256, 0, stream>>>(p);
      decide_kernel<T, Q><<<seqs, 256, 0, stream>>>(p);
      mass_kernel<T, Q><<<dim3(groups, seqs), 256, 0, stream>>>(p);
      pick_kernel<T, Q><<<seqs, kWave, 0, stream>>>(p);
      return hipGetLastError();
    });
  });
}

}  // namespace le
