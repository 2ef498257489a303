// Verification of drafted tokens against the target model's logits.
//
// Per sequence with drafts x_0..x_{d-1} and target rows l_0..l_d:
//     p_j = softmax(l_j / T)          (T <= 0: 1 at the row's first maximum)
//     x_j is accepted while u_j q_j(x_j) < p_j(x_j)
//     the first rejected row is sampled from max(p_j - q_j, 0), or, after all
//     drafts, row d from p_d: the first token whose running mass exceeds
//     u * (whole mass); where max(p - q, 0) is nothing, from p.
//
// A token's weight is e = exp2((l - m) log2(e) / T) in fp32, at most 1, and its
// mass max(e / S - q, 0), fp32 too; the factors log2(e) / T and 1 / S are kept in
// two terms each, since their rounding would shift every weight of a row alike.
// Sums (past eight tokens) and everything compared with a random number are
// fp64: a border of the running mass is then off by about 1e-9, where an fp32
// sum over 10^5 tokens moves it by 1e-5. (fp64 masses, which the weights' own
// roundings do not merit: 64 sequences x 151936 tokens 4 us slower.)
//
// Two launches. The first reads every target row once, a workgroup a piece of
// kVerifyPiece tokens, and leaves the piece's (max, sum, first maximum). The
// second has several workgroups for a sequence, about two a CU in all: each
// forms the decision from the rows' piece statistics (some KB; a launch of its
// own for it costs more), then the masses of its pieces of max(p - q, 0); the
// last one to arrive picks the token. A row without a draft's probabilities to
// subtract has its pieces' masses in the statistics already: its first workgroup
// picks alone, after it has summed the piece of a rejected token without it.
//
// The second launch is a chain of short steps, each run once: what bounds it is
// how many memory round trips and cross-lane reductions follow each other, and
// fetching its instructions. So a workgroup has 16 waves, a row's statistics or
// 512 of the piece's tokens each, reductions are register moves (DPP) instead of
// LDS ones, and loops are not unrolled (four waves, shuffles and 25 KB of code
// took 18 us for one sequence, without the copies of code 14; now 9). A workgroup
// a piece, 1216 of them, took 30 us for 64 sequences x 151936 tokens, the 512 of
// two a CU 19. The first launch is bound by HBM: 245 fp32 rows x 151936 in 26 us,
// 5.6 TB/s.
#include <algorithm>
#include <type_traits>

#include "le_common.h"
#include "le_internal.h"

namespace le {
namespace {

constexpr int kLaneTokens = 8;                     // consecutive tokens a lane takes at a time
constexpr int kStepTokens = kWave * kLaneTokens;   // and a wave
constexpr int kThreads = 256, kWaves = kThreads / kWave;  // the first launch
constexpr int kSteps = kVerifyPiece / (kWaves * kStepTokens);
constexpr int kPickWaves = kVerifyPiece / kStepTokens, kPickThreads = kPickWaves * kWave;  // the second
static_assert(kPickWaves == 16);
constexpr int kOwnPieces = 32;                     // pieces of one workgroup there, at most

struct PieceStat {  // 16 bytes
  float m;          // largest logit of the piece (-inf: none)
  int32_t arg;      // its first index, -1: none
  double s;         // sum of exp((l - m) / T)
};

// The row to sample from.
struct Choice {
  int64_t row;      // target row
  int64_t q_row;    // its draft row, to be subtracted; -1: none
  int32_t draft;    // the rejected token (drafts without probabilities: its mass is taken out); -1: none
  int32_t column;   // where the token goes
  float m, c_hi, c_lo;
  int32_t only;     // >= 0: the token is this one (T <= 0, or no logit above -inf)
  float s_hi, s_lo; // 1 / sum of the row's weights
};

// A lane's eight tokens from i on, and `skip`: the first of them that are not its
// own. Past the row's end the last eight tokens are read again and skipped, so
// there is one way to read a row; rows of fewer than eight tokens (TINY) are
// read one by one. Rows need no more than their element's alignment: the vector
// loads say so (memory takes them at any address).
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Eight { T v[8]; };
template <bool TINY> struct Place {
  int first, skip;  // token of the first element, elements of another lane
  __device__ __forceinline__ Place(int i, int vocab) {
    first = TINY ? 0 : min(i, vocab - kLaneTokens);
    skip = i - first;
  }
  template <typename T> __device__ __forceinline__ void load(const T* row, int vocab, float* o) const {
    if constexpr (TINY) {
#pragma unroll
      for (int e = 0; e < kLaneTokens; e++) o[e] = elem<T>::load1(row + min(e, vocab - 1));
    } else {
      const Eight<T> r = *reinterpret_cast<const Eight<T>*>(row + first);
#pragma unroll
      for (int e = 0; e < kLaneTokens; e++) o[e] = elem<T>::load1(&r.v[e]);
    }
  }
  __device__ __forceinline__ bool has(int e, int vocab) const { return e >= skip && (!TINY || e < vocab); }
};

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

// Eight weights in fp32 (three roundings), to be added up in fp64.
__device__ __forceinline__ double sum8(const float* w) {
  return static_cast<double>(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])));
}

// Cross-lane moves of 64-bit values; a lane that CTRL gives no source gets 0.
template <int CTRL> __device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, 0xF, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double f64_of(uint32_t lo, uint32_t hi) {
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// Sum over the wave, the same in every lane.
__device__ __forceinline__ double wave_sum_f64(double v) {
  v += dpp_f64<dpp::kXor1>(v);
  v += dpp_f64<dpp::kXor2>(v);
  v += dpp_f64<dpp::kHalfMirror>(v);
  v += dpp_f64<dpp::kMirror>(v);
  uint64_t u = __builtin_bit_cast(uint64_t, v);
  auto lo = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(u), static_cast<uint32_t>(u), false, false);
  auto hi = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(u >> 32), static_cast<uint32_t>(u >> 32), false, false);
  u = __builtin_bit_cast(uint64_t, f64_of(lo[0], hi[0]) + f64_of(lo[1], hi[1]));
  lo = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(u), static_cast<uint32_t>(u), false, false);
  hi = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(u >> 32), static_cast<uint32_t>(u >> 32), false, false);
  return f64_of(lo[0], hi[0]) + f64_of(lo[1], hi[1]);
}
// Inclusive sums over the lanes: within the rows of 16, then with the totals
// of the rows before.
__device__ __forceinline__ double lane_f64(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return f64_of(__builtin_amdgcn_readlane(static_cast<int>(u), lane), __builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane));
}
__device__ __forceinline__ double wave_scan_f64(double v) {
  v += dpp_f64<0x111>(v);  // row_shr:1
  v += dpp_f64<0x112>(v);
  v += dpp_f64<0x114>(v);
  v += dpp_f64<0x118>(v);
  const int row = (threadIdx.x & (kWave - 1)) >> 4;
  const double r0 = lane_f64(v, 15), r1 = r0 + lane_f64(v, 31), r2 = r1 + lane_f64(v, 47);
  return row == 0 ? v : v + (row == 1 ? r0 : row == 2 ? r1 : r2);
}
template <int CTRL> __device__ __forceinline__ int dpp_i32(int v) {
  return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ int wave_min_i32(int v) {
  v = min(v, dpp_i32<dpp::kXor1>(v));
  v = min(v, dpp_i32<dpp::kXor2>(v));
  v = min(v, dpp_i32<dpp::kHalfMirror>(v));
  v = min(v, dpp_i32<dpp::kMirror>(v));
  return min(min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             min(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
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
template <typename T, bool TINY>
__global__ __launch_bounds__(kThreads) void stats_kernel(VerifyParams p) {
  __shared__ PieceStat part[kWaves];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  const int piece = blockIdx.x, j = blockIdx.y, seq = blockIdx.z;
  if (piece == 0 && j == 0 && threadIdx.x == 0) p.arrivals[seq] = 0;
  int begin, n;
  if (!span_of(p, seq, begin, n) || j > n) return;
  const int64_t row = static_cast<int64_t>(begin) + seq + j;
  const T* l = static_cast<const T*>(p.logits) + row * p.logits_stride;
  const float t = temperature_of(p, seq);
  const int first = piece * kVerifyPiece + wave * kSteps * kStepTokens;
  auto place = [&](int k) { return Place<TINY>(first + k * kStepTokens + lane * kLaneTokens, p.vocab); };
  float x[kSteps][kLaneTokens];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kSteps; k++) place(k).load(l, p.vocab, x[k]);
  if (first + kSteps * kStepTokens > p.vocab) {  // what another lane has too, or nobody
#pragma unroll
    for (int k = 0; k < kSteps; k++)
#pragma unroll
      for (int e = 0; e < kLaneTokens; e++)
        if (!place(k).has(e, p.vocab)) x[k][e] = -INFINITY;
  }
#pragma unroll
  for (int k = 0; k < kSteps; k++)
#pragma unroll
    for (int e = 0; e < kLaneTokens; e++) m = fmaxf(m, x[k][e]);  // NaN is passed over
  m = wave_max(m);
  float c_hi = 0.f, c_lo = 0.f;
  int arg = INT32_MAX;
  double s = 0.0;
  if (t > 0.f) {
    factor(t, c_hi, c_lo);
    if (c_hi > 1e-30f && m < INFINITY) {
      // the weight without its special cases: what is too far below m to count,
      // -inf and NaN (a maximum passes over it) come to a weight of 2^-200, 0
      const float least = -200.f / c_hi;
#pragma unroll
      for (int k = 0; k < kSteps; k++) {
        float w[kLaneTokens];
#pragma unroll
        for (int e = 0; e < kLaneTokens; e++) {
          const float d = fmaxf(x[k][e] - m, least);
          w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(d, c_hi, d * c_lo));
        }
        s += sum8(w);
      }
      if (!(m > -INFINITY)) s = 0.0;
    } else if (m > -INFINITY) {
#pragma unroll 1
      for (int k = 0; k < kSteps; k++) {
        const Place<TINY> at = place(k);
        float y[kLaneTokens];
        at.load(l, p.vocab, y);
#pragma unroll
        for (int e = 0; e < kLaneTokens; e++) s += at.has(e, p.vocab) ? weight(y[e], m, c_hi, c_lo) : 0.f;
      }
    }
    s = wave_sum_f64(s);
  } else if (m > -INFINITY) {
#pragma unroll 1
    for (int k = kSteps - 1; k >= 0; k--) {
      const Place<TINY> at = place(k);
      float y[kLaneTokens];
      at.load(l, p.vocab, y);
#pragma unroll
      for (int e = kLaneTokens - 1; e >= 0; e--)
        if (at.has(e, p.vocab) && y[e] == m) arg = at.first + e;
    }
    arg = wave_min_i32(arg);
  }
  if (lane == 0) part[wave] = PieceStat{m, arg, s};
  __syncthreads();
  if (threadIdx.x == 0) {
    PieceStat all{part[0].m, INT32_MAX, 0.0};
    for (int w = 1; w < kWaves; w++) all.m = fmaxf(all.m, part[w].m);
    for (int w = 0; w < kWaves; w++) {
      if (part[w].m == all.m) all.arg = min(all.arg, part[w].arg);
      if (part[w].m > -INFINITY) all.s += part[w].s * static_cast<double>(weight(part[w].m, all.m, c_hi, c_lo));
    }
    static_cast<PieceStat*>(p.stats)[row * p.n_pieces + piece] = all;
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
  PieceStat own{-INFINITY, INT32_MAX, 0.0};  // of this lane's pieces
  for (int i = lane; i < p.n_pieces; i += kWave) {
    const PieceStat a = st[i];
    if (!(a.m > -INFINITY)) continue;
    if (a.m > own.m) {
      own.s = a.s + (own.m > -INFINITY ? own.s * static_cast<double>(weight(own.m, a.m, c_hi, c_lo)) : 0.0);
      own.m = a.m;
      own.arg = a.arg;
    } else {
      own.s += a.s * static_cast<double>(weight(a.m, own.m, c_hi, c_lo));
      if (a.m == own.m) own.arg = min(own.arg, a.arg);
    }
  }
  const float m = wave_max(own.m);
  const double s = own.m > -INFINITY ? own.s * static_cast<double>(weight(own.m, m, c_hi, c_lo)) : 0.0;
  return RowStat{m, wave_min_i32(own.m == m ? own.arg : INT32_MAX), wave_sum_f64(s)};
}

// exp((l - m) / T) in fp64, for the one token that is compared with a random number
__device__ __forceinline__ double weight_f64(float l, float m, float t) {
  if (l == m) return 1.0;
  if (!(l < m) || l == -INFINITY || m == INFINITY) return 0.0;
  return exp((static_cast<double>(l) - static_cast<double>(m)) / static_cast<double>(t));
}

// The masses of a lane's eight tokens; residual: less the draft's.
template <typename T, typename Q, bool TINY>
__device__ __forceinline__ void masses(const VerifyParams& p, const Choice& c, const Place<TINY>& at, bool residual,
                                       float* w) {
  float l[kLaneTokens], q[kLaneTokens];
  at.load(static_cast<const T*>(p.logits) + c.row * p.logits_stride, p.vocab, l);
  const bool less = residual && c.q_row >= 0;
#pragma unroll
  for (int e = 0; e < kLaneTokens; e++) q[e] = 0.f;
  if (less) at.load(static_cast<const Q*>(p.draft_probs) + c.q_row * p.probs_stride, p.vocab, q);
#pragma unroll
  for (int e = 0; e < kLaneTokens; e++) {
    const float x = weight(l[e], c.m, c.c_hi, c.c_lo);
    const float left = fmaxf(__builtin_fmaf(x, c.s_hi, __builtin_fmaf(x, c.s_lo, -q[e])), 0.f);  // (of a NaN: nothing)
    w[e] = at.has(e, p.vocab) && !(residual && at.first + e == c.draft) ? left : 0.f;
  }
}
// ---- the decision, the masses of the row to sample from, and the token ----
struct VerifySmem {
  Choice choice;
  int first;              // the first row that is not accepted
  int last;               // this workgroup arrived last
  double sum[kOwnPieces][kPickWaves];
  double border, before;  // random number times the whole mass; mass before the piece
  int piece, residual;
};

// A sequence's number of accepted drafts, and the row that its next token comes
// from, left in sm.choice. Every workgroup of the sequence comes to the same.
template <typename T, typename Q>
__device__ __forceinline__ int decide(const VerifyParams& p, VerifySmem& sm, int seq, int begin, int n, float t) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) sm.first = n;
  __syncthreads();
  float c_hi = 0.f, c_lo = 0.f;
  if (t > 0.f) factor(t, c_hi, c_lo);
  const T* logits = static_cast<const T*>(p.logits);
  const Q* probs = static_cast<const Q*>(p.draft_probs);
  // a wave's rows, up to its first that is rejected, or row n
  RowStat r{};
  int mine = n + 1, x = -1;
#pragma unroll 1
  for (int j = wave; j <= n; j += kPickWaves) {
    const int64_t row = static_cast<int64_t>(begin) + seq + j;
    // the draft's own values, on their way beside the statistics
    x = -1;
    float u = 0.f, l = 0.f, q = 1.f;
    if (j < n) {
      x = p.draft_tokens[begin + j];
      u = p.accept_u[begin + j];
      if (x >= 0 && x < p.vocab) {
        l = elem<T>::load1(logits + row * p.logits_stride + x);
        if (probs) q = elem<Q>::load1(probs + (static_cast<int64_t>(begin) + j) * p.probs_stride + x);
      }
    }
    r = row_stat(p, row, c_hi, c_lo);
    bool ok = false;
    if (x >= 0 && x < p.vocab) {
      double w, s = 1.0;
      if (t > 0.f && r.m > -INFINITY) {
        w = weight_f64(l, r.m, t);
        s = r.s;
      } else {
        w = x == (r.m > -INFINITY ? r.arg : 0) ? 1.0 : 0.0;
      }
      ok = static_cast<double>(u) * static_cast<double>(q) * s < w;
    }
    if (!ok) {
      mine = j;
      break;
    }
  }
  if (lane == 0) atomicMin(&sm.first, mine);
  __syncthreads();
  const int acc = sm.first;
  if (mine == acc && lane == 0) {
    Choice c;
    c.row = static_cast<int64_t>(begin) + seq + acc;
    c.q_row = acc < n && probs ? static_cast<int64_t>(begin) + acc : -1;
    c.draft = acc < n && !probs && x < p.vocab ? x : -1;
    c.column = acc;
    c.m = r.m;
    c.c_hi = c_hi;
    c.c_lo = c_lo;
    c.only = !(r.m > -INFINITY) ? 0 : (t > 0.f ? -1 : r.arg);
    const double inv = 1.0 / r.s;
    c.s_hi = static_cast<float>(inv);
    c.s_lo = static_cast<float>(inv - static_cast<double>(c.s_hi));
    sm.choice = c;
  }
  __syncthreads();
  return acc;
}

// The token: the piece that the border falls into, the wave's share of it, the
// place in that.
template <typename T, typename Q, bool TINY>
__device__ __forceinline__ void pick(const VerifyParams& p, VerifySmem& sm, int seq, float t, int32_t* out) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  const Choice c = sm.choice;
  if (wave == 0) {
    const double u = static_cast<double>(p.sample_u[seq]);
    double* mass = p.mass + static_cast<int64_t>(seq) * p.n_pieces;
    const PieceStat* st = static_cast<const PieceStat*>(p.stats) + c.row * p.n_pieces;
    bool residual = c.q_row >= 0 || c.draft >= 0;
    const int less = c.draft >= 0 ? c.draft / kVerifyPiece : -1;  // the rejected token's piece, summed without it
    const double rest = less >= 0 ? wave_sum_f64(lane < kPickWaves ? sm.sum[0][lane] : 0.0) : 0.0;
    const double inv = static_cast<double>(c.s_hi) + static_cast<double>(c.s_lo);
    auto piece_mass = [&](int i) {
      if (i >= p.n_pieces) return 0.0;
      // written by this launch's workgroups (read past this XCD's L2)
      if (residual && c.q_row >= 0) return __hip_atomic_load(mass + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (residual && i == less) return rest;
      const PieceStat a = st[i];
      // (in fp64: an fp32 factor would move all of the piece's mass by up to 6e-8 of it)
      return a.m > -INFINITY ? a.s * (weight_f64(a.m, c.m, t) * inv) : 0.0;
    };
    double w0 = 0.0, total = 0.0;  // w0: of this lane's first piece
#pragma unroll 1
    for (;;) {
      w0 = piece_mass(lane);
      total = w0;
#pragma unroll 1
      for (int i = kWave + lane; i < p.n_pieces; i += kWave) total += piece_mass(i);
      total = wave_sum_f64(total);
      if (!residual || total > 0.0) break;
      residual = false;  // nothing is left of p: all of it
    }
    const double border = u * total;
    // the first piece whose running mass exceeds the border; the last one with
    // any mass where none does (u of 1 or more, NaN, or the sums' last bits)
    int piece = 0;
    double before = 0.0, run = 0.0;
#pragma unroll 1
    for (int i0 = 0; i0 < p.n_pieces; i0 += kWave) {
      const double w = i0 == 0 ? w0 : piece_mass(i0 + lane);
      const double sum = run + wave_scan_f64(w);
      const uint64_t over = __builtin_amdgcn_ballot_w64(w > 0.0 && sum > border);
      const uint64_t any = __builtin_amdgcn_ballot_w64(w > 0.0);
      if (any) {
        const int at = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any);
        piece = i0 + at;
        before = lane_f64(sum - w, at);
      }
      if (over) break;
      run = lane_f64(sum, kWave - 1);
    }
    if (lane == 0) {
      sm.piece = piece;
      sm.before = before;
      sm.border = border;
      sm.residual = residual;
    }
  }
  __syncthreads();
  const double border = sm.border;
  const Place<TINY> at(sm.piece * kVerifyPiece + wave * kStepTokens + lane * kLaneTokens, p.vocab);
  float w[kLaneTokens];
  double own = 0.0;
  masses<T, Q>(p, c, at, sm.residual != 0, w);
#pragma unroll
  for (int e = 0; e < kLaneTokens; e++) own += w[e];
  const double mine = wave_scan_f64(own);
  if (lane == kWave - 1) sm.sum[0][wave] = mine;
  __syncthreads();
  // the first wave whose running mass exceeds the border has the token; the
  // last one with any mass where none does
  const double share = lane < kPickWaves ? sm.sum[0][lane] : 0.0;
  const double upto = sm.before + wave_scan_f64(share);
  const uint64_t over = __builtin_amdgcn_ballot_w64(share > 0.0 && upto > border);
  const uint64_t any = __builtin_amdgcn_ballot_w64(share > 0.0);
  const int who = over ? __builtin_ctzll(over) : any ? 63 - __builtin_clzll(any) : 0;
  if (wave != who) return;
  double x = lane_f64(upto - share, who) + (mine - own);
  int first = INT32_MAX, tail = -1;
#pragma unroll
  for (int e = 0; e < kLaneTokens; e++) {
    x += w[e];
    if (w[e] > 0.0) {
      tail = at.first + e;
      if (x > border) first = min(first, tail);
    }
  }
  first = wave_min_i32(first);
  tail = -wave_min_i32(-tail);  // the last token with any mass
  if (lane == 0) *out = first != INT32_MAX ? first : max(tail, 0);
}

template <typename T, typename Q, bool TINY>
__global__ __launch_bounds__(kPickThreads, 8) void verify_kernel(VerifyParams p) {
  __shared__ VerifySmem sm;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  // this workgroup's pieces: first, first + step, ...
  const int first = blockIdx.x, step = gridDim.x, seq = blockIdx.y;
  int32_t* out = p.out + static_cast<int64_t>(seq) * (p.max_drafts + 1);
  const float t = temperature_of(p, seq);
  int begin, n;
  if (!span_of(p, seq, begin, n)) {
    if (first == 0) {
#pragma unroll 1
      for (int i = threadIdx.x; i <= p.max_drafts; i += kPickThreads) out[i] = -1;
      if (threadIdx.x == 0) p.n_accepted[seq] = -1;
    }
    return;
  }
  if (first > 0 && (n == 0 || !(t > 0.f))) return;  // nothing to subtract
  const int acc = decide<T, Q>(p, sm, seq, begin, n, t);
  const Choice& c = sm.choice;
  const bool subtract = c.only < 0 && c.q_row >= 0;
  if (first > 0 && !subtract) return;
  if (subtract) {
    const Choice mine = c;
    int count = 0;
#pragma unroll 2
    for (int piece = first; piece < p.n_pieces; piece += step, count++) {
      float w[kLaneTokens];
      masses<T, Q>(p, mine, Place<TINY>(piece * kVerifyPiece + wave * kStepTokens + lane * kLaneTokens, p.vocab), true, w);
      const double s = wave_sum_f64(sum8(w));
      if (lane == 0) sm.sum[count][wave] = s;
    }
    __syncthreads();
#pragma unroll 1
    for (int i = wave; i < count; i += kPickWaves) {
      const double all = wave_sum_f64(lane < kPickWaves ? sm.sum[i][lane] : 0.0);
      if (lane == 0)
        __hip_atomic_store(p.mass + static_cast<int64_t>(seq) * p.n_pieces + first + i * step, all, __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
    }
    __builtin_amdgcn_s_waitcnt(0);  // the masses are where every XCD reads them before the arrival counts
    __syncthreads();
    if (threadIdx.x == 0)
      sm.last = __hip_atomic_fetch_add(p.arrivals + seq, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == step - 1;
  }
  if (c.only < 0 && c.draft >= 0) {
    const Choice mine = c;
    float w[kLaneTokens];
    const int piece = mine.draft / kVerifyPiece;
    masses<T, Q>(p, mine, Place<TINY>(piece * kVerifyPiece + wave * kStepTokens + lane * kLaneTokens, p.vocab), true, w);
    const double s = wave_sum_f64(sum8(w));
    if (lane == 0) sm.sum[0][wave] = s;
    __syncthreads();
  }
  if (first == 0) {
#pragma unroll 1
    for (int i = threadIdx.x; i <= p.max_drafts; i += kPickThreads)
      if (i != acc) out[i] = i < acc ? p.draft_tokens[begin + i] : -1;
    if (threadIdx.x == 0) {
      p.n_accepted[seq] = acc;
      if (c.only >= 0) out[acc] = c.only;
    }
    if (c.only >= 0) return;
  }
  if (subtract) {
    __syncthreads();
    if (!sm.last) return;
  }
  pick<T, Q, TINY>(p, sm, seq, t, out + acc);
}

}  // namespace

size_t verify_workspace(int64_t n_seqs, int64_t n_drafts, int vocab) {
  const size_t pieces = (static_cast<size_t>(vocab) + kVerifyPiece - 1) / kVerifyPiece;
  return static_cast<size_t>(n_seqs + n_drafts) * pieces * sizeof(PieceStat) +
         static_cast<size_t>(n_seqs) * (pieces * sizeof(double) + sizeof(int32_t));
}

hipError_t verify_drafts(const VerifyParams& in, int logits_dtype, int probs_dtype, void* workspace,
                         hipStream_t stream) {
  VerifyParams p = in;
  p.n_pieces = (p.vocab - 1) / kVerifyPiece + 1;
  char* ws = static_cast<char*>(workspace);
  p.stats = ws;
  ws += static_cast<size_t>(p.n_seqs + p.n_drafts) * p.n_pieces * sizeof(PieceStat);
  p.mass = reinterpret_cast<double*>(ws);
  p.arrivals = reinterpret_cast<int32_t*>(ws + static_cast<size_t>(p.n_seqs) * p.n_pieces * sizeof(double));
  const unsigned pieces = static_cast<unsigned>(p.n_pieces), seqs = static_cast<unsigned>(p.n_seqs);
  // two workgroups of the second launch fit on a CU
  const unsigned share = p.draft_probs ? std::min(pieces, std::max({512u / seqs, (pieces + kOwnPieces - 1) / kOwnPieces, 1u})) : 1u;
  return with_dtype(logits_dtype, [&](auto a) {
    return with_dtype(probs_dtype, [&](auto b) {
      using T = decltype(a);
      using Q = decltype(b);
      auto launch = [&](auto tiny) {
        constexpr bool TINY = decltype(tiny)::value;
        stats_kernel<T, TINY><<<dim3(pieces, static_cast<unsigned>(p.max_drafts + 1), seqs), kThreads, 0, stream>>>(p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        verify_kernel<T, Q, TINY><<<dim3(share, seqs), kPickThreads, 0, stream>>>(p);
        return hipGetLastError();
      };
      return p.vocab < kLaneTokens ? launch(std::true_type{}) : launch(std::false_type{});
    });
  });
}

}  // namespace le
