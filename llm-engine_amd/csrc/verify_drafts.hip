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
// Two launches. The first reads every target row once, a workgroup a piece of
// kVerifyPiece tokens, and leaves the piece's (max, sum, first maximum). The
// second has a workgroup for every (sequence, piece): each forms the decision
// from the rows' piece statistics (some KB; a launch of its own for it costs
// more), then the mass of its piece of max(p - q, 0); the last one to arrive
// picks the token. A row without drafts' probabilities to subtract has its
// pieces' masses in the statistics already: its first workgroup picks alone.
#include "le_common.h"
#include "le_internal.h"

namespace le {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kLaneTokens = 8;                          // consecutive tokens a lane takes at a time
constexpr int kWavePiece = kVerifyPiece / kWaves;       // consecutive tokens of a wave
constexpr int kSteps = kWavePiece / (kWave * kLaneTokens);
constexpr int kHeldRows = 32;                           // rows whose statistics a workgroup keeps

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
  const int64_t first = static_cast<int64_t>(piece) * kVerifyPiece + wave * kWavePiece;
  float x[kSteps][kLaneTokens];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kSteps; k++) {
    const int64_t i = first + (k * kWave + lane) * kLaneTokens;
    load_tokens(l, i, p.vocab - i, -INFINITY, x[k]);
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
        // eight weights in fp32 (three roundings), the rest of the row in fp64
        s += static_cast<double>(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])));
      }
      if (!(m > -INFINITY)) s = 0.0;
    } else {
#pragma unroll
      for (int k = 0; k < kSteps; k++)
#pragma unroll
        for (int e = 0; e < kLaneTokens; e++) s += m > -INFINITY ? weight(x[k][e], m, c_hi, c_lo) : 0.f;
    }
    s = wave_sum_f64(s);
  } else if (m > -INFINITY) {
#pragma unroll
    for (int k = kSteps - 1; k >= 0; k--)
#pragma unroll
      for (int e = kLaneTokens - 1; e >= 0; e--)
        if (x[k][e] == m) arg = static_cast<int>(first) + (k * kWave + lane) * kLaneTokens + e;
    arg = wave_min_i32(arg);
  }
  if (lane == 0) part[wave] = PieceStat{m, arg, s};
  __syncthreads();
  if (threadIdx.x == 0) {
    PieceStat all = part[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++) all.m = fmaxf(all.m, part[w].m);
    all.arg = INT32_MAX;
    all.s = 0.0;
#pragma unroll
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

__device__ __forceinline__ double wave_scan_f64(double v) {  // inclusive
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const double o = __shfl_up(v, d, kWave);
    if (lane >= d) v += o;
  }
  return v;
}

// ---- the decision, the masses of the row to sample from, and the token ----
struct VerifySmem {
  RowStat rows[kHeldRows];
  Choice choice;
  int first;             // the first row that is not accepted
  int last;              // this workgroup arrived last
  double sum[kWaves];
  double border, before;  // random number times the whole mass; mass before the piece
  int piece, residual, token, tail;
};

// A sequence's accepted drafts, and the row its next token comes from: left in
// sm.choice. Every workgroup of the sequence comes to the same result; `writes`
// one of them writes it out.
template <typename T, typename Q>
__device__ __forceinline__ void decide(const VerifyParams& p, VerifySmem& sm, int seq, int begin, int n, bool writes) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) sm.first = n;
  __syncthreads();
  const float t = temperature_of(p, seq);
  float c_hi = 0.f, c_lo = 0.f;
  if (t > 0.f) factor(t, c_hi, c_lo);
  const T* logits = static_cast<const T*>(p.logits);
  const Q* probs = static_cast<const Q*>(p.draft_probs);
  for (int j = wave; j <= n; j += kWaves) {
    const int64_t row = static_cast<int64_t>(begin) + seq + j;
    // the draft's own values, on their way beside the statistics
    int x = -1;
    float u = 0.f, l = 0.f, q = 1.f;
    if (j < n) {
      x = p.draft_tokens[begin + j];
      u = p.accept_u[begin + j];
      if (x >= 0 && x < p.vocab) {
        l = elem<T>::load1(logits + row * p.logits_stride + x);
        if (probs) q = elem<Q>::load1(probs + (static_cast<int64_t>(begin) + j) * p.probs_stride + x);
      }
    }
    const RowStat r = row_stat(p, row, c_hi, c_lo);
    if (lane == 0) {
      if (j < kHeldRows) sm.rows[j] = r;
      if (j < n) {
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
        if (!ok) atomicMin(&sm.first, j);
      }
    }
  }
  __syncthreads();
  const int acc = sm.first;
  if (wave == 0) {
    const int64_t row = static_cast<int64_t>(begin) + seq + acc;
    const RowStat r = acc < kHeldRows ? sm.rows[acc] : row_stat(p, row, c_hi, c_lo);
    if (lane == 0) {
      Choice c;
      c.row = row;
      c.q_row = acc < n && probs ? static_cast<int64_t>(begin) + acc : -1;
      c.draft = acc < n && !probs ? p.draft_tokens[begin + acc] : -1;
      c.column = acc;
      c.m = r.m;
      c.c_hi = c_hi;
      c.c_lo = c_lo;
      c.only = !(r.m > -INFINITY) ? 0 : (t > 0.f ? -1 : r.arg);
      c.inv_s = 1.0 / r.s;
      sm.choice = c;
    }
  }
  if (writes) {
    int32_t* out = p.out + static_cast<int64_t>(seq) * (p.max_drafts + 1);
    for (int i = threadIdx.x; i <= p.max_drafts; i += kThreads)
      if (i != acc) out[i] = i < acc ? p.draft_tokens[begin + i] : -1;
    if (threadIdx.x == 0) p.n_accepted[seq] = acc;
  }
  __syncthreads();
}

// The token: the piece that the border falls into, then the place in it.
template <typename T, typename Q>
__device__ __forceinline__ int pick(const VerifyParams& p, VerifySmem& sm, int seq) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  const Choice c = sm.choice;
  if (wave == 0) {
    double* mass = p.mass + static_cast<int64_t>(seq) * p.n_pieces;
    const PieceStat* st = static_cast<const PieceStat*>(p.stats) + c.row * p.n_pieces;
    // written by this launch's workgroups where something is subtracted (read past this XCD's L2)
    bool residual = c.q_row >= 0 || c.draft >= 0;
    auto piece_mass = [&](int i) {
      if (i >= p.n_pieces) return 0.0;
      if (residual) return __hip_atomic_load(mass + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const PieceStat a = st[i];
      return a.m > -INFINITY ? a.s * static_cast<double>(weight(a.m, c.m, c.c_hi, c.c_lo)) * c.inv_s : 0.0;
    };
    auto total_of = [&]() {
      double s = 0.0;
      for (int i = lane; i < p.n_pieces; i += kWave) s += piece_mass(i);
      return wave_sum_f64(s);
    };
    double total = total_of();
    if (residual && !(total > 0.0)) {
      residual = false;
      total = total_of();
    }
    const double border = static_cast<double>(p.sample_u[seq]) * total;
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
    if (lane == 0) {
      sm.piece = piece >= 0 ? piece : max(last, 0);
      sm.before = piece >= 0 ? before : last_before;
      sm.border = border;
      sm.residual = residual;
      sm.token = INT32_MAX;
      sm.tail = 0;
    }
  }
  __syncthreads();
  const bool residual = sm.residual != 0;
  const double border = sm.border;
  const int64_t first = static_cast<int64_t>(sm.piece) * kVerifyPiece + wave * kWavePiece;
  double w[kSteps][kLaneTokens], own[kSteps], all = 0.0;
#pragma unroll
  for (int k = 0; k < kSteps; k++) {
    masses<T, Q>(p, c, first + (k * kWave + lane) * kLaneTokens, residual, w[k]);
    own[k] = 0.0;
#pragma unroll
    for (int e = 0; e < kLaneTokens; e++) own[k] += w[k][e];
    all += own[k];
  }
  all = wave_sum_f64(all);
  if (lane == 0) sm.sum[wave] = all;
  __syncthreads();
  double run = sm.before;
  for (int i = 0; i < wave; i++) run += sm.sum[i];
  int mine = INT32_MAX, tail = -1;
#pragma unroll
  for (int k = 0; k < kSteps; k++) {
    const double upto = run + wave_scan_f64(own[k]);
    double at = upto - own[k];
    const int i = static_cast<int>(first) + (k * kWave + lane) * kLaneTokens;
#pragma unroll
    for (int e = 0; e < kLaneTokens; e++) {
      at += w[k][e];
      if (w[k][e] > 0.0) {
        if (at > border) mine = min(mine, i + e);
        tail = i + e;
      }
    }
    run = __shfl(upto, kWave - 1, kWave);
  }
  if (mine != INT32_MAX) atomicMin(&sm.token, mine);
  if (tail >= 0) atomicMax(&sm.tail, tail);  // the last token of the piece with any mass
  __syncthreads();
  return sm.token != INT32_MAX ? sm.token : sm.tail;
}

template <typename T, typename Q>
__global__ __launch_bounds__(kThreads) void verify_kernel(VerifyParams p) {
  __shared__ VerifySmem sm;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  const int piece = blockIdx.x, seq = blockIdx.y;
  int32_t* out = p.out + static_cast<int64_t>(seq) * (p.max_drafts + 1);
  int begin, n;
  if (!span_of(p, seq, begin, n)) {
    if (piece == 0) {
      for (int i = threadIdx.x; i <= p.max_drafts; i += kThreads) out[i] = -1;
      if (threadIdx.x == 0) p.n_accepted[seq] = -1;
    }
    return;
  }
  if (piece > 0 && (n == 0 || !(temperature_of(p, seq) > 0.f))) return;  // nothing to subtract
  decide<T, Q>(p, sm, seq, begin, n, piece == 0);
  const Choice& c = sm.choice;
  if (c.only >= 0) {
    if (piece == 0 && threadIdx.x == 0) out[c.column] = c.only;
    return;
  }
  if (c.q_row < 0 && c.draft < 0) {
    if (piece > 0) return;
  } else {
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < kSteps; k++) {
      double w[kLaneTokens];
      masses<T, Q>(p, c, static_cast<int64_t>(piece) * kVerifyPiece + wave * kWavePiece + (k * kWave + lane) * kLaneTokens,
                   true, w);
#pragma unroll
      for (int e = 0; e < kLaneTokens; e++) s += w[e];
    }
    s = wave_sum_f64(s);
    if (lane == 0) sm.sum[wave] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      double all = 0.0;
#pragma unroll
      for (int w = 0; w < kWaves; w++) all += sm.sum[w];
      __hip_atomic_store(p.mass + static_cast<int64_t>(seq) * p.n_pieces + piece, all, __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
      __builtin_amdgcn_s_waitcnt(0);  // the mass is where every XCD reads it before the arrival counts
      sm.last = __hip_atomic_fetch_add(p.arrivals + seq, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == p.n_pieces - 1;
    }
    __syncthreads();
    if (!sm.last) return;
  }
  const int token = pick<T, Q>(p, sm, seq);
  if (threadIdx.x == 0) out[c.column] = token;
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
  return with_dtype(logits_dtype, [&](auto a) {
    return with_dtype(probs_dtype, [&](auto b) {
      using T = decltype(a);
      using Q = decltype(b);
      stats_kernel<T><<<dim3(pieces, static_cast<unsigned>(p.max_drafts + 1), seqs), kThreads, 0, stream>>>(p);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
      verify_kernel<T, Q><<<dim3(pieces, seqs), kThreads, 0, stream>>>(p);
      return hipGetLastError();
    });
  });
}

}  // namespace le
