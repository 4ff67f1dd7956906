// Distillation from a teacher's best tokens: what the forward, the gradient and the one-pass kernel
// share.
//
// The teacher's row is K pairs (token, log-probability); its set of tokens is here called the kept
// tokens, every other token of the vocabulary the tail.
//   p = softmax(x / temperature), q_k = c exp(lp_k), r: the teacher's mass outside the kept tokens
//     bucket:       c = 1,             r = max(0, 1 - sum exp(lp)), 0 up to 2^-20 (rounding of lp)
//     renormalize:  c = 1 / sum exp(lp), r = 0
//   kl = sum_k q_k (log q_k - log p_k) + r (log r - log R),  R = sum of p over the tail
//   accept = sum_k min(p_k, q_k) + min(r, R)
//   ce = log sum exp(x) - x_t (temperature 1)
//   dx_j = g_kl / temperature (p_j (sum q + r) - q_j [j kept] - r p_j / R [j in the tail])
//          + g_ce (softmax(x)_j - [j = t])
//
// R is summed over the tail itself, relative to the tail's own maximum: 1 - sum of the kept p would
// cancel for a student that puts nearly everything on the kept tokens, and terms relative to the
// row's maximum would underflow for one that does so by 90 nats. So the kept tokens are taken out of
// the registers that hold the row (set to -inf) before its maximum and sums are taken, and are added
// from their own K values. In the tail dx_j = e_j w with one factor w per row. The K-term sums are
// in 64 bits: r is a difference of near-equal numbers for a confident teacher, and log q - log p one
// for a student that has learned.
#pragma once

#include "vocab_rows.h"

namespace aspec {
namespace distill {

using namespace vocab;

constexpr int kStats = 8;  // per row: M, S, tail maximum, tail sum, r, c, sum q + r, S at temperature 1
constexpr double kNoTail = 0x1p-20;

// exp and log of the K-term sums in 64 bits: what the library's do in fewer registers (the kernels
// hold a row in theirs).
// exp(x) = 2^k exp(x - k ln2), |x - k ln2| <= 0.35: its series to the 10th power leaves 2e-13.
__device__ __forceinline__ double exp64(float x) {
  const float k = rintf(fminf(fmaxf(x, -800.f), 700.f) * kLog2e);
  const double t = fma(static_cast<double>(k), -0.693147180559945309, static_cast<double>(x));
  double s = 1.;
#pragma unroll
  for (int n = 10; n > 0; --n) s = fma(s, t * (1. / n), 1.);
  return x < -800.f ? 0. : ldexp(s, static_cast<int>(k));
}
// log(x) = (e + log2 m) ln2 with m in [1/2, 1): the hardware's log2 of m is off by 2^-24 at most.
__device__ __forceinline__ double log64(float x) {
  const float e = static_cast<float>(__builtin_amdgcn_frexp_expf(x));
  const double l = static_cast<double>(e) + static_cast<double>(__builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(x)));
  return x == 0.f ? -INFINITY : l * 0.693147180559945309;
}

struct Args {
  const void* x;
  int64_t rows, stride;
  int V, parts, part_chunks, K;
  const int64_t* targets;  // may be null
  int64_t ignore_index;
  const void* tokens;      // [trows][K], 32 or 64 bits
  int tokens64;
  const float* logprobs;   // [trows][K]
  const int64_t* trow;     // per row, may be null
  int64_t trows;
  int renormalize;
  float inv_t;
  float* ce;               // null without targets
  float* kl;
  float* accept;
  int64_t* argmax;         // may be null
  float* stats;            // the forward's may be null
  float* part_sums;        // [rows][parts][4]: tail maximum, S, S1
  uint64_t* part_arg;      // [rows][parts]
  int32_t* status;         // may be null
  const float* g_ce;       // may be null
  const float* g_kl;       // may be null
  void* dx;
  int64_t dx_stride;
};

struct Target {
  int token;   // -1: none
  bool bad;
};

// The kept tokens of a row in LDS, and their chains: entry k hangs in the chain of the thread that
// holds its token.
template <int T>
struct Kept {
  int head[T];
  int next[kMaxTop], token[kMaxTop];
  float x[kMaxTop], lp[kMaxTop], value[kMaxTop + 1];
  double q[kMaxTop];   // exp(lp); 0 for an unused slot
  int poison;          // an index that the row cannot be computed with
  // A used entry's logit and probability, an unused one's absence.
  __device__ __forceinline__ void fill(int k, float logit) {
    x[k] = token[k] >= 0 ? logit : kNegInf;
    q[k] = token[k] >= 0 ? exp64(lp[k]) : 0.;
  }
};

// The teacher's row, or -1.
__device__ __forceinline__ int64_t teacher_row(const Args& a, int64_t row) {
  if (!a.trow) return row;
  const int64_t t = a.trow[row];
  return t < 0 || t >= a.trows ? -1 : t;
}

// Entry k of teacher row t: its token as two words (read alike whatever its type, so that no load
// waits in a branch) and its log-probability. Places that are not there read entry 0 of row 0.
struct RawEntry {
  uint32_t low, high;
  float lp;
};
__device__ __forceinline__ RawEntry load_entry(const Args& a, int64_t t, int k) {
  const int64_t at = max(t, static_cast<int64_t>(0)) * a.K + (k < a.K ? k : 0);
  const auto* words = reinterpret_cast<const uint32_t*>(a.tokens) + (a.tokens64 ? 2 * at : at);
  return RawEntry{words[0], words[a.tokens64], a.logprobs[at]};
}
// The token, -1 where there is none; `bad` where it is out of range.
__device__ __forceinline__ int token_of(const Args& a, int64_t t, int k, const RawEntry& e, bool& bad) {
  if (t < 0 || k >= a.K) return -1;
  const int token = static_cast<int>(e.low);
  const int high = a.tokens64 ? static_cast<int>(e.high) : token >> 31;
  if (high == 0 && token >= 0 && token < a.V) return token;
  bad |= token != -1 || high != -1;
  return -1;
}

__device__ __forceinline__ Target read_target(const Args& a, int64_t row) {
  if (!a.targets) return Target{-1, false};
  const int64_t t = a.targets[row];
  if (t == a.ignore_index) return Target{-1, false};
  if (t < 0 || t >= a.V) return Target{-1, true};
  return Target{static_cast<int>(t), false};
}

// The tail's sums relative to its maximum: at the temperature, and at temperature 1 where both are
// wanted.
struct Tail {
  float M, S, S1;
};
template <bool TWO>
__device__ __forceinline__ Tail merge_wave(const Tail& t, float scale) {
  Tail r;
  r.M = wave_allmax(t.M);
  r.S = wave_allsum(t.S * rebase(t.M, r.M, scale));
  r.S1 = TWO ? wave_allsum(t.S1 * rebase(t.M, r.M, kLog2e)) : r.S;
  return r;
}

__device__ __forceinline__ uint64_t wave_allmax_u64(uint64_t v) {
  for (int off = 32; off > 0; off >>= 1) {
    const uint64_t o = __shfl_xor(v, off);
    v = o > v ? o : v;
  }
  return v;
}

// What the gradient takes from a row's statistics.
struct Factors {
  float base;    // of the tail's exponents
  float w, w1;   // dx_j = w exp2((x - base) scale) + w1 exp2((x - base) log2e) in the tail
  float M, inv_s, inv_s1, gk, gc, mass, c;  // for the kept tokens
  template <bool TWO>
  __device__ __forceinline__ float tail(float x, float scale) const {
    float v = w * fast_exp2((x - base) * scale);
    if constexpr (TWO) v = fmaf(w1, fast_exp2((x - base) * kLog2e), v);
    return v;
  }
  // A kept token with teacher probability q; `target`: it is the row's target too.
  template <bool TWO>
  __device__ __forceinline__ float kept(float x, float q, bool target, float scale) const {
    const float p = fast_exp2((x - M) * scale) * inv_s;
    const float p1 = TWO ? fast_exp2((x - M) * kLog2e) * inv_s1 : p;
    return gk * (mass * p - q) + gc * (p1 - (target ? 1.f : 0.f));
  }
};

template <bool TWO>
__device__ __forceinline__ Factors factors_of(const float (&st)[kStats], float g_kl, float g_ce, float inv_t) {
  const float M = st[0], S = st[1], Mt = st[2], St = st[3], r = st[4], c = st[5], mass = st[6], S1 = st[7];
  Factors f{};
  if (S == 0.f) return f;  // no finite logit: nothing has a probability, nothing a gradient
  const float scale = inv_t * kLog2e;
  f.base = base_of(Mt);
  f.M = M;
  f.inv_s = 1.f / S;
  f.inv_s1 = 1.f / S1;
  f.gk = g_kl * inv_t;
  f.gc = g_ce;
  f.mass = mass;
  f.c = c;
  const float outside = St == 0.f ? 0.f : r / St;
  f.w = f.gk * (mass * rebase(Mt, M, scale) * f.inv_s - outside);
  if constexpr (TWO) f.w1 = g_ce * rebase(Mt, M, kLog2e) * f.inv_s1;
  else f.w += g_ce * rebase(Mt, M, scale) * f.inv_s;
  return f;
}

// The row's results from the tail's sums and the kept entries in LDS, by one wave. Writes the losses
// and statistics, and returns the statistics.
template <bool TWO, typename KeptT>
__device__ __forceinline__ void finish_row(const Args& a, int64_t row, int lane, Tail tail, const KeptT& kept,
                                           const Target& target, float x_target, float (&st)[kStats]) {
  const float scale = a.inv_t * kLog2e;
  const bool poison = kept.poison != 0;
  float MK = kNegInf;
  double Q = 0.;
  int used = 0;
#pragma unroll 1
  for (int k = lane; k < a.K; k += 64)
    if (kept.token[k] >= 0) {
      MK = fmaxf(MK, kept.x[k]);
      Q += kept.q[k];
      ++used;
    }
  Q = wave_allsum_f64(Q);
  used = wave_allsum_u32(used);
  const float M = fmaxf(wave_allmax(MK), tail.M), base = base_of(M);
  float S = 0.f, S1 = 0.f;
#pragma unroll 1
  for (int k = lane; k < a.K; k += 64)
    if (kept.token[k] >= 0) {
      S += fast_exp2((kept.x[k] - base) * scale);
      if constexpr (TWO) S1 += fast_exp2((kept.x[k] - base) * kLog2e);
    }
  const float in_row = tail.S * rebase(tail.M, M, scale);
  S = wave_allsum(S) + in_row;
  S1 = TWO ? wave_allsum(S1) + tail.S1 * rebase(tail.M, M, kLog2e) : S;
  if (poison) S = S1 = __builtin_nanf("");

  double c = 1., r = 0., mass = 0.;
  if (a.renormalize) {
    c = Q > 0. ? 1. / Q : Q == 0. ? 0. : Q;
    mass = Q == 0. ? 0. : 1.;
  } else if (used > 0) {
    r = 1. - Q;
    if (r <= kNoTail) r = 0.;
    mass = Q + r;
  }
  const bool empty = S == 0.f;
  const double inv_t = static_cast<double>(a.inv_t), log_s = log64(S), log_c = log64(static_cast<float>(c));
  double kl = 0.;
  float accept = 0.f;
#pragma unroll 1
  for (int k = lane; k < a.K; k += 64)
    if (kept.token[k] >= 0 && kept.q[k] != 0.) {
      const double q = c * kept.q[k];
      const double log_p = static_cast<double>(kept.x[k] - base) * inv_t - log_s;
      kl += q * (static_cast<double>(kept.lp[k]) + log_c - log_p);
      accept += fminf(fast_exp2((kept.x[k] - base) * scale) / S, static_cast<float>(q));
    }
  kl = wave_allsum_f64(kl);
  accept = wave_allsum(accept);
  if (r > 0.) {
    const double log_tail = tail.S == 0.f ? -INFINITY
                                          : static_cast<double>(tail.M - base) * inv_t +
                                                log64(tail.S) - log_s;
    kl += r * (log64(static_cast<float>(r)) - log_tail);
    accept += fminf(static_cast<float>(r), in_row / S);
  }
  accept = fminf(accept, 1.f);  // but for the rounding of the log-probabilities it is
  if (empty) {
    kl = mass > 0. ? static_cast<double>(INFINITY) : 0.;
    accept = 0.f;
  }
  if (S != S) kl = accept = __builtin_nanf("");  // fminf skips a NaN
  if (used == 0 || mass == 0.) kl = accept = 0.f;
  if (poison) kl = accept = __builtin_nanf("");
  st[0] = M;
  st[1] = S;
  st[2] = tail.M;
  st[3] = poison ? __builtin_nanf("") : tail.S;
  st[4] = static_cast<float>(r);
  st[5] = static_cast<float>(c);
  st[6] = static_cast<float>(mass);
  st[7] = S1;
  if (lane == 0) {
    a.kl[row] = static_cast<float>(kl);
    a.accept[row] = accept;
    if (a.targets) {
      float ce = 0.f;
      if (target.token >= 0) ce = empty ? INFINITY : static_cast<float>(log64(S1) - static_cast<double>(x_target - base));
      if (target.bad) {
        ce = __builtin_nanf("");
        report(a.status, kBadTarget);
      }
      a.ce[row] = ce;
    }
    if (a.stats) {
      float4* o = reinterpret_cast<float4*>(a.stats + row * kStats);
      o[0] = make_float4(st[0], st[1], st[2], st[3]);
      o[1] = make_float4(st[4], st[5], st[6], st[7]);
    }
  }
}

// The forward of one part of a row (GRAD: of a whole row, then its gradient from the registers that
// hold it).
template <typename E, int T, int NV, bool TWO, bool GRAD>
__device__ __forceinline__ void forward_unit(const Args& a, int64_t unit, Kept<T>& kept, float (&s_m)[T / 64],
                                             float (&s_s)[T / 64], float (&s_s1)[T / 64], uint64_t& s_arg,
                                             Factors& s_factors) {
  constexpr int W = T / 64;
  using P = Part<E, T, NV>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float scale = a.inv_t * kLog2e;
  const int64_t row = a.parts == 1 ? unit : unit / a.parts;
  const int part = a.parts == 1 ? 0 : static_cast<int>(unit - row * a.parts);
  const auto* x = reinterpret_cast<const typename E::bits*>(a.x) + row * a.stride;
  auto* dx = reinterpret_cast<typename E::bits*>(a.dx) + row * a.dx_stride;
  const RowCut cut = RowCut::at<E>(GRAD ? static_cast<const void*>(dx) : x, a.V);

  // What the row's end needs is read now, so that no load of its own is waited for there: the teacher's
  // entries by the first wave (their logits are on the way while the row is reduced), the target and
  // the weights as scalars.
  const int64_t trow = teacher_row(a, row);
  const Target target = read_target(a, row);
  const typename E::bits raw_target = x[max(target.token, 0)];
  float g_kl = 0.f, g_ce = 0.f;
  if constexpr (GRAD) {
    if (a.g_kl) g_kl = a.g_kl[row];
    if (a.g_ce) g_ce = a.g_ce[row];
  }
  RawEntry entry[2];
  if (wave == 0) {
    entry[0] = load_entry(a, trow, lane);
    entry[1] = load_entry(a, trow, lane + 64);
  }
  P p;
  p.load(x, cut, part, a.part_chunks);
  kept.head[threadIdx.x] = -1;
  if (threadIdx.x == 0) {
    kept.poison = 0;
    s_arg = 0;
  }
  __syncthreads();
  typename E::bits raw[2] = {0, 0};
  if (wave == 0) {
    bool bad = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = lane + 64 * h;
      const int token = token_of(a, trow, k, entry[h], bad);
      raw[h] = x[max(token, 0)];
      if (k < a.K) {
        int owner = 0;
        if (token >= 0 && P::place(cut, part, a.part_chunks, token, owner) >= 0)
          kept.next[k] = atomicExch(&kept.head[owner], k);
        kept.token[k] = token;
        kept.lp[k] = entry[h].lp;
      }
    }
    if ((__any(bad) || trow < 0) && lane == 0) {
      kept.poison = 1;
      report(a.status, trow < 0 ? kBadTeacherRow : kBadTeacherToken);
    }
  }
  __syncthreads();
  p.arrive();
  // ---- the kept tokens leave the registers
  for (int k = kept.head[threadIdx.x]; k >= 0; k = kept.next[k]) {
    int owner;
    p.knock_out(P::place(cut, part, a.part_chunks, kept.token[k], owner));
    for (int j = kept.next[k]; j >= 0; j = kept.next[j])
      if (kept.token[j] == kept.token[k]) {
        kept.poison = 1;
        report(a.status, kRepeatedToken);
      }
  }
  // ---- the tail's maximum and sums
  const float m = p.largest();
  const float wm = wave_allmax(m), wbase = base_of(wm);
  p.forget();
  float S = 0.f, S1 = 0.f;
  p.each_value([&](float v) {
    S += fast_exp2((v - wbase) * scale);
    if constexpr (TWO) S1 += fast_exp2((v - wbase) * kLog2e);
  });
  p.forget();
  S = wave_allsum(S);
  if constexpr (TWO) S1 = wave_allsum(S1);
  if (lane == 0) {
    s_m[wave] = wm;
    s_s[wave] = S;
    s_s1[wave] = S1;
  }
  __syncthreads();
  if (a.argmax) {
    // the largest logit of the tail, NaN above all, ties to the lower index
    float top = s_m[0];
    bool nan = s_s[0] != s_s[0];
    for (int w = 1; w < W; ++w) {
      top = fmaxf(top, s_m[w]);
      nan |= s_s[w] != s_s[w];
    }
    if (m == top || nan) {
      uint64_t best = 0;
      p.each([&](float v, int at) {
        if (v == top || v != v) {
          const uint64_t rank = ranked(order_key(v), at);
          best = rank > best ? rank : best;
        }
      });
      atomicMax(reinterpret_cast<unsigned long long*>(&s_arg), static_cast<unsigned long long>(best));
    }
    p.forget();
    __syncthreads();
  }
  if (wave == 0) {
    Tail t{kNegInf, 0.f, 0.f};
    if (lane < W) t = Tail{s_m[lane], s_s[lane], s_s1[lane]};
    t = merge_wave<TWO>(t, scale);
    if (a.parts > 1) {
      if (lane == 0) {
        const float poison = kept.poison ? __builtin_nanf("") : 0.f;
        *reinterpret_cast<float4*>(a.part_sums + unit * 4) = make_float4(t.M, t.S + poison, t.S1, 0.f);
        a.part_arg[unit] = s_arg;
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (lane + 64 * h < a.K) kept.fill(lane + 64 * h, E::widen(raw[h]));
      const float x_target = E::widen(raw_target);
      float st[kStats];
      finish_row<TWO>(a, row, lane, t, kept, target, x_target, st);
      if (a.argmax) {
        uint64_t best = s_arg;
#pragma unroll 1
        for (int k = lane; k < a.K; k += 64)
          if (kept.token[k] >= 0) {
            const uint64_t rank = ranked(order_key(kept.x[k]), kept.token[k]);
            best = rank > best ? rank : best;
          }
        best = wave_allmax_u64(best);
        if (lane == 0) a.argmax[row] = ranked_index(best);
      }
      if constexpr (GRAD) {
        // a bad target's NaN takes the whole row of the gradient
        const float gc = target.bad ? __builtin_nanf("") : target.token >= 0 ? g_ce : 0.f;
        const Factors f = factors_of<TWO>(st, g_kl, gc, a.inv_t);
#pragma unroll 1
        for (int k = lane; k < a.K; k += 64)
          if (kept.token[k] >= 0)
            kept.value[k] = st[1] == 0.f ? 0.f
                                         : f.template kept<TWO>(kept.x[k], static_cast<float>(kept.q[k]) * f.c,
                                                                kept.token[k] == target.token, scale);
        if (lane == 0) {
          kept.value[kMaxTop] = target.token < 0 || st[1] == 0.f ? 0.f : f.template tail<TWO>(x_target, scale) - gc;
          s_factors = f;
        }
      }
    }
  }
  if constexpr (GRAD) {
    __syncthreads();
    const Factors f = s_factors;
    p.store(dx, [&](float v) { return f.template tail<TWO>(v, scale); });
    // behind the dense values, by the thread that wrote those
    bool kept_target = false;
    for (int k = kept.head[threadIdx.x]; k >= 0; k = kept.next[k]) {
      dx[kept.token[k]] = E::narrow(kept.value[k]);
      kept_target |= kept.token[k] == target.token;
    }
    int owner = -1;
    if (target.token >= 0) P::place(cut, part, a.part_chunks, target.token, owner);
    if (owner == static_cast<int>(threadIdx.x) && !kept_target) dx[target.token] = E::narrow(kept.value[kMaxTop]);
  }
}

}  // namespace distill
}  // namespace aspec
