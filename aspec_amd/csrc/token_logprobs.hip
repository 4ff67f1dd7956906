// Log-probabilities of given tokens, entropy and the K best alternatives of rows of logits, and
// their gradient.
//
//   z = x / temperature, m = max z, S = sum exp(z - m), logp_j = z_j - m - log S, p = exp(logp)
//   logprob = logp_t,  entropy = log S - sum exp(z - m) (z - m) / S   (two terms >= 0: no cancellation)
//   dx_j = 1/temperature * ( -G p_j - g_H p_j (logp_j + H) + g_t [j = t] + sum_i g_i [j = top_i] ),
//   G = g_t + sum_i g_i
//
// HBM-bound: the forward reads each logit once, the backward reads it once and writes the gradient
// once. A row (or a part of a long one) lies in registers while its maximum, sums and best tokens
// are taken. 8192 x 32000 bf16: forward 92 us back to back (5.7 TB/s; leaving out the exponentials or
// the entropy does not shorten it) and 111-130 behind 524 MB of gradient writes, backward 171 us
// (6.1 TB/s read and written). Holding the next row's loads in flight as well was slower (113 us against
// 128: 95 registers leave two workgroups to a CU in place of four).
//
// The K best: at least K tokens are >= the K-th largest of the maxima of groups of threads, and few
// more than K of them are unless the large ones share groups. One wave finds that bound by bisection
// over the maxima's ordered bits; the tokens at or above it go to a list in LDS, and each one's
// place is the number of list entries above it. Order is by logit, ties by index: (ordered bits,
// ~index) as one 64-bit number, no two alike. A list that overflows (long runs of equal logits,
// large ones that share threads) is replaced by exactly the K best: the K-th largest value, found by
// bisection with counts over the part, and its ties in order.
// 4096 x 32000 bf16 with the 64 best: 61 us against 46 without them, 295 MB read (the row, and the
// chunks of the listed tokens again). What is left is the chain behind a row's last load (four
// barriers, the bisection, the list, the places; about 4 us), in which its workgroup asks for nothing,
// with four workgroups to a CU; asking for the next row ahead of it costs the registers of two of the
// four, and was slower (95 us). 8192 x 32000: random 87 us without alternatives, 102 with 1, 110 with
// 20, 117 with 64, 155 with 128; 64 of rows that are all equal 400, of rows masked but for 40 tokens
// 434, of ascending rows (the list overflows, and 64-fold ties) 1066.
#include "vocab_rows.h"

namespace aspec {
namespace {

using namespace vocab;

constexpr int kStats = 4;       // per row: maximum, S, D / S, 0 (16 bytes)
constexpr int kList = 512;      // tokens at or above the bound that are ranked without a search

struct FwdArgs {
  const void* x;
  int64_t rows, stride;
  int V, parts, part_chunks, K;
  const int64_t* ids;
  int64_t ignore_index;
  float inv_t;
  float* logprobs;
  float* entropy;
  float* top_logprobs;
  int64_t* top_indices;
  float* stats;
  float* part_sums;   // [rows][parts][3]: maximum, S, D
  uint64_t* part_top; // [rows][parts][K], descending, 0 behind a part's last token
  int32_t* status;
};

struct BwdArgs {
  const void* x;
  int64_t rows, stride;
  int V, parts, part_chunks, K;
  const int64_t* ids;
  int64_t ignore_index;
  float inv_t;
  const int64_t* top_indices;
  const float* stats;
  const float* g_logprob;
  const float* g_entropy;
  const float* g_top;
  void* dx;
  int64_t dx_stride;
};

// S and D = sum e log2 e over terms relative to m (in units of log2).
struct Sums {
  float m, S, D;
  // Both relative to M >= m.
  __device__ __forceinline__ Sums at(float M, float scale) const {
    const float f = rebase(m, M, scale);
    const float shift = m == kNegInf ? 0.f : (m - M) * scale;
    // S = 0: no term, whatever the shift
    return Sums{M, S * f, S == 0.f ? 0.f : f * fmaf(S, fmaxf(shift, -1000.f), D)};
  }
};

// Merges the sums of the first n lanes (others hold m = -inf, S = D = 0).
__device__ __forceinline__ Sums merge_wave(const Sums& s, float scale) {
  Sums r = s.at(wave_allmax(s.m), scale);
  r.S = wave_allsum(r.S);
  r.D = wave_allsum(r.D);
  return r;
}

struct RowResult {
  float M, inv_t, log_s;
  bool empty;
  __device__ __forceinline__ float logprob(float x) const {
    return empty ? kNegInf : (x - M) * inv_t - log_s;
  }
};

// The row's results from its sums, written by one lane; `id` and its logit are read by the caller.
__device__ __forceinline__ RowResult finish_row(const FwdArgs& a, int64_t row, const Sums& s, bool writer,
                                                int64_t id, float at_id) {
  const bool empty = s.S == 0.f;  // no finite logit: nothing has a probability
  const float log_s = logf(s.S);
  const RowResult r{s.m, a.inv_t, log_s, empty};
  if (writer) {
    const float entropy = empty ? 0.f : log_s - kLn2 * s.D / s.S;
    a.entropy[row] = entropy;
    if (a.stats)
      *reinterpret_cast<float4*>(a.stats + row * kStats) = make_float4(s.m, s.S, empty ? 0.f : s.D / s.S, 0.f);
    if (a.ids) {
      float lp = 0.f;
      if (id != a.ignore_index) {
        lp = r.logprob(at_id);
        if (id < 0 || id >= a.V) {
          lp = __builtin_nanf("");
          report(a.status, kBadTokenId);
        }
      }
      a.logprobs[row] = lp;
    }
  }
  return r;
}

// The given token, and its logit's bits; ignore_index (logit 0 of the row) where there is none. Read
// by every lane alike, as scalars.
template <typename E>
__device__ __forceinline__ int64_t given_token(const FwdArgs& a, int64_t row, typename E::bits& raw) {
  const int64_t id = a.ids ? a.ids[row] : a.ignore_index;
  raw = reinterpret_cast<const typename E::bits*>(a.x)[row * a.stride + (id >= 0 && id < a.V ? id : 0)];
  return id;
}

// Block-wide count of what a thread counted; every thread gets it. `scratch` holds one word per wave.
template <int T>
__device__ __forceinline__ uint32_t block_count(uint32_t n, uint32_t* scratch) {
  n = wave_allsum_u32(n);
  if constexpr (T == 64) return n;
  __syncthreads();  // the last count has been read
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = n;
  __syncthreads();
  uint32_t sum = 0;
  for (int w = 0; w < T / 64; ++w) sum += scratch[w];
  return sum;
}

// Of what the threads counted: how much the lower lanes of the wave did.
__device__ __forceinline__ uint32_t wave_prefix(uint32_t n) {
  const int lane = threadIdx.x & 63;
  uint32_t sum = n;
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const uint32_t lower = __shfl_up(sum, off);
    if (lane >= off) sum += lower;
  }
  return sum - n;
}
// Adds what the lower waves counted, and returns the block's count; `scratch` holds a word per wave.
template <int T>
__device__ __forceinline__ uint32_t block_prefix(uint32_t& before, uint32_t n, uint32_t* scratch) {
  const int wave = threadIdx.x >> 6;
  __syncthreads();  // the last count has been read
  if ((threadIdx.x & 63) == 63) scratch[wave] = before + n;
  __syncthreads();
  uint32_t all = 0;
  for (int w = 0; w < T / 64; ++w) {
    if (w < wave) before += scratch[w];
    all += scratch[w];
  }
  return all;
}

template <typename E, int T, int NV, bool TOP>
__global__ __launch_bounds__(T, 8) void token_logprobs_kernel(FwdArgs a) {
  using P = Part<E, T, NV>;
  constexpr int W = T / 64;
  __shared__ float s_m[W], s_S[W], s_D[W];
  __shared__ uint16_t s_reach[TOP ? T * NV : 1];  // chunks whose maximum reaches the bound
  __shared__ uint32_t s_reached;
  __shared__ uint32_t s_best[TOP ? T : 1], s_count[W];
  __shared__ uint32_t s_n, s_bound, s_high;
  __shared__ float s_row[4];
  __shared__ __attribute__((aligned(16))) uint64_t s_list[TOP ? kList : 2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float scale = a.inv_t * kLog2e;
  const int64_t unit = unit_of_block();
  if (unit >= a.rows * a.parts) return;
  const int64_t row = a.parts == 1 ? unit : unit / a.parts;
  const int part = a.parts == 1 ? 0 : static_cast<int>(unit - row * a.parts);
  const auto* x = reinterpret_cast<const typename E::bits*>(a.x) + row * a.stride;
  typename E::bits raw_id;  // read before the row, so that nothing waits for it at the end
  const int64_t id = given_token<E>(a, row, raw_id);
  const RowCut cut = RowCut::at<E>(x, a.V);
  P p;
  p.load(x, cut, part, a.part_chunks);

  p.arrive();
  // ---- maximum and sums
  const float m = p.largest();
  const float wm = wave_allmax(m), base = base_of(wm);
  p.forget();
  float S = 0.f, D = 0.f;
  p.each_value([&](float v) {
    const float d = (v - base) * scale, e = fast_exp2(d);
    S += e;
    D = fmaf(e, fmaxf(d, -200.f), D);  // e = 0 there; -inf would make it NaN
  });
  p.forget();
  S = wave_allsum(S);
  D = wave_allsum(D);
  if (lane == 0) {
    s_m[wave] = wm;
    s_S[wave] = S;
    s_D[wave] = D;
  }
  if constexpr (TOP) {
    // at most the key of the thread's largest token (the maximum skips a NaN, the highest key)
    s_best[threadIdx.x] = order_key(m);
    if (threadIdx.x == 0) s_n = s_reached = 0;
  }
  __syncthreads();
  RowResult r{0.f, 0.f, 0.f, false};
  if (wave == 0) {
    Sums s{kNegInf, 0.f, 0.f};
    if (lane < W) s = Sums{s_m[lane], s_S[lane], s_D[lane]};
    s = merge_wave(s, scale);
    if (a.parts == 1) {
      r = finish_row(a, row, s, lane == 0, id, E::widen(raw_id));
      if constexpr (TOP) {
        if (lane == 0) {
          s_row[0] = r.M;
          s_row[1] = r.log_s;
          s_row[2] = r.empty ? 1.f : 0.f;
        }
      }
    } else if (lane == 0) {
      float* o = a.part_sums + unit * 3;
      o[0] = s.m;
      o[1] = s.S;
      o[2] = s.D;
    }
  }
  if constexpr (TOP) {
    // ---- the bound: the K-th largest maximum of groups of threads, or a little below it. Four times as
    // many groups as tokens wanted keep the list short (G groups: G ln(G / (G - K)) tokens of a random
    // row reach it) and the wave's counts few. The first wave is busy with the sums.
    if (wave == (W > 1 ? 1 : 0)) {
      uint32_t key[W], low = 0xffffffffu, high = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        key[w] = s_best[w * 64 + lane];
        high = max(high, key[w]);
      }
      high = wave_allmax_u32(high);
      const uint32_t K = a.K, enough = K + K / 8 + 4;
      const auto search = [&](const auto& group) {
        constexpr int G = sizeof(group) / sizeof(uint32_t);
#pragma unroll
        for (int w = 0; w < G; ++w) low = min(low, group[w]);
        low = wave_allmin(low);
        uint32_t top = high;
        while (low < top) {  // count(>= low) >= K throughout
          const uint32_t mid = low + (top - low) / 2 + ((top - low) & 1);
          uint32_t n = 0;
#pragma unroll
          for (int w = 0; w < G; ++w) n += __popcll(__ballot(group[w] >= mid));
          if (n >= K) {
            low = mid;
            if (n <= enough) break;
          } else {
            top = mid - 1;
          }
        }
      };
      const auto search_groups = [&](auto held) {
        constexpr int G = held.value;
        uint32_t group[G];
#pragma unroll
        for (int w = 0; w < W; ++w) group[w % G] = w < G ? key[w] : max(group[w % G], key[w]);
        search(group);
      };
      if (W == 1 && K > 32) {
        // the groups are half chunks, of which this wave holds the row's all: the 64 maxima alone leave the
        // whole row to be listed (65536 x 2000 bf16 with 128 wanted: 309 us for 1082). With fewer half
        // chunks than tokens wanted every token is listed too.
        uint32_t group[2 * NV];
#pragma unroll
        for (int h = 0; h < 2 * NV; ++h) group[h] = order_key(p.largest_of_half(h));
        search(group);
      } else if (W > 1 && K <= 16) search_groups(std::integral_constant<int, 1>{});
      else if (W > 2 && K <= 32) search_groups(std::integral_constant<int, W < 2 ? W : 2>{});
      else if (W > 4 && K <= 64) search_groups(std::integral_constant<int, W < 4 ? W : 4>{});
      else search_groups(std::integral_constant<int, W>{});
      if (lane == 0) {
        s_bound = low;
        s_high = high;
      }
    }
    __syncthreads();
    // ---- the list: the few chunks whose largest token reaches the bound are dealt out to all threads,
    // which read them again and list what reaches it
    const uint32_t bound = s_bound;
    const float bound_value = key_value(bound);  // a NaN bound lists every token
    const int chunks = P::chunks_in(cut, part, a.part_chunks);
    const auto append = [&](float v, int at) {
      const uint32_t slot = atomicAdd(&s_n, 1u);
      if (slot < kList) s_list[slot] = ranked(order_key(v), at);
    };
    if (!(m < bound_value) || S != S) {
      uint32_t reach = S != S ? (1u << NV) - 1 : p.chunks_reaching(bound_value);  // the maxima skip a NaN
      for (; reach; reach &= reach - 1)
        s_reach[atomicAdd(&s_reached, 1u)] = static_cast<uint16_t>(threadIdx.x + __builtin_ctz(reach) * T);
    }
    if (p.edge_at >= 0 && !(p.edge < bound_value)) append(p.edge, p.edge_at);
    __syncthreads();
    const int tasks = s_reached;
    for (int task = threadIdx.x; task < tasks; task += T) {
      if (*static_cast<volatile uint32_t*>(&s_n) > kList) break;  // the list is lost already
      const int c = s_reach[task];
      if (c >= chunks) continue;
      const int first = P::index_of(cut, part, a.part_chunks, c);
      const uint4 w = load16<E>(x, first);
      uint32_t hits = 0;
#pragma unroll
      for (int i = 0; i < P::CH; ++i) hits |= element<E>(w, i) < bound_value ? 0u : 1u << i;
      for (; hits; hits &= hits - 1) {
        const int i = __builtin_ctz(hits);
        append(element_at<E>(w, i), first + i);
      }
    }
    __syncthreads();
    if (s_n > kList) {
      // ---- exactly the K best: the K-th largest value by bisection, with counts over the part, which
      // is read again (from L2) for each; then its ties in the order of their indices
      constexpr int kDrop = E::kKeyDrop;
      const uint32_t K = a.K;
      const auto key = [](float v) { return order_key(v) >> kDrop; };
      const auto hits = [&](uint4 w, auto pred) {  // one bit for each element of a chunk
        uint32_t h = 0;
#pragma unroll
        for (int i = 0; i < P::CH; ++i) h |= pred(key(element<E>(w, i))) ? 1u << i : 0u;
        return h;
      };
      const auto count = [&](auto pred) {
        uint32_t n = p.edge_at >= 0 && pred(key(p.edge)) ? 1 : 0;
#pragma unroll 1
        for (int c = threadIdx.x; c < chunks; c += T)
          n += __popc(hits(load16<E>(x, P::index_of(cut, part, a.part_chunks, c)), pred));
        return block_count<T>(n, s_count);
      };
      uint32_t low = bound >> kDrop, high = s_high >> kDrop;  // count(>= low) >= K throughout
      uint32_t larger_ones = count([&](uint32_t k) { return k > low; });
      if (larger_ones >= K) {
        if (count([&](uint32_t k) { return k > high; }) >= K) {  // NaN, which the maxima skip
          low = high;
          high = 0xffffffffu >> kDrop;
        }
        while (low < high) {
          const uint32_t mid = low + (high - low) / 2 + ((high - low) & 1);
          if (count([&](uint32_t k) { return k >= mid; }) >= K) low = mid;
          else high = mid - 1;
        }
        larger_ones = count([&](uint32_t k) { return k > low; });
      }
      const auto above = [&](uint32_t k) { return k > low; };
      const auto tie = [&](uint32_t k) { return k == low; };
      const uint32_t ties = K - larger_ones;
      uint32_t seen = 0;
      __syncthreads();
      if (threadIdx.x == 0) s_n = 0;
      __syncthreads();
      // Everything above; of the ties the first ones: the edge before the chunks, then T chunks at a
      // time, then the edge behind them, each thread knowing the number of ties before its own.
      const auto ties_before = [&](uint32_t tied) {  // and `seen` moves past these threads
        uint32_t before = wave_prefix(tied);
        const uint32_t all = block_prefix<T>(before, tied, s_count);
        before += seen;
        seen += all;
        return before;
      };
      const bool edge = p.edge_at >= 0, in_front = edge && p.edge_at < cut.lead;
      const bool edge_tie = edge && tie(key(p.edge));
      if (edge && above(key(p.edge))) append(p.edge, p.edge_at);
      if (ties_before(in_front && edge_tie ? 1 : 0) < ties && in_front && edge_tie) append(p.edge, p.edge_at);
#pragma unroll 1
      for (int c0 = 0; c0 < chunks; c0 += T) {
        const int c = c0 + static_cast<int>(threadIdx.x), first = P::index_of(cut, part, a.part_chunks, c);
        uint4 w = {};
        uint32_t larger = 0, tied = 0;
        if (c < chunks) {
          w = load16<E>(x, first);
          larger = hits(w, above);
          tied = hits(w, tie);
        }
        const uint32_t before = ties_before(__popc(tied));
        for (uint32_t left = larger | tied; left; left &= left - 1) {
          const int i = __builtin_ctz(left);
          const bool is_tie = (tied >> i) & 1;
          if (!is_tie || before + __popc(tied & ((1u << i) - 1)) < ties) append(element_at<E>(w, i), first + i);
        }
      }
      if (ties_before(!in_front && edge_tie ? 1 : 0) < ties && !in_front && edge_tie) append(p.edge, p.edge_at);
      __syncthreads();
    }
    int n = s_n;
    if (n > a.K + a.K / 2 + 32) {
      // ---- a list much longer than wanted (few groups for many tokens) is thinned out first, by the K-th
      // largest value in it or one a little below: the places take n^2 steps. 65536 x 500 bf16 with 64
      // wanted, where every token was listed: 189 us for 1783.
      __syncthreads();
      if (wave == 0) {
        constexpr int H = kList / 64;
        uint32_t key[H];
#pragma unroll
        for (int h = 0; h < H; ++h)
          key[h] = lane + 64 * h < n ? static_cast<uint32_t>(s_list[lane + 64 * h] >> 32) >> E::kKeyDrop : 0;
        const uint32_t K = a.K, enough = K + K / 4 + 8;
        uint32_t low = 0, top = ~0u >> E::kKeyDrop;
        while (low < top) {  // count(>= low) >= K throughout
          const uint32_t mid = low + (top - low) / 2 + ((top - low) & 1);
          uint32_t count = 0;
#pragma unroll
          for (int h = 0; h < H; ++h) count += __popcll(__ballot(key[h] >= mid));
          if (count >= K) {
            low = mid;
            if (count <= enough) break;
          } else {
            top = mid - 1;
          }
        }
        int kept = 0;
#pragma unroll
        for (int h = 0; h < H; ++h) {  // an entry moves to a place that has been read
          const bool keep = lane + 64 * h < n && key[h] >= low;
          const uint64_t entry = s_list[lane + 64 * h], lanes = __ballot(keep);
          if (keep) s_list[kept + __popcll(lanes & ((uint64_t{1} << lane) - 1))] = entry;
          kept += __popcll(lanes);
        }
        if (lane == 0) s_n = kept;
      }
      __syncthreads();
      n = s_n;
    }
    // ---- each entry's place; at least K entries, or all of a part that has fewer
    const RowResult rr{s_row[0], a.inv_t, s_row[1], s_row[2] != 0.f};
    for (int base = 0; base < n; base += T / 4) {  // four threads to an entry
      const int i = base + static_cast<int>(threadIdx.x >> 2);
      const uint64_t mine = i < n ? s_list[i] : 0;
      uint32_t place = 0;
      for (int j = 2 * (threadIdx.x & 3); j < n; j += 8) {
        const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(s_list + j);
        place += (two.x > mine ? 1u : 0u) + (j + 1 < n && two.y > mine ? 1u : 0u);
      }
      place += dpp_u32<0xB1>(place);
      place += dpp_u32<0x4E>(place);
      if (i >= n || (threadIdx.x & 3) != 0 || place >= static_cast<uint32_t>(a.K)) continue;
      if (a.parts == 1) {
        a.top_logprobs[row * a.K + place] = rr.logprob(ranked_value(mine));
        a.top_indices[row * a.K + place] = ranked_index(mine);
      } else {
        a.part_top[unit * a.K + place] = mine;
      }
    }
    if (a.parts > 1)
      for (int i = n + threadIdx.x; i < a.K; i += T) a.part_top[unit * a.K + i] = 0;
  }
}

// Joins the parts of long rows: the sums by one wave, the ordered lists pairwise. An entry's place
// in a pair's merged list is its own place plus the number of the other list's entries above it (a
// binary search); entries past K are dropped.
// The lists take parts * K * 12 bytes of LDS (48 KB at most), and a wave does where they are short, so
// that many rows fit a CU: 1536 rows of ten lists of 8 take 10 us so, 14 with LDS for the longest.
template <typename E, int T>
__global__ __launch_bounds__(T) void token_logprobs_join_kernel(FwdArgs a) {
  extern __shared__ uint64_t s_lists[];
  uint64_t *const s_a = s_lists, *const s_b = s_lists + a.parts * a.K;
  __shared__ float s_row[4];
  const int lane = threadIdx.x & 63;
  const float scale = a.inv_t * kLog2e;
  const int K = a.K;
  const int64_t row = unit_of_block();
  if (row >= a.rows) return;
  // all the reads before the first wait
  typename E::bits raw_id;
  const int64_t id = given_token<E>(a, row, raw_id);
  const float* o = a.part_sums + (row * a.parts + min(lane, a.parts - 1)) * 3;
  Sums s{o[0], o[1], o[2]};
  for (int i = threadIdx.x; i < a.parts * K; i += T) s_a[i] = a.part_top[row * a.parts * K + i];
  if (threadIdx.x < 64) {
    if (lane >= a.parts) s = Sums{kNegInf, 0.f, 0.f};
    s = merge_wave(s, scale);
    const RowResult r = finish_row(a, row, s, lane == 0, id, E::widen(raw_id));
    if (lane == 0) {
      s_row[0] = r.M;
      s_row[1] = r.log_s;
      s_row[2] = r.empty ? 1.f : 0.f;
    }
  }
  __syncthreads();
  uint64_t *from = s_a, *to = s_b;
  for (int lists = a.parts; lists > 1; lists = (lists + 1) / 2) {
    for (int i = threadIdx.x; i < lists * K; i += T) {
      const int list = i / K, at = i - list * K, other = list ^ 1;
      const uint64_t mine = from[i];
      int place = at;
      if (other < lists) {
        // entries of the other list before this one: larger, or equal (both 0) in the left list
        const uint64_t* o = from + other * K;
        int lo = 0, hi = K;
        while (lo < hi) {
          const int mid = (lo + hi) / 2;
          if (list & 1 ? o[mid] >= mine : o[mid] > mine) lo = mid + 1;
          else hi = mid;
        }
        place += lo;
      }
      if (place < K) to[(list / 2) * K + place] = mine;
    }
    __syncthreads();
    uint64_t* t = from;
    from = to;
    to = t;
  }
  const RowResult r{s_row[0], a.inv_t, s_row[1], s_row[2] != 0.f};
  for (int i = threadIdx.x; i < K; i += T) {
    a.top_logprobs[row * K + i] = r.logprob(ranked_value(from[i]));
    a.top_indices[row * K + i] = ranked_index(from[i]);
  }
}

// Gradient: dense over a part, then the few elements that carry a token of their own, written
// behind the dense values by the thread that wrote those.
template <typename E, int T, int NV, bool ENTROPY>
__global__ __launch_bounds__(T, 8) void token_logprobs_bwd_kernel(BwdArgs a) {
  using P = Part<E, T, NV>;
  __shared__ int s_head[T];
  __shared__ int s_next[kMaxTop], s_token[kMaxTop];
  __shared__ float s_value[kMaxTop], s_lost;
  const float scale = a.inv_t * kLog2e;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t unit = unit_of_block();
  if (unit >= a.rows * a.parts) return;
  const int64_t row = a.parts == 1 ? unit : unit / a.parts;
  const int part = a.parts == 1 ? 0 : static_cast<int>(unit - row * a.parts);
  const auto* x = reinterpret_cast<const typename E::bits*>(a.x) + row * a.stride;
  auto* dx = reinterpret_cast<typename E::bits*>(a.dx) + row * a.dx_stride;
  const RowCut cut = RowCut::at<E>(dx, a.V);
  // the given token, with its gradient, and the alternatives: read before the row
  int given = -1;
  float g_given = 0.f;
  if (a.ids && a.g_logprob && a.ids[row] != a.ignore_index) {
    const int64_t id = a.ids[row];
    if (id >= 0 && id < a.V) given = static_cast<int>(id);
    g_given = given >= 0 ? a.g_logprob[row] : __builtin_nanf("");  // the forward's check has the error
  }
  const typename E::bits raw_given = x[max(given, 0)];
  const float4 st = *reinterpret_cast<const float4*>(a.stats + row * kStats);
  const bool empty = st.y == 0.f;  // nothing has a probability, nothing a gradient
  const float base = base_of(st.x), inv_s = empty ? 0.f : 1.f / st.y;
  const float gh = ENTROPY && !empty ? a.g_entropy[row] : 0.f;
  int64_t token[2];
  float g[2];
  const bool top = a.K > 0;
  if (top && wave == 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t at = row * a.K + min(lane + 64 * h, a.K - 1);
      token[h] = a.top_indices[at];
      g[h] = a.g_top[at];
    }
  }
  P p;
  p.load(x, cut, part, a.part_chunks);
  float lost = g_given;  // G
  if (top) {
    s_head[threadIdx.x] = -1;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = lane + 64 * h;
        if (k >= a.K) g[h] = 0.f;
        const int t = k < a.K && token[h] >= 0 && token[h] < a.V ? static_cast<int>(token[h]) : -1;
        int owner = 0;
        if (t >= 0 && P::place(cut, part, a.part_chunks, t, owner) >= 0) {
          s_next[k] = atomicExch(&s_head[owner], k);
          s_token[k] = t;
          s_value[k] = g[h];
        }
      }
      lost += wave_allsum(g[0] + g[1]);
      if (lane == 0) s_lost = lost;
    }
    __syncthreads();
    lost = s_lost;
  }
  // logp + H = ln2 (d - D / S), so dx = e (u + v d) with e = exp2(d)
  const float v = -gh * kLn2 * inv_s * a.inv_t;
  const float u = empty ? 0.f : (gh * kLn2 * st.z - lost) * inv_s * a.inv_t;
  const auto dense = [&](float xv) {
    const float d = (xv - base) * scale, e = fast_exp2(d);
    if constexpr (ENTROPY) return e * fmaf(v, fmaxf(d, -200.f), u);
    else return e * u;
  };
  const float direct = empty ? 0.f : a.inv_t;  // of a token's own gradient
  p.arrive();
  p.store(dx, dense);
  // an alternative may be the given token too
  bool both = false;
  if (top)
    for (int k = s_head[threadIdx.x]; k >= 0; k = s_next[k]) {
      const bool is_given = s_token[k] == given;
      both |= is_given;
      dx[s_token[k]] = E::narrow(dense(E::widen(x[s_token[k]])) + (s_value[k] + (is_given ? g_given : 0.f)) * direct);
    }
  int owner = -1;
  if (given >= 0 && P::place(cut, part, a.part_chunks, given, owner) >= 0 && owner == static_cast<int>(threadIdx.x) &&
      !both)
    dx[given] = E::narrow(dense(E::widen(raw_given)) + g_given * direct);
}

// The tokens' range alone: a host that must know before it goes on waits for this and not for the
// logits' pass queued behind it.
__global__ __launch_bounds__(256) void token_logprobs_check_kernel(const int64_t* ids, int64_t rows, int64_t V,
                                                                   int64_t ignore_index, int32_t* status) {
  const int64_t row = unit_of_block() * 256 + threadIdx.x;
  if (row >= rows) return;
  const int64_t id = ids[row];
  if (id != ignore_index && (id < 0 || id >= V)) report(status, kBadTokenId);
}

template <typename E, int T, int NV>
void launch_fwd(const FwdArgs& a, hipStream_t stream) {
  const dim3 grid = grid_of(a.rows * a.parts);
  if (a.K) token_logprobs_kernel<E, T, NV, true><<<grid, T, 0, stream>>>(a);
  else token_logprobs_kernel<E, T, NV, false><<<grid, T, 0, stream>>>(a);
  if (a.parts == 1) return;
  const unsigned entries = static_cast<unsigned>(a.parts * a.K);
  const unsigned lds = 8 * (entries + (a.parts + 1) / 2 * a.K);
  if (entries <= 128) token_logprobs_join_kernel<E, 64><<<grid_of(a.rows), 64, lds, stream>>>(a);
  else token_logprobs_join_kernel<E, 256><<<grid_of(a.rows), 256, lds, stream>>>(a);
}

template <typename E, int T, int NV>
void launch_bwd(const BwdArgs& a, hipStream_t stream) {
  const dim3 grid = grid_of(a.rows * a.parts);
  if (a.g_entropy) token_logprobs_bwd_kernel<E, T, NV, true><<<grid, T, 0, stream>>>(a);
  else token_logprobs_bwd_kernel<E, T, NV, false><<<grid, T, 0, stream>>>(a);
}

int check_rows(int dtype, int64_t rows, int64_t vocab, int64_t row_stride, float temperature, int64_t top_k) {
  if (dtype != ASPEC_MASK_BF16 && dtype != ASPEC_MASK_F16 && dtype != ASPEC_MASK_F32)
    return set_error(ASPEC_ERR_UNSUPPORTED, "token log-probabilities take bf16, fp16 or fp32 logits");
  if (rows < 0 || vocab <= 0 || row_stride < vocab)
    return set_error(ASPEC_ERR_INVALID, "token log-probabilities need a vocabulary and rows at least as far apart");
  if (vocab > kMaxVocab)
    return set_error(ASPEC_ERR_UNSUPPORTED, "token log-probabilities support at most %d logits per row",
                     static_cast<int>(kMaxVocab));
  if (!usable_temperature(temperature))
    return set_error(ASPEC_ERR_INVALID, "temperature must be > 0, and its inverse a normal number");
  if (top_k < 0 || top_k > vocab)
    return set_error(ASPEC_ERR_INVALID, "top_k must lie in [0, vocab]");
  if (top_k > kMaxTop)
    return set_error(ASPEC_ERR_UNSUPPORTED, "at most %d alternatives per row are supported", kMaxTop);
  return ASPEC_OK;
}

}  // namespace
}  // namespace aspec

using namespace aspec;

extern "C" int aspec_token_logprobs_stats_floats(void) { return kStats; }

extern "C" int aspec_token_logprobs_workspace_bytes(int dtype, int64_t rows, int64_t vocab, int64_t top_k,
                                                    size_t* bytes) {
  if (const int e = check_rows(dtype, rows, vocab, vocab, 1.f, top_k)) return e;
  if (!bytes) return set_error(ASPEC_ERR_INVALID, "null pointer passed to token log-probabilities");
  const vocab::Shape s = vocab::shape_of(rows, vocab, vocab::per_chunk_of(dtype));
  *bytes = s.parts == 1 ? 0 : static_cast<size_t>(rows) * s.parts * (top_k * 8 + 3 * 4);
  return ASPEC_OK;
}

extern "C" int aspec_token_logprobs_check(const int64_t* token_ids, int64_t rows, int64_t vocab, int64_t ignore_index,
                                          int32_t* status_words, void* stream) {
  if (const int e = check_rows(ASPEC_MASK_F32, rows, vocab, vocab, 1.f, 0)) return e;
  if (rows == 0) return ASPEC_OK;
  if (!token_ids || !status_words)
    return set_error(ASPEC_ERR_INVALID, "null pointer passed to token log-probabilities");
  token_logprobs_check_kernel<<<vocab::grid_of((rows + 255) / 256), 256, 0, static_cast<hipStream_t>(stream)>>>(
      token_ids, rows, vocab, ignore_index, status_words);
  return check_launch("token_logprobs_check_kernel");
}

extern "C" int aspec_token_logprobs_fwd(const void* logits, int dtype, int64_t rows, int64_t vocab,
                                        int64_t row_stride, const int64_t* token_ids, int64_t ignore_index,
                                        float temperature, int64_t top_k, float* logprobs, float* entropy,
                                        float* top_logprobs, int64_t* top_indices, float* stats,
                                        void* workspace, int32_t* status_words, void* stream) {
  if (const int e = check_rows(dtype, rows, vocab, row_stride, temperature, top_k)) return e;
  if (rows == 0) return ASPEC_OK;
  const vocab::Shape s = vocab::shape_of(rows, vocab, vocab::per_chunk_of(dtype));
  if (!logits || !entropy || (token_ids && !logprobs) || (top_k && (!top_logprobs || !top_indices)) ||
      (s.parts > 1 && !workspace))
    return set_error(ASPEC_ERR_INVALID, "null pointer passed to token log-probabilities");
  FwdArgs a{};
  a.x = logits;
  a.rows = rows;
  a.stride = row_stride;
  a.V = static_cast<int>(vocab);
  a.parts = static_cast<int>(s.parts);
  a.part_chunks = static_cast<int>(s.part_chunks);
  a.K = static_cast<int>(top_k);
  a.ids = token_ids;
  a.ignore_index = ignore_index;
  a.inv_t = 1.f / temperature;
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.top_logprobs = top_logprobs;
  a.top_indices = top_indices;
  a.stats = stats;
  a.part_top = static_cast<uint64_t*>(workspace);
  a.part_sums = reinterpret_cast<float*>(a.part_top + rows * s.parts * top_k);
  a.status = status_words;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  dispatch(dtype, s, [&](auto e, auto t, auto nv) { launch_fwd<decltype(e), t.value, nv.value>(a, st); });
  return check_launch("token_logprobs_kernel");
}

extern "C" int aspec_token_logprobs_bwd(const void* logits, int dtype, int64_t rows, int64_t vocab,
                                        int64_t row_stride, const int64_t* token_ids, int64_t ignore_index,
                                        float temperature, int64_t top_k, const int64_t* top_indices,
                                        const float* stats, const float* grad_logprobs,
                                        const float* grad_entropy, const float* grad_top, void* grad_logits,
                                        int64_t grad_stride, void* stream) {
  if (const int e = check_rows(dtype, rows, vocab, row_stride, temperature, top_k)) return e;
  if (grad_stride < vocab)
    return set_error(ASPEC_ERR_INVALID, "token log-probabilities need a vocabulary and rows at least as far apart");
  if (rows == 0) return ASPEC_OK;
  if (!logits || !stats || !grad_logits || (grad_top && !top_indices) || (grad_logprobs && !token_ids))
    return set_error(ASPEC_ERR_INVALID, "null pointer passed to the token log-probability gradient");
  if (grad_logits == logits)
    return set_error(ASPEC_ERR_INVALID, "the token log-probability gradient is not computed in place");
  const vocab::Shape s = vocab::shape_of(rows, vocab, vocab::per_chunk_of(dtype));
  BwdArgs a{};
  a.x = logits;
  a.rows = rows;
  a.stride = row_stride;
  a.V = static_cast<int>(vocab);
  a.parts = static_cast<int>(s.parts);
  a.part_chunks = static_cast<int>(s.part_chunks);
  a.K = grad_top ? static_cast<int>(top_k) : 0;
  a.ids = token_ids;
  a.ignore_index = ignore_index;
  a.inv_t = 1.f / temperature;
  a.top_indices = top_indices;
  a.stats = stats;
  a.g_logprob = grad_logprobs;
  a.g_entropy = grad_entropy;
  a.g_top = grad_top;
  a.dx = grad_logits;
  a.dx_stride = grad_stride;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  dispatch(dtype, s, [&](auto e, auto t, auto nv) { launch_bwd<decltype(e), t.value, nv.value>(a, st); });
  return check_launch("token_logprobs_bwd_kernel");
}
