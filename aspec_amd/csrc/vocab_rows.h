// Rows of logits held in registers: what the token log-probability and the top-logit distillation
// kernels share.
//
// A row of V logits (bf16, fp16 or fp32, any element alignment) is cut at 16-byte boundaries: the
// interior as 16-byte chunks, dealt out to the threads of a workgroup round robin (thread t holds
// chunks t, t + T, ...: coalesced), and up to 2 * (chunk - 1) elements before the first and after
// the last boundary, one to a thread. So no access leaves the row and every vector access is
// aligned, whatever the row's length and start. A row longer than T * NV chunks is cut into parts
// of whole chunks; each part is a workgroup's.
//
// All exponentials are exp2((x - m) * scale) with scale = log2(e) / temperature: the difference
// first, so nothing is rounded at the maximum itself, whatever its size.
#pragma once

#include <math.h>

#include <type_traits>

#include "common.h"

namespace aspec {
namespace vocab {

constexpr int kMaxTop = 128;     // alternatives per row, teacher tokens per row
constexpr int kMaxParts = 32;    // workgroups that share one row
constexpr float kNegInf = -INFINITY;

// The words of status_words, each set to 1 by plain stores: host memory serves as well as the device's.
enum Status { kBadTeacherRow, kBadTarget, kBadTokenId, kBadTeacherToken, kRepeatedToken };
__device__ __forceinline__ void report(int32_t* words, Status s) {
  if (words) __hip_atomic_store(words + s, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// ---- element types -------------------------------------------------------------------------------
struct Bf16 {
  using bits = uint16_t;
  static constexpr int kPerChunk = 8;
  static constexpr int kKeyDrop = 16;  // low bits that no two order_key()s differ in alone
  static constexpr uint32_t kNegInfBits = 0xff80u;
  static __device__ __forceinline__ float widen(uint16_t b) { return bf16_to_f32(b); }
  static __device__ __forceinline__ uint16_t narrow(float f) { return f32_to_bf16_bits(f); }
  static __device__ __forceinline__ float from_word(uint32_t w, int high) {
    return __uint_as_float(high ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ uint32_t to_word(float lo, float hi) { return pack_bf16x2(lo, hi); }
};
struct F16 {
  using bits = uint16_t;
  static constexpr int kPerChunk = 8;
  static constexpr int kKeyDrop = 13;  // low bits that no two order_key()s differ in alone
  static constexpr uint32_t kNegInfBits = 0xfc00u;
  static __device__ __forceinline__ float widen(uint16_t b) {
    return static_cast<float>(__builtin_bit_cast(_Float16, b));
  }
  static __device__ __forceinline__ uint16_t narrow(float f) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
  }
  static __device__ __forceinline__ float from_word(uint32_t w, int high) {
    return widen(static_cast<uint16_t>(high ? (w >> 16) : (w & 0xffffu)));
  }
  static __device__ __forceinline__ uint32_t to_word(float lo, float hi) {
    return static_cast<uint32_t>(narrow(lo)) | (static_cast<uint32_t>(narrow(hi)) << 16);
  }
};
struct F32 {
  using bits = uint32_t;
  static constexpr int kPerChunk = 4;
  static constexpr int kKeyDrop = 0;  // low bits that no two order_key()s differ in alone
  static constexpr uint32_t kNegInfBits = 0xff800000u;
  static __device__ __forceinline__ float widen(uint32_t b) { return __uint_as_float(b); }
  static __device__ __forceinline__ uint32_t narrow(float f) { return __float_as_uint(f); }
};

__device__ __forceinline__ uint32_t word_of(const uint4& w, int j) {
  return j == 0 ? w.x : j == 1 ? w.y : j == 2 ? w.z : w.w;
}
__device__ __forceinline__ void set_word(uint4& w, int j, uint32_t v) {
  if (j == 0) w.x = v;
  else if (j == 1) w.y = v;
  else if (j == 2) w.z = v;
  else w.w = v;
}

// Element i of a chunk (i a constant after unrolling).
template <typename E>
__device__ __forceinline__ float element(const uint4& w, int i) {
  if constexpr (E::kPerChunk == 4) return __uint_as_float(word_of(w, i));
  else return E::from_word(word_of(w, i >> 1), i & 1);
}

// Element i of a chunk, i at run time.
template <typename E>
__device__ __forceinline__ float element_at(const uint4& w, int i) {
  constexpr int per = E::kPerChunk / 4;
  const int j = i / per;
  const uint32_t a = j & 1 ? w.y : w.x, b = j & 1 ? w.w : w.z, word = j & 2 ? b : a;
  if constexpr (per == 1) return __uint_as_float(word);
  else return E::widen(static_cast<uint16_t>(i & 1 ? word >> 16 : word));
}

template <typename E>
__device__ __forceinline__ uint4 all_neg_inf() {
  const uint32_t v = E::kPerChunk == 4 ? E::kNegInfBits : (E::kNegInfBits | (E::kNegInfBits << 16));
  return make_uint4(v, v, v, v);
}

// 16 bytes of a row from element `at` on, at any element alignment: gradient and logits rows may be
// aligned differently. The byte offset has 32 bits (rows have at most 2 MB), so that the row's
// address stays in scalar registers.
template <typename E>
__device__ __forceinline__ uint4 load16(const typename E::bits* row, int at) {
  const uint32_t off = static_cast<uint32_t>(at) * static_cast<uint32_t>(sizeof(typename E::bits));
  return load_chunk(reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(row) + off));
}
template <typename E>
__device__ __forceinline__ void store16(typename E::bits* row, int at, const uint4& v) {
  const uint32_t off = static_cast<uint32_t>(at) * static_cast<uint32_t>(sizeof(typename E::bits));
  store_chunk(reinterpret_cast<uint16_t*>(reinterpret_cast<char*>(row) + off), v);
}

__device__ const uint4 kNoChunk = {};

// ---- how a row is cut ----------------------------------------------------------------------------
// `lead` elements, then `chunks` whole chunks, then the rest up to V.
struct RowCut {
  int lead, chunks, V;
  template <typename E>
  static __device__ __forceinline__ RowCut at(const void* row, int V) {
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(typename E::bits));
    const int lead = min(V, (E::kPerChunk - off) % E::kPerChunk);
    return RowCut{lead, (V - lead) / E::kPerChunk, V};
  }
};

// One part of a row in the registers of a workgroup of T threads: chunks [c0, c1) of the row and,
// in part 0, its edge elements (thread t < lead: element t; thread kPerChunk + t: the t-th element
// behind the last chunk).
template <typename E, int T, int NV>
struct Part {
  static constexpr int CH = E::kPerChunk;
  static constexpr int kSkip = NV > 4 ? NV * 2 / 5 : 1;
  uint4 w[NV];
  float edge;     // -inf where this thread has none
  typename E::bits edge_raw;
  int edge_at;    // its index in the row, or -1
  int held;       // chunks that this thread has
  int first;      // index in the row of its first chunk; the next ones are T chunks apart each

  // Every load is made, of the row's first chunk where the thread has none: a load in a branch is
  // waited for at the branch's end, one latency each. arrive() puts -inf there; what is done between
  // the two does not wait for the row.
  __device__ __forceinline__ void load(const typename E::bits* row, const RowCut& rc, int part, int part_chunks) {
    const int t = threadIdx.x, c0 = part * part_chunks;
    held = max(0, (min(part_chunks, rc.chunks - c0) - t + T - 1) / T);
    first = rc.lead + (c0 + t) * CH;
    const int behind = rc.lead + rc.chunks * CH + t - CH;
    edge_at = part != 0 ? -1 : t < rc.lead ? t : t >= CH && behind < rc.V ? behind : -1;
    edge_raw = row[max(edge_at, 0)];
    const bool any = rc.chunks > 0;  // a row without a whole chunk reads one that is nobody's
    const auto* src = any ? row : reinterpret_cast<const typename E::bits*>(&kNoChunk);
    const int none = any ? rc.lead : 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) w[v] = load16<E>(src, v < held ? first + v * (T * CH) : none);
  }
  __device__ __forceinline__ void arrive() {
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (v >= held) w[v] = all_neg_inf<E>();
    edge = edge_at >= 0 ? E::widen(edge_raw) : kNegInf;
  }

  // Makes the chunks opaque to the compiler, so that the next pass over them widens them, compares
  // and computes addresses again: otherwise it keeps one pass's floats, masks and addresses for the
  // next, more registers than the row itself.
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int v = 0; v < NV; ++v) asm volatile("" : "+v"(w[v].x), "+v"(w[v].y), "+v"(w[v].z), "+v"(w[v].w));
    asm volatile("" : "+v"(held), "+v"(first));
  }

  // The largest element of chunks [from, to) of the thread; a NaN is skipped, or is the result.
  // Sixteen-bit floats are compared as whole numbers, two to an instruction and without widening:
  // where any is positive, the largest number is the largest float; where none is, the smallest is.
  template <int FROM, int TO>
  __device__ __forceinline__ float largest_of() const {
    if constexpr (CH == 4) {
      float m = kNegInf;
#pragma unroll
      for (int v = FROM; v < TO; ++v)
#pragma unroll
        for (int i = 0; i < CH; ++i) m = fmaxf(m, element<E>(w[v], i));
      return m;
    } else {
      typedef __attribute__((ext_vector_type(2))) short pair;
      const auto fold = [&](auto op) {
        pair r = __builtin_bit_cast(pair, w[FROM].x);
#pragma unroll
        for (int v = FROM; v < TO; ++v)
#pragma unroll
          for (int j = 0; j < 4; ++j) r = op(r, __builtin_bit_cast(pair, word_of(w[v], j)));
        return r;
      };
      const pair high = fold([](pair a, pair b) { return __builtin_elementwise_max(a, b); });
      short best = high.x > high.y ? high.x : high.y;
      if (best < 0) {
        const pair low = fold([](pair a, pair b) { return __builtin_elementwise_min(a, b); });
        best = low.x < low.y ? low.x : low.y;
      }
      return E::widen(static_cast<uint16_t>(best));
    }
  }
  __device__ __forceinline__ float largest() const { return fmaxf(largest_of<0, NV>(), edge); }
  // The largest element of half of a chunk; a NaN is skipped, or is the result.
  __device__ __forceinline__ float largest_of_half(int h) const {
    constexpr int HALF = CH / 2;
    float m = element<E>(w[h / 2], h % 2 * HALF);
#pragma unroll
    for (int i = 1; i < HALF; ++i) m = fmaxf(m, element<E>(w[h / 2], h % 2 * HALF + i));
    return m;
  }
  // One bit for each chunk whose largest element is not below a bound.
  template <int V = 0>
  __device__ __forceinline__ uint32_t chunks_reaching(float bound) const {
    if constexpr (V < NV) {
      return (largest_of<V, V + 1>() < bound ? 0u : 1u << V) | chunks_reaching<V + 1>(bound);
    } else {
      return 0;
    }
  }

  // f(value) of every element that the thread holds; -inf for some of the places it does not fill. From
  // chunk kSkip on, the wave leaves out the ones that no lane has: the shapes above 4 chunks to a thread
  // fill at least that many, and a row between two shapes' sizes does not pay for the larger one
  // (log-probabilities of 8192 x 20000 76 -> 56 us, losses and gradient of 2048 x 100000 228 -> 211).
  template <typename F>
  __device__ __forceinline__ void each_value(F f) const {
    const int any = __builtin_amdgcn_readfirstlane(held);  // no lane of the wave holds more than its first
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (v >= kSkip && v >= any) continue;
#pragma unroll
      for (int i = 0; i < CH; ++i) f(element<E>(w[v], i));
    }
    f(edge);
  }
  // f(value, index in the row) of the elements that are there.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (v < held) {
#pragma unroll
        for (int i = 0; i < CH; ++i) f(element<E>(w[v], i), first + v * (T * CH) + i);
      }
    if (edge_at >= 0) f(edge, edge_at);
  }

  // Chunks of a part, and the row's chunk that is the part's c-th.
  static __device__ __forceinline__ int chunks_in(const RowCut& rc, int part, int part_chunks) {
    return max(0, min(part_chunks, rc.chunks - part * part_chunks));
  }
  static __device__ __forceinline__ int index_of(const RowCut& rc, int part, int part_chunks, int c) {
    return rc.lead + (part * part_chunks + c) * CH;
  }
  // Where a token of the row is held: its place within the thread and, through `owner`, the thread;
  // -1 if another part holds it.
  static __device__ __forceinline__ int place(const RowCut& rc, int part, int part_chunks, int token, int& owner) {
    const int in = token - rc.lead;
    const int c = in / CH;
    if (in >= 0 && c < rc.chunks) {
      const int local = c - part * part_chunks;
      if (local < 0 || local >= part_chunks) return -1;
      owner = local % T;
      return (local / T) * CH + in % CH;
    }
    if (part != 0) return -1;
    owner = in < 0 ? token : CH + token - (rc.lead + rc.chunks * CH);
    return NV * CH;
  }
  // Sets the element at a place to -inf: the masks of its word first, so that the branch for its chunk
  // is one instruction a word (lanes whose chunks differ take the branches one after another; with the
  // places compared in each branch 1536 x 151936 and 128 kept tokens took 228 us for 223).
  __device__ __forceinline__ void knock_out(int at) {
    if (at == NV * CH) edge = kNegInf;
    const int i = at % CH, word = CH == 4 ? i : i / 2;
    const uint32_t bits = CH == 4 ? ~0u : i % 2 ? 0xffff0000u : 0xffffu;
    constexpr uint32_t none = CH == 4 ? E::kNegInfBits : E::kNegInfBits * 0x10001u;
    uint32_t mask[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) mask[j] = word == j ? bits : 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (v != at / CH) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) set_word(w[v], j, (word_of(w[v], j) & ~mask[j]) | (none & mask[j]));
    }
  }
  // Writes g(value) of every element to a row cut alike.
  template <typename F>
  __device__ __forceinline__ void store(typename E::bits* row, F g) const {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (v >= held) continue;
      uint4 o;
      if constexpr (CH == 4) {
        o = make_uint4(E::narrow(g(element<E>(w[v], 0))), E::narrow(g(element<E>(w[v], 1))),
                       E::narrow(g(element<E>(w[v], 2))), E::narrow(g(element<E>(w[v], 3))));
      } else {
        o = make_uint4(E::to_word(g(element<E>(w[v], 0)), g(element<E>(w[v], 1))),
                       E::to_word(g(element<E>(w[v], 2)), g(element<E>(w[v], 3))),
                       E::to_word(g(element<E>(w[v], 4)), g(element<E>(w[v], 5))),
                       E::to_word(g(element<E>(w[v], 6)), g(element<E>(w[v], 7))));
      }
      store16<E>(row, first + v * (T * CH), o);
    }
    if (edge_at >= 0) row[edge_at] = E::narrow(g(edge));
  }
};

// A maximum to take differences from: a part without a finite logit sums exp2(-inf) = 0 terms.
__device__ __forceinline__ float base_of(float m) { return m == kNegInf ? 0.f : m; }

// The factor that takes sums relative to maximum m to ones relative to M >= m (1 where the sum has
// no term; a NaN sum stays NaN).
__device__ __forceinline__ float rebase(float m, float M, float scale) {
  return m == kNegInf ? 1.f : fast_exp2((m - M) * scale);
}

// ---- order ---------------------------------------------------------------------------------------
// Whole numbers in the order of the floats, -0 as +0 and every NaN above +inf.
__device__ __forceinline__ uint32_t order_key(float f) {
  uint32_t u = __float_as_uint(f);
  if (f != f) return 0xffffffffu;
  if (f == 0.f) u = 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
// Larger first, then the lower index; 0 is below every token.
__device__ __forceinline__ uint64_t ranked(uint32_t key, int index) {
  return (static_cast<uint64_t>(key) << 32) | (0xffffffffu - static_cast<uint32_t>(index));
}
__device__ __forceinline__ int ranked_index(uint64_t r) {
  return static_cast<int>(0xffffffffu - static_cast<uint32_t>(r));
}
__device__ __forceinline__ float ranked_value(uint64_t r) { return key_value(static_cast<uint32_t>(r >> 32)); }

__device__ __forceinline__ uint32_t wave_allmax_u32(uint32_t v) {
  return wave_allreduce_bits(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ uint32_t wave_allsum_u32(uint32_t v) {
  return wave_allreduce_bits(v, [](uint32_t a, uint32_t b) { return a + b; });
}
__device__ __forceinline__ double wave_allsum_f64(double v) {
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// ---- launch shapes -------------------------------------------------------------------------------
// A shape is (threads of a workgroup, chunks a thread holds).
struct Shape {
  int threads, held;
  int64_t parts, part_chunks;
};
constexpr int64_t kMaxVocab = int64_t{1} << 19;  // 32 parts of 4096 chunks of four fp32 logits

// Whether 1 / temperature is a normal number (a subnormal one is 0 to the kernels).
inline bool usable_temperature(float t) { return t > 0.f && 1.f / t >= 0x1p-126f && !isinf(1.f / t); }

inline int per_chunk_of(int dtype) { return dtype == ASPEC_MASK_F32 ? 4 : 8; }

// Rows of up to 256 chunks take a wave each, up to 1024 a workgroup of 256 threads. Longer rows take
// workgroups of 512 threads where that makes two of them for each of the 256 CUs, and 256 x 4 chunks
// otherwise: with few rows the time is one workgroup's, and four times as many share a row. The 512
// hold 8 chunks each, or 4 where that leaves a tenth fewer places empty: 16384 x 4096 logits of 16 bits
// took 143 us with 512 x 8 (one chunk to a thread, seven places empty), 44 with 256 x 4; 4096 x 16384
// took 39 with 512 x 8 and take 25 with 512 x 4.
inline Shape shape_of(int64_t rows, int64_t V, int per_chunk) {
  const int64_t chunks = V / per_chunk;
  const auto parts = [chunks](int64_t places) { return (chunks + places - 1) / places; };
  Shape s{64, 4, 1, 0};
  if (chunks > 64 * 4) {
    const int64_t few = parts(256 * 4), half = parts(512 * 4), full = parts(512 * 8);
    if (few == 1 || (rows * full < 512 && few <= kMaxParts)) s = Shape{256, 4, few, 0};
    else if (half <= kMaxParts && 10 * half * 4 < 9 * full * 8) s = Shape{512, 4, half, 0};
    else s = Shape{512, 8, full, 0};
  }
  s.part_chunks = (chunks + s.parts - 1) / s.parts;
  return s;
}

// Waves per SIMD that the compiler keeps registers for where a workgroup holds a row for its losses and
// its gradient: three workgroups of 512 threads to a CU (80 registers), so that one's reductions hide
// behind another's loads; with 20 chunks to a thread, two of 512 or one of 1024 (128). Kernels without
// the gradient fit eight waves (64).
constexpr int min_waves(int held) { return held == 20 ? 4 : 6; }

// One workgroup per unit (a row or a part of one), not a loop over units: what a loop body of this
// size keeps in registers across units costs the kernels half their occupancy. A grid has fewer than
// 2^32 threads in x.
inline dim3 grid_of(int64_t units) {
  const int64_t x = units < (int64_t{1} << 21) ? units : (int64_t{1} << 21);
  return dim3(static_cast<unsigned>(x), static_cast<unsigned>((units + x - 1) / x));
}
__device__ __forceinline__ int64_t unit_of_block() {
  return static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x;
}

// f(element type, threads, chunks held) for a launch's type and shape.
template <typename E, typename F>
void dispatch_shape(const Shape& s, F f) {
  if (s.threads == 64) f(E{}, std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
  else if (s.threads == 256) f(E{}, std::integral_constant<int, 256>{}, std::integral_constant<int, 4>{});
  else if (s.held == 4) f(E{}, std::integral_constant<int, 512>{}, std::integral_constant<int, 4>{});
  else f(E{}, std::integral_constant<int, 512>{}, std::integral_constant<int, 8>{});
}
template <typename F>
void dispatch(int dtype, const Shape& s, F f) {
  if (dtype == ASPEC_MASK_BF16) dispatch_shape<Bf16>(s, f);
  else if (dtype == ASPEC_MASK_F16) dispatch_shape<F16>(s, f);
  else dispatch_shape<F32>(s, f);
}

}  // namespace vocab
}  // namespace aspec
