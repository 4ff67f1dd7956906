// Distillation from a teacher's best tokens: forward and gradient as two passes (the formulas are in
// topk_distill.h, the one-pass kernel in topk_distill_fused.hip).
//
// HBM-bound: the forward reads each logit once, the gradient reads it once and writes once; the
// teacher's K pairs a row are a few hundred bytes. The gradient is dense over a part of a row in
// registers; the kept tokens and the target, which have values of their own, are written behind the
// dense ones by the thread that wrote those.
//
// 8192 x 32000 bf16, 64 kept tokens: forward 124-142 us behind the last gradient's writes (533 MB
// read, VALU busy 0.8 with the second exponential of a temperature), gradient 180 us (1097 MB, 6.1 TB/s
// read and written). 1024 x 65536 fp32, 32 kept, forward alone: 42 us (281 MB, 6.7 TB/s) and 5 us of
// joining parts. At 16 rows each launch takes 4-5 us, the chain of one workgroup: the teacher's
// entries, their logits, the row, the K-term sums in 64 bits.
#include "topk_distill.h"

namespace aspec {

// topk_distill_fused.hip: whether rows of V logits fit one workgroup's registers, and the launch.
bool topk_distill_fused_fits(int64_t V, int per_chunk);
void topk_distill_fused_launch(int dtype, bool two, const distill::Args& a, hipStream_t stream);

namespace {

using namespace distill;

template <typename E, int T, int NV, bool TWO>
__global__ __launch_bounds__(T, 8) void topk_distill_kernel(Args a) {
  __shared__ Kept<T> kept;
  __shared__ float s_m[T / 64], s_s[T / 64], s_s1[T / 64];
  __shared__ uint64_t s_arg;
  __shared__ Factors s_factors;
  const int64_t unit = unit_of_block();
  if (unit < a.rows * a.parts)
    forward_unit<E, T, NV, TWO, false>(a, unit, kept, s_m, s_s, s_s1, s_arg, s_factors);
}

// Joins the parts of long rows, a wave to a row.
template <typename E, bool TWO>
__global__ __launch_bounds__(64) void topk_distill_join_kernel(Args a) {
  __shared__ Kept<1> kept;
  const int lane = threadIdx.x;
  const float scale = a.inv_t * kLog2e;
  const int64_t row = unit_of_block();
  if (row >= a.rows) return;
  const auto* x = reinterpret_cast<const typename E::bits*>(a.x) + row * a.stride;
  const int64_t trow = teacher_row(a, row);
  const Target target = read_target(a, row);
  const float x_target = E::widen(x[max(target.token, 0)]);
  bool bad = trow < 0;  // reported by the parts
  uint64_t best = 0;
  for (int k = lane; k < a.K; k += 64) {
    const RawEntry entry = load_entry(a, trow, k);
    kept.token[k] = token_of(a, trow, k, entry, bad);
    kept.lp[k] = entry.lp;
    kept.fill(k, E::widen(x[max(kept.token[k], 0)]));
    if (kept.token[k] >= 0) best = max(best, ranked(order_key(kept.x[k]), kept.token[k]));
  }
  Tail t{kNegInf, 0.f, 0.f};
  if (lane < a.parts) {
    const float4 s = *reinterpret_cast<const float4*>(a.part_sums + (row * a.parts + lane) * 4);
    t = Tail{s.x, s.y, s.z};
    best = max(best, a.part_arg[row * a.parts + lane]);
  }
  t = merge_wave<TWO>(t, scale);
  if (lane == 0) kept.poison = 0;
  __syncthreads();
  if (__any(bad) && lane == 0) kept.poison = 1;
  __syncthreads();
  float st[kStats];
  finish_row<TWO>(a, row, lane, t, kept, target, x_target, st);
  if (a.argmax) {
    best = wave_allmax_u64(best);
    if (lane == 0) a.argmax[row] = ranked_index(best);
  }
}

// Gradient from the forward's statistics; it may go to the logits' own buffer (every element is read
// before the barrier that the first one is written behind).
template <typename E, int T, int NV, bool TWO>
__global__ __launch_bounds__(T, 8) void topk_distill_bwd_kernel(Args a) {
  using P = Part<E, T, NV>;
  __shared__ int s_head[T];
  __shared__ int s_next[kMaxTop], s_token[kMaxTop];
  __shared__ float s_value[kMaxTop];
  const float scale = a.inv_t * kLog2e;
  const int64_t unit = unit_of_block();
  if (unit >= a.rows * a.parts) return;
  const int64_t row = a.parts == 1 ? unit : unit / a.parts;
  const int part = a.parts == 1 ? 0 : static_cast<int>(unit - row * a.parts);
  const auto* x = reinterpret_cast<const typename E::bits*>(a.x) + row * a.stride;
  auto* dx = reinterpret_cast<typename E::bits*>(a.dx) + row * a.dx_stride;
  const RowCut cut = RowCut::at<E>(dx, a.V);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t trow = teacher_row(a, row);
  const Target target = read_target(a, row);
  const typename E::bits raw_target = x[max(target.token, 0)];
  float st[kStats];
#pragma unroll
  for (int i = 0; i < kStats; ++i) st[i] = a.stats[row * kStats + i];
  const float g_kl = a.g_kl ? a.g_kl[row] : 0.f, g_ce = a.g_ce ? a.g_ce[row] : 0.f;
  RawEntry entry[2];
  if (wave == 0) {
    entry[0] = load_entry(a, trow, lane);
    entry[1] = load_entry(a, trow, lane + 64);
  }
  P p;
  p.load(x, cut, part, a.part_chunks);
  s_head[threadIdx.x] = -1;
  const float gc = target.bad ? __builtin_nanf("") : target.token >= 0 ? g_ce : 0.f;
  const Factors f = factors_of<TWO>(st, g_kl, gc, a.inv_t);
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = lane + 64 * h;
      bool bad = false;  // the forward has made such a row's statistics NaN
      const int token = token_of(a, trow, k, entry[h], bad);
      const typename E::bits raw = x[max(token, 0)];
      int owner = 0;
      if (token < 0 || P::place(cut, part, a.part_chunks, token, owner) < 0) continue;
      s_next[k] = atomicExch(&s_head[owner], k);
      s_token[k] = token;
      s_value[k] = st[1] == 0.f ? 0.f
                                : f.template kept<TWO>(E::widen(raw), expf(entry[h].lp) * f.c, token == target.token,
                                                       scale);
    }
  }
  __syncthreads();
  p.arrive();
  p.store(dx, [&](float v) { return f.template tail<TWO>(v, scale); });
  bool kept_target = false;
  for (int k = s_head[threadIdx.x]; k >= 0; k = s_next[k]) {
    dx[s_token[k]] = E::narrow(s_value[k]);
    kept_target |= s_token[k] == target.token;
  }
  int owner = -1;
  if (target.token >= 0 && P::place(cut, part, a.part_chunks, target.token, owner) >= 0 &&
      owner == static_cast<int>(threadIdx.x) && !kept_target)
    dx[target.token] =
        E::narrow(st[1] == 0.f ? 0.f : f.template tail<TWO>(E::widen(raw_target), scale) - gc);
}

// The indices alone, a wave to a row: what is wrong with them goes to the status words. It reads a few
// hundred bytes a row (8192 rows of 64 tokens: 4 us), so a host that must know before it goes on waits
// for this and not for the logits' pass queued behind it.
constexpr int kCheckRows = 4;
constexpr int kSeenBits = 1 << 15;
__global__ __launch_bounds__(64 * kCheckRows) void topk_distill_check_kernel(Args a) {
  __shared__ uint4 s_seen[kCheckRows][kSeenBits / 128];
  const int lane = threadIdx.x & 63;
  const int64_t row = unit_of_block() * kCheckRows + (threadIdx.x >> 6);
  const bool live = row < a.rows;
  const int64_t trow = live ? teacher_row(a, row) : -1;  // no row: no token
  const bool bad_target = live && read_target(a, row).bad;
  bool bad = false;
  int token[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) token[h] = token_of(a, trow, lane + 64 * h, load_entry(a, trow, lane + 64 * h), bad);
  // a token that finds its bit (its index modulo 2^15) set may be there twice, and is counted
  uint4* words = s_seen[threadIdx.x >> 6];
#pragma unroll
  for (int i = 0; i < kSeenBits / 128 / 64; ++i) words[lane + 64 * i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  bool twice = false;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    bool seen = false;
    if (token[h] >= 0) {
      const uint32_t bit = 1u << (token[h] & 31);
      seen = (atomicOr(reinterpret_cast<uint32_t*>(words) + (token[h] % kSeenBits >> 5), bit) & bit) != 0;
    }
    for (uint64_t lanes = __ballot(seen); lanes; lanes &= lanes - 1) {
      const int t = __builtin_amdgcn_readlane(token[h], __ffsll(static_cast<unsigned long long>(lanes)) - 1);
      twice |= __popcll(__ballot(token[0] == t)) + __popcll(__ballot(token[1] == t)) > 1;
    }
  }
  const bool any_bad = __any(bad);
  if (lane != 0 || !live) return;
  if (trow < 0) report(a.status, kBadTeacherRow);
  if (bad_target) report(a.status, kBadTarget);
  if (any_bad) report(a.status, kBadTeacherToken);
  if (twice) report(a.status, kRepeatedToken);
}

template <typename E, int T, int NV>
void launch_fwd(const Args& a, bool two, hipStream_t stream) {
  const dim3 grid = grid_of(a.rows * a.parts);
  if (two) topk_distill_kernel<E, T, NV, true><<<grid, T, 0, stream>>>(a);
  else topk_distill_kernel<E, T, NV, false><<<grid, T, 0, stream>>>(a);
  if (a.parts == 1) return;
  if (two) topk_distill_join_kernel<E, true><<<grid_of(a.rows), 64, 0, stream>>>(a);
  else topk_distill_join_kernel<E, false><<<grid_of(a.rows), 64, 0, stream>>>(a);
}

template <typename E, int T, int NV>
void launch_bwd(const Args& a, bool two, hipStream_t stream) {
  const dim3 grid = grid_of(a.rows * a.parts);
  if (two) topk_distill_bwd_kernel<E, T, NV, true><<<grid, T, 0, stream>>>(a);
  else topk_distill_bwd_kernel<E, T, NV, false><<<grid, T, 0, stream>>>(a);
}

int check_distill(int dtype, int64_t rows, int64_t vocab, int64_t row_stride, int token_dtype, int64_t kept,
                  const int64_t* teacher_rows, int64_t num_teacher_rows, float temperature) {
  if (dtype != ASPEC_MASK_BF16 && dtype != ASPEC_MASK_F16 && dtype != ASPEC_MASK_F32)
    return set_error(ASPEC_ERR_UNSUPPORTED, "top-logit distillation takes bf16, fp16 or fp32 logits");
  if (rows < 0 || vocab <= 0 || row_stride < vocab)
    return set_error(ASPEC_ERR_INVALID, "top-logit distillation needs a vocabulary and rows at least as far apart");
  if (vocab > kMaxVocab)
    return set_error(ASPEC_ERR_UNSUPPORTED, "top-logit distillation supports at most %d logits per row",
                     static_cast<int>(kMaxVocab));
  if (token_dtype != ASPEC_MASK_I64 && token_dtype != ASPEC_MASK_I32)
    return set_error(ASPEC_ERR_INVALID, "teacher tokens are int64 or int32");
  if (teacher_rows ? num_teacher_rows < 1 && rows > 0 : num_teacher_rows != rows)
    return set_error(ASPEC_ERR_INVALID, "a teacher has a row per logit row, or a table of at least one");
  if (kept < 1) return set_error(ASPEC_ERR_INVALID, "top-logit distillation needs a teacher token per row");
  if (kept > kMaxTop)
    return set_error(ASPEC_ERR_UNSUPPORTED, "at most %d teacher tokens per row are supported", kMaxTop);
  if (!usable_temperature(temperature))
    return set_error(ASPEC_ERR_INVALID, "temperature must be > 0, and its inverse a normal number");
  return ASPEC_OK;
}

Args make_args(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
               const int64_t* targets, int64_t ignore_index, const void* tokens, int token_dtype,
               const float* logprobs, int64_t kept, const int64_t* teacher_rows, int64_t num_teacher_rows,
               int renormalize, float temperature, float* ce, float* kl, float* accept, int64_t* argmax, float* stats,
               void* workspace, int32_t* status) {
  const Shape s = shape_of(rows, vocab, per_chunk_of(dtype));
  Args a{};
  a.x = logits;
  a.rows = rows;
  a.stride = row_stride;
  a.V = static_cast<int>(vocab);
  a.parts = static_cast<int>(s.parts);
  a.part_chunks = static_cast<int>(s.part_chunks);
  a.K = static_cast<int>(kept);
  a.targets = targets;
  a.ignore_index = ignore_index;
  a.tokens = tokens;
  a.tokens64 = token_dtype == ASPEC_MASK_I64;
  a.logprobs = logprobs;
  a.trow = teacher_rows;
  a.trows = num_teacher_rows;
  a.renormalize = renormalize;
  a.inv_t = 1.f / temperature;
  a.ce = ce;
  a.kl = kl;
  a.accept = accept;
  a.argmax = argmax;
  a.stats = stats;
  a.part_sums = static_cast<float*>(workspace);
  a.part_arg = reinterpret_cast<uint64_t*>(a.part_sums + rows * s.parts * 4);
  a.status = status;
  return a;
}

// CE is at temperature 1: a second sum where the divergence is at another.
bool two_sums(const Args& a) { return a.targets && a.inv_t != 1.f; }

void run_fwd(int dtype, const Args& a, hipStream_t stream) {
  dispatch(dtype, shape_of(a.rows, a.V, per_chunk_of(dtype)),
           [&](auto e, auto t, auto nv) { launch_fwd<decltype(e), t.value, nv.value>(a, two_sums(a), stream); });
}
void run_bwd(int dtype, const Args& a, hipStream_t stream) {
  dispatch(dtype, shape_of(a.rows, a.V, per_chunk_of(dtype)),
           [&](auto e, auto t, auto nv) { launch_bwd<decltype(e), t.value, nv.value>(a, two_sums(a), stream); });
}

int null_pointer() { return set_error(ASPEC_ERR_INVALID, "null pointer passed to top-logit distillation"); }

}  // namespace
}  // namespace aspec

using namespace aspec;

extern "C" int aspec_topk_distill_stats_floats(void) { return kStats; }

extern "C" int aspec_topk_distill_workspace_bytes(int dtype, int64_t rows, int64_t vocab, size_t* bytes) {
  if (const int e = check_distill(dtype, rows, vocab, vocab, ASPEC_MASK_I64, 1, nullptr, rows, 1.f)) return e;
  if (!bytes) return null_pointer();
  const Shape s = shape_of(rows, vocab, per_chunk_of(dtype));
  *bytes = s.parts == 1 ? 0 : static_cast<size_t>(rows) * s.parts * (4 * 4 + 8);
  return ASPEC_OK;
}

extern "C" int aspec_topk_distill_reads(int dtype, int64_t vocab) {
  return topk_distill_fused_fits(vocab, per_chunk_of(dtype)) ? 1 : 2;
}

extern "C" int aspec_topk_distill_check(int64_t rows, int64_t vocab, const int64_t* targets, int64_t ignore_index,
                                        const void* teacher_tokens, int token_dtype, const float* teacher_logprobs,
                                        int64_t kept, const int64_t* teacher_rows, int64_t num_teacher_rows,
                                        int32_t* status_words, void* stream) {
  if (const int e = check_distill(ASPEC_MASK_F32, rows, vocab, vocab, token_dtype, kept, teacher_rows,
                                  num_teacher_rows, 1.f))
    return e;
  if (rows == 0) return ASPEC_OK;
  if (!teacher_tokens || !teacher_logprobs || !status_words) return null_pointer();
  const Args a = make_args(nullptr, ASPEC_MASK_F32, rows, vocab, vocab, targets, ignore_index, teacher_tokens,
                           token_dtype, teacher_logprobs, kept, teacher_rows, num_teacher_rows, 0, 1.f, nullptr,
                           nullptr, nullptr, nullptr, nullptr, nullptr, status_words);
  topk_distill_check_kernel<<<grid_of((rows + kCheckRows - 1) / kCheckRows), 64 * kCheckRows, 0,
                              static_cast<hipStream_t>(stream)>>>(a);
  return check_launch("topk_distill_check_kernel");
}

extern "C" int aspec_topk_distill_fwd(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                                      const int64_t* targets, int64_t ignore_index, const void* teacher_tokens,
                                      int token_dtype, const float* teacher_logprobs, int64_t kept,
                                      const int64_t* teacher_rows, int64_t num_teacher_rows, int renormalize,
                                      float temperature, float* ce, float* kl, float* accept, int64_t* argmax,
                                      float* stats, void* workspace, int32_t* status_words, void* stream) {
  if (const int e = check_distill(dtype, rows, vocab, row_stride, token_dtype, kept, teacher_rows, num_teacher_rows,
                                  temperature))
    return e;
  if (rows == 0) return ASPEC_OK;
  const Args a = make_args(logits, dtype, rows, vocab, row_stride, targets, ignore_index, teacher_tokens, token_dtype,
                           teacher_logprobs, kept, teacher_rows, num_teacher_rows, renormalize, temperature, ce, kl,
                           accept, argmax, stats, workspace, status_words);
  if (!logits || !teacher_tokens || !teacher_logprobs || (targets && !ce) || !kl || !accept ||
      (a.parts > 1 && !workspace))
    return null_pointer();
  run_fwd(dtype, a, static_cast<hipStream_t>(stream));
  return check_launch("topk_distill_kernel");
}

extern "C" int aspec_topk_distill_bwd(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                                      const int64_t* targets, int64_t ignore_index, const void* teacher_tokens,
                                      int token_dtype, const float* teacher_logprobs, int64_t kept,
                                      const int64_t* teacher_rows, int64_t num_teacher_rows, float temperature,
                                      const float* stats, const float* grad_ce, const float* grad_kl,
                                      void* grad_logits, int64_t grad_stride, void* stream) {
  if (const int e = check_distill(dtype, rows, vocab, row_stride, token_dtype, kept, teacher_rows, num_teacher_rows,
                                  temperature))
    return e;
  if (grad_stride < vocab)
    return set_error(ASPEC_ERR_INVALID, "top-logit distillation needs a vocabulary and rows at least as far apart");
  if (rows == 0) return ASPEC_OK;
  Args a = make_args(logits, dtype, rows, vocab, row_stride, targets, ignore_index, teacher_tokens, token_dtype,
                     teacher_logprobs, kept, teacher_rows, num_teacher_rows, 0, temperature, nullptr, nullptr, nullptr,
                     nullptr, const_cast<float*>(stats), nullptr, nullptr);
  a.g_ce = grad_ce;
  a.g_kl = grad_kl;
  a.dx = grad_logits;
  a.dx_stride = grad_stride;
  if (!logits || !teacher_tokens || !teacher_logprobs || !stats || !grad_logits || (grad_ce && !targets))
    return null_pointer();
  if (grad_logits == logits && grad_stride != row_stride)
    return set_error(ASPEC_ERR_INVALID, "a gradient in place has the logits' row stride");
  run_bwd(dtype, a, static_cast<hipStream_t>(stream));
  return check_launch("topk_distill_bwd_kernel");
}

extern "C" int aspec_topk_distill_fused_fwd_bwd(
    const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride, const int64_t* targets,
    int64_t ignore_index, const void* teacher_tokens, int token_dtype, const float* teacher_logprobs, int64_t kept,
    const int64_t* teacher_rows, int64_t num_teacher_rows, int renormalize, float temperature, const float* grad_ce,
    const float* grad_kl, float* ce, float* kl, float* accept, int64_t* argmax, float* stats, void* workspace,
    void* grad_logits, int64_t grad_stride, int32_t* status_words, void* stream) {
  if (const int e = check_distill(dtype, rows, vocab, row_stride, token_dtype, kept, teacher_rows, num_teacher_rows,
                                  temperature))
    return e;
  if (grad_stride < vocab)
    return set_error(ASPEC_ERR_INVALID, "top-logit distillation needs a vocabulary and rows at least as far apart");
  if (rows == 0) return ASPEC_OK;
  Args a = make_args(logits, dtype, rows, vocab, row_stride, targets, ignore_index, teacher_tokens, token_dtype,
                     teacher_logprobs, kept, teacher_rows, num_teacher_rows, renormalize, temperature, ce, kl, accept,
                     argmax, stats, workspace, status_words);
  a.g_ce = grad_ce;
  a.g_kl = grad_kl;
  a.dx = grad_logits;
  a.dx_stride = grad_stride;
  const bool fits = topk_distill_fused_fits(vocab, per_chunk_of(dtype));
  if (!logits || !teacher_tokens || !teacher_logprobs || (targets && !ce) || !kl || !accept ||
      !grad_logits || (grad_ce && !targets) || (!fits && (!stats || (a.parts > 1 && !workspace))))
    return null_pointer();
  if (grad_logits == logits && grad_stride != row_stride)
    return set_error(ASPEC_ERR_INVALID, "a gradient in place has the logits' row stride");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (fits) {
    a.parts = 1;
    a.part_chunks = static_cast<int>(vocab / per_chunk_of(dtype));
    topk_distill_fused_launch(dtype, two_sums(a), a, st);
  } else {
    run_fwd(dtype, a, st);
    run_bwd(dtype, a, st);
  }
  return check_launch("topk_distill_fused_kernel");
}
