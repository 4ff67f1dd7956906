// Distillation from a teacher's best tokens, losses and gradient in one pass: a workgroup holds a
// whole row in registers, takes its statistics and writes the row's gradient from there. Each logit
// is read once and written once (the formulas are in topk_distill.h).
//
// HBM-bound up to 32768 16-bit logits to a row: 8192 x 32000 bf16, 64 kept tokens, 195 us for 1084 MB
// (5.6 TB/s, a copy's rate; forward and gradient apart take 310). Longer rows fill 80 of a thread's 128
// registers: up to 81920 logits 512 threads, two workgroups to a CU (8192 x 36000 244 us, 4.8 TB/s; 364
// with 1024 threads of 10 chunks, one to a CU), beyond that 1024, one to a CU, so that nothing is read
// while a row is reduced and written: 1536 x 151936 bf16 220 us (952 MB, 4.3 TB/s; forward and gradient
// apart read 480 MB more). Loading the next row ahead spilled 28-41 registers, whose reloads wait for
// those loads: 288.
#include "topk_distill.h"

namespace aspec {
namespace {

using namespace distill;

template <typename E, int T, int NV, bool TWO>
__global__ __launch_bounds__(T, min_waves(NV)) void topk_distill_fused_kernel(Args a) {
  __shared__ Kept<T> kept;
  __shared__ float s_m[T / 64], s_s[T / 64], s_s1[T / 64];
  __shared__ uint64_t s_arg;
  __shared__ Factors s_factors;
  const int64_t row = unit_of_block();
  if (row < a.rows)
    forward_unit<E, T, NV, TWO, true>(a, row, kept, s_m, s_s, s_s1, s_arg, s_factors);
}

template <typename E, int T, int NV>
void launch(const Args& a, bool two, hipStream_t stream) {
  const dim3 grid = grid_of(a.rows);
  if (two) topk_distill_fused_kernel<E, T, NV, true><<<grid, T, 0, stream>>>(a);
  else topk_distill_fused_kernel<E, T, NV, false><<<grid, T, 0, stream>>>(a);
}

template <typename E>
void launch_type(const Args& a, bool two, hipStream_t stream) {
  if (a.part_chunks <= 64 * 4) launch<E, 64, 4>(a, two, stream);
  else if (a.part_chunks <= 256 * 4) launch<E, 256, 4>(a, two, stream);
  else if (a.part_chunks <= 512 * 4) launch<E, 512, 4>(a, two, stream);
  else if (a.part_chunks <= 512 * 8) launch<E, 512, 8>(a, two, stream);
  else if (a.part_chunks <= 512 * 20) launch<E, 512, 20>(a, two, stream);
  else launch<E, 1024, 20>(a, two, stream);
}

}  // namespace

// 20 chunks a thread (80 registers) in the largest workgroup: 163840 16-bit logits, 81920 of fp32.
bool topk_distill_fused_fits(int64_t V, int per_chunk) { return V / per_chunk <= 1024 * 20; }

void topk_distill_fused_launch(int dtype, bool two, const distill::Args& a, hipStream_t stream) {
  if (dtype == ASPEC_MASK_BF16) launch_type<Bf16>(a, two, stream);
  else if (dtype == ASPEC_MASK_F16) launch_type<F16>(a, two, stream);
  else launch_type<F32>(a, two, stream);
}

}  // namespace aspec
