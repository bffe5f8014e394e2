// Causal attention with tiles of 256 rows (qvl_decoder_wide.h), in a file of its own for its compiler flags.
#include "qvl_decoder_wide.h"

namespace qvl {

template <int D>
__global__ __launch_bounds__(256, 1) void causal_wide_kernel(AttnParams P, const int32_t* items, int n_parts) {
  using U = WideUnit<D>;
  __shared__ __attribute__((aligned(16))) char smem[U::kLds];
  Item x;
  if (!item_of(P, items, n_parts, U::kRows, U::kBN, x)) return;
  Wave<bf16, D> A, B;
  U::run_all(P, x.u, A, B, x.u.row0, smem, x.t0, x.t1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto write = [&](const Wave<bf16, D>& w, int first) {
    const int r = first + (threadIdx.x & 31);
    const int64_t at = (int64_t)max(x.slot, 0) * U::kRows + r;
    write_rows<bf16, D>(P, x.u, w, smem + wave * kWriteLds, x.u.row0 + r, x.slot >= 0 ? P.part_o + at * D : nullptr, P.part_ml + at, w.lim > x.t0 * U::kBN);
  };
  write(A, wave * 64);
  write(B, wave * 64 + 32);
}

void launch_causal_wide(void* stream, int32_t head_dim, const AttnParams& P, const int32_t* items, int64_t n_items, int64_t n_parts) {
  const dim3 grid((unsigned)n_items);
  if (head_dim == 128) hipLaunchKernelGGL(causal_wide_kernel<128>, grid, dim3(256), 0, (hipStream_t)stream, P, items, (int)n_parts);
  else hipLaunchKernelGGL(causal_wide_kernel<64>, grid, dim3(256), 0, (hipStream_t)stream, P, items, (int)n_parts);
}

}  // namespace qvl
