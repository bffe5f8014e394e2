// Causal attention with tiles of 256 rows (qvl_decoder_wide.h), in a file of its own for its compiler flags.
#include "qvl_decoder_wide.h"

namespace qvl {

template <int D>
__global__ __launch_bounds__(256, 1) void causal_wide_kernel(AttnParams P, const int32_t* items, int n_whole) {
  using U = WideUnit<D>;
  __shared__ __attribute__((aligned(16))) char smem[U::kLds];
  const int32_t* it = items + 8 * (int64_t)blockIdx.x;
  const int q0 = it[0], n_new = it[1], len = it[2], row0 = it[3], kvh = it[4] & kItemHeadMask;
  const int part = (it[4] >> kItemPartShift) & 0xff, parts = (it[4] >> kItemPartsShift) & 0xff, slot = it[5];
  const int64_t start = (int64_t)(((uint64_t)(uint32_t)it[7] << 32) | (uint32_t)it[6]);
  if (q0 < 0 || n_new <= 0 || row0 < 0 || kvh >= P.hkv || q0 + (int64_t)n_new > P.n_tokens || len < 0 || start < 0 ||
      start > P.kv_rows - len || row0 >= n_new * P.group || (parts && (part >= parts || slot < 0 || slot >= (int)gridDim.x - n_whole))) return;
  const Unit u{P.k.p + start * P.k.row + kvh * P.k.head, P.v.p + start * P.v.row + kvh * P.v.head, len, len - n_new + 1, q0,
               n_new * P.group, row0, kvh};
  const int last = min(row0 + U::kRows, u.rows) - 1;
  const int k_hi = max(min(u.lim0 + (int)((uint32_t)last / (uint32_t)P.group), len), 0);
  const int n_t = (k_hi + U::kBN - 1) / U::kBN;
  const int t0 = parts ? (int)((int64_t)n_t * part / parts) : 0, t1 = parts ? (int)((int64_t)n_t * (part + 1) / parts) : n_t;
  Wave<bf16, D> A, B;
  U::run_all(P, u, A, B, row0, smem, t0, t1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto write = [&](const Wave<bf16, D>& w, int first) {
    const int r = first + (threadIdx.x & 31);
    const int64_t at = (int64_t)slot * U::kRows + r;
    write_rows<bf16, D>(P, u, w, smem + wave * kWriteLds, row0 + r, parts ? P.part_o + at * D : nullptr, P.part_ml + at, w.lim > t0 * U::kBN);
  };
  write(A, wave * 64);
  write(B, wave * 64 + 32);
}

void launch_causal_wide(void* stream, int32_t head_dim, const AttnParams& P, const int32_t* items, int64_t n_items, int64_t n_whole) {
  const dim3 grid((unsigned)n_items);
  if (head_dim == 128) hipLaunchKernelGGL(causal_wide_kernel<128>, grid, dim3(256), 0, (hipStream_t)stream, P, items, (int)n_whole);
  else hipLaunchKernelGGL(causal_wide_kernel<64>, grid, dim3(256), 0, (hipStream_t)stream, P, items, (int)n_whole);
}

}  // namespace qvl
