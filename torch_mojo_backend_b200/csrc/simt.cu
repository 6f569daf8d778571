// The exact-fp32 kernels on fp32 storage, and the choice by storage type.
#include "simt.cuh"

namespace b200fa {

extern template cudaError_t simt_fwd<__nv_bfloat16>(const FwdParams&, cudaStream_t);
extern template cudaError_t simt_bwd<__nv_bfloat16>(const BwdParams&, cudaStream_t);
extern template cudaError_t simt_fwd<__half>(const FwdParams&, cudaStream_t);
extern template cudaError_t simt_bwd<__half>(const BwdParams&, cudaStream_t);

cudaError_t launch_fwd_simt(const FwdParams& p, int dtype, cudaStream_t stream, int* launches) {
  cudaError_t e = cudaErrorInvalidValue;
  if (dtype == kF32) e = simt_fwd<float>(p, stream);
  else if (dtype == kBF16) e = simt_fwd<__nv_bfloat16>(p, stream);
  else if (dtype == kF16) e = simt_fwd<__half>(p, stream);
  if (e == cudaSuccess && launches) *launches += 1;
  return e;
}

cudaError_t launch_bwd_simt(const BwdParams& p, int dtype, cudaStream_t stream, int* launches) {
  cudaError_t e = cudaErrorInvalidValue;
  if (dtype == kF32) e = simt_bwd<float>(p, stream);
  else if (dtype == kBF16) e = simt_bwd<__nv_bfloat16>(p, stream);
  else if (dtype == kF16) e = simt_bwd<__half>(p, stream);
  if (e == cudaSuccess && launches) *launches += 3 + (p.window && p.sink_chunks > 1);
  return e;
}

// B200, us, one block per tile with sinks / shared: B3 Hq8 Hkv4 S777 D64, window 200, 3 sinks: dK/dV kernel 170 / 92 and 2.7 for the sums
int simt_sink_chunks(const BwdParams& p, int* tile_rows) {
  const int rows = *tile_rows = key_rows(p);
  if (!p.window) return 1;
  const int64_t m_tiles = (p.S + kBN - 1) / kBN, n_tiles = (p.Sk + rows - 1) / rows, group = p.Hq / p.Hkv;
  return sink_chunks_for(static_cast<int64_t>(p.B) * p.Hkv, n_tiles, std::min<int64_t>(n_tiles, (p.sinks + rows - 1) / rows), group * m_tiles,
                         group * std::min<int64_t>(m_tiles, (p.window + rows - 1) / kBN + 2), 2 * 148, 4);
}

}  // namespace b200fa
