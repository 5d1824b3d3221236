// Products of linear_act cut along K: partial sums in fp32, joined by finish_kernel (linear_act.cu) in the order of the slices.
#define B200GRU_LINEAR_GEMM_IMPL
#include "linear_gemm.cuh"

namespace b200gru {
namespace lin {

template <>
int launch_gemm<void>(const Gemm& g, const Plan& plan, cudaStream_t st) {
  return g.planes == 2 ? launch_plan<2, void>(g, plan, st) : launch_plan<1, void>(g, plan, st);
}

template <>
int gemm_status<void>(int reset) { return unit_status(reset); }

}  // namespace lin
}  // namespace b200gru
