// Products of linear_act with results in __half.
#define B200GRU_LINEAR_GEMM_IMPL
#include "linear_gemm.cuh"

namespace b200gru {
namespace lin {

template <>
int launch_gemm<__half>(const Gemm& g, const Plan& plan, cudaStream_t st) {
  return launch_plan<1, __half>(g, plan, st);
}

template <>
int gemm_status<__half>(int reset) { return unit_status(reset); }

}  // namespace lin
}  // namespace b200gru
