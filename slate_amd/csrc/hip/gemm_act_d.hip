#include "gemm_act_launch.hpp"
namespace slate_hip {
template void gemm_act<double>(GemmActArgs, char, char, const GemmActPlan&, hipStream_t);
}
