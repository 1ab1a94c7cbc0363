#include "gemm_act_launch.hpp"
namespace slate_hip {
template void gemm_act<_Float16>(GemmActArgs, char, char, const GemmActPlan&, hipStream_t);
}
