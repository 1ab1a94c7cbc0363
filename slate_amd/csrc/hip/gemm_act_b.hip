#include "gemm_act_launch.hpp"
namespace slate_hip {
template i64 gemm_act<__bf16>(GemmActArgs, char, char, hipStream_t);
}
