#include "gemm_act_launch.hpp"
namespace slate_hip {
template i64 gemm_act<float>(GemmActArgs, char, char, hipStream_t);
}
