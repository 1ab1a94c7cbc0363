// Copies to, from and between the 16-bit element types (bf16, f16): the
// precision conversion of matrices that the fused products read and write.
// Memory bound; rows are coalesced, a transposed copy goes through LDS.
#include "ffn.hpp"

namespace slate_hip {

namespace {

__device__ inline bool in_uplo(char uplo, i64 i, i64 j) {
    return uplo == 'L' ? i >= j : (uplo == 'U' ? i <= j : true);
}
// one rounding: straight from 64 to 16 bits, and between the 16-bit types
// through 32, which holds either exactly
template <typename Ts, typename Td> __device__ inline Td cvt16(Ts x) {
    if constexpr (sizeof(Ts) == 2 && sizeof(Td) == 2 && !std::is_same<Ts, Td>::value) return (Td)(float)x;
    else return (Td)x;
}

// A whole matrix: 8 elements a thread and access, two of them in flight
// (8192^2 bf16 -> f32 74 us, 5.4 TB/s; one element a thread 147).
template <typename T, int V> struct vec_of { typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T)))); };
template <typename Ts, typename Td>
__global__ void __launch_bounds__(256) copy16_whole_kernel(i64 m, i64 n, const Ts* A, i64 lda, Td* B, i64 ldb) {
    constexpr int E = 8, U = 2;
    using vS = typename vec_of<Ts, E>::type;
    using vD = typename vec_of<Td, E>::type;
    const i64 nv = (m + E - 1) / E, first = (i64)blockIdx.x * (256 * U), c0 = first / nv;
    const uint32_t r0 = (uint32_t)(first - c0 * nv) + threadIdx.x, nv32 = (uint32_t)nv;
    vS x[U];
    #pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t r = r0 + u * 256, q = r / nv32;
        const i64 j = c0 + q, i = (i64)(r - q * nv32) * E;
        if (j < n && i + E <= m) x[u] = *reinterpret_cast<const vS*>(A + i + j * lda);
    }
    #pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t r = r0 + u * 256, q = r / nv32;
        const i64 j = c0 + q, i = (i64)(r - q * nv32) * E;
        if (j >= n) continue;
        if (i + E <= m) {
            vD y;
            #pragma unroll
            for (int e = 0; e < E; ++e) y[e] = cvt16<Ts, Td>((Ts)x[u][e]);
            *reinterpret_cast<vD*>(B + i + j * ldb) = y;
        } else {
            for (i64 k = i; k < m; ++k) B[k + j * ldb] = cvt16<Ts, Td>(A[k + j * lda]);
        }
    }
}

template <typename Ts, typename Td>
__global__ void __launch_bounds__(256) copy16_kernel(char uplo, i64 m, i64 n, const Ts* A, i64 lda, Td* B, i64 ldb) {
    const i64 i = (i64)blockIdx.x * 256 + threadIdx.x;
    if (i >= m) return;
    for (i64 j = blockIdx.y; j < n; j += gridDim.y)
        if (in_uplo(uplo, i, j)) B[i + j * ldb] = cvt16<Ts, Td>(A[i + j * lda]);
}

template <typename Ts, typename Td>
__global__ void __launch_bounds__(256) transpose16_kernel(char uplo, i64 m, i64 n, const Ts* A, i64 lda, Td* B, i64 ldb) {
    __shared__ Td tile[32][33];
    const int tx = threadIdx.x, ty = threadIdx.y;
    const i64 bi = (i64)blockIdx.x * 32;
    for (i64 bj = (i64)blockIdx.y * 32; bj < n; bj += (i64)gridDim.y * 32) {
        for (int r = ty; r < 32; r += 8)
            if (bj + tx < n && bi + r < m) tile[r][tx] = cvt16<Ts, Td>(A[bj + tx + (bi + r) * lda]);
        __syncthreads();
        for (int c = ty; c < 32; c += 8)
            if (bi + tx < m && bj + c < n && in_uplo(uplo, bi + tx, bj + c)) B[bi + tx + (bj + c) * ldb] = tile[tx][c];
        __syncthreads();
    }
}

}  // namespace

template <typename Ts, typename Td>
void gecopy16(char uplo, char trans, i64 m, i64 n, const Ts* A, i64 lda, Td* B, i64 ldb, hipStream_t s) {
    if (m <= 0 || n <= 0) return;
    if (trans == 'N' && uplo != 'L' && uplo != 'U') {
        const i64 vectors = (m + 7) / 8 * n;
        hipLaunchKernelGGL((copy16_whole_kernel<Ts, Td>), dim3((unsigned)((vectors + 511) / 512)), dim3(256), 0, s, m, n, A,
                           lda, B, ldb);
    } else if (trans == 'N') {
        const dim3 grid((unsigned)((m + 255) / 256), (unsigned)std::min<i64>(n, 4096));
        hipLaunchKernelGGL((copy16_kernel<Ts, Td>), grid, dim3(256), 0, s, uplo, m, n, A, lda, B, ldb);
    } else {
        const dim3 grid((unsigned)((m + 31) / 32), (unsigned)std::min<i64>((n + 31) / 32, 65535));
        hipLaunchKernelGGL((transpose16_kernel<Ts, Td>), grid, dim3(32, 8), 0, s, uplo, m, n, A, lda, B, ldb);
    }
    HIP_LAUNCH_CHECK();
}

#define INST(A, B) template void gecopy16<A, B>(char, char, i64, i64, const A*, i64, B*, i64, hipStream_t);
#define INSTS(A) INST(A, __bf16) INST(A, _Float16) INST(A, float) INST(A, double)
INSTS(__bf16) INSTS(_Float16) INSTS(float) INSTS(double)

}  // namespace slate_hip
