// Launcher of the fused-epilogue products (one translation unit per type).
#pragma once
#include "gemm_act.hpp"

namespace slate_hip {

namespace {

template <typename T, bool AKC, bool BKC, int BM, int BN, int WVM, int WVN, bool GATED>
void ga_launch(const GemmActArgs& a, hipStream_t s) {
    constexpr int BMI = GATED ? BM / 2 : BM, LDS = GaEpi<T, BM, BN, WVM, WVN>::LDS;
    auto kern = gemm_act_kernel<T, AKC, BKC, BM, BN, WVM, WVN, GATED>;
    if constexpr (LDS > 65536)
        HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                      LDS));
    const i64 gx = ((a.m + BMI - 1) / BMI) * ((a.n + BN - 1) / BN);
    hipLaunchKernelGGL(kern, dim3((unsigned)gx, (unsigned)a.splits, a.mode == GA_PAIR ? 2 : 1),
                       dim3(64 * WVM * WVN), LDS, s, a);
    HIP_LAUNCH_CHECK();
}

template <typename T, bool AKC, bool BKC, bool GATED>
void ga_tile(const GemmActArgs& a, int tile, hipStream_t s) {
    if constexpr (sizeof(T) == 2)
        if (tile == 0) return ga_launch<T, AKC, BKC, 256, 256, 2, 4, GATED>(a, s);
    if (tile <= 1) return ga_launch<T, AKC, BKC, 128, 128, 2, 2, GATED>(a, s);
    if (tile == 2) return ga_launch<T, AKC, BKC, 64, 64, 2, 2, GATED>(a, s);
    return ga_launch<T, AKC, BKC, 128, 16, 4, 1, GATED>(a, s);
}

template <typename T, bool GATED>
void ga_layout(const GemmActArgs& a, bool akc, bool bkc, int tile, hipStream_t s) {
    if (akc) bkc ? ga_tile<T, true, true, GATED>(a, tile, s) : ga_tile<T, true, false, GATED>(a, tile, s);
    else bkc ? ga_tile<T, false, true, GATED>(a, tile, s) : ga_tile<T, false, false, GATED>(a, tile, s);
}

}  // namespace

template <typename T>
void gemm_act(GemmActArgs a, char ta, char tb, const GemmActPlan& p, hipStream_t s) {
    constexpr int ES = sizeof(T), E = 16 / ES, KB = 128 / ES;
    if (a.m <= 0 || a.n <= 0) return;
    const bool gated = a.mode == GA_GATED, akc = ta != 'N', bkc = tb == 'N';
    const int na = a.mode == GA_PLAIN ? 1 : 2, nb = a.mode == GA_SUM || a.mode == GA_PAIR ? 2 : 1;
    auto on = [](const void* q, i64 ld, int bytes) {
        return ((uintptr_t)q % bytes) == 0 && (ld * ES) % bytes == 0;
    };
    // LDS-DMA moves 16 bytes from 16-byte-aligned addresses at 32-bit offsets
    // inside a tile; a slab whose last chunk would pass the end of the last
    // column goes through registers, as the ragged end of K does
    bool dma = true;
    a.nsteps = (int)((a.k + KB - 1) / KB);
    a.nfull = (int)(a.k / KB);
    auto look = [&](const void* q, i64 ld, bool kc, i64 rows) {
        dma = dma && on(q, ld, 16) && (kc ? 256 : KB) * ld * ES < (i64)1 << 31;
        if (!kc && rows % E) a.nfull = std::min<int>(a.nfull, (int)((a.k - 1) / KB));
    };
    for (int i = 0; i < na; ++i) look(a.A[i], a.lda[i], akc, a.m);
    for (int i = 0; i < nb; ++i) look(a.B[i], a.ldb[i], bkc, a.n);
    if (!dma) a.nfull = 0;
    auto row = [&](const void* q, i64 ld) { return !q || on(q, ld, 16); };
    a.vec = (row(a.C[0], a.ldc[0]) && row(a.C[1], a.ldc[1]) ? 1 : 0) | (row(a.R, a.ldr) ? 2 : 0) |
            (row(a.Z[0], a.ldz[0]) && row(a.Z[1], a.ldz[1]) ? 4 : 0) |
            (a.incb == 1 && (uintptr_t)a.bias % 16 == 0 ? 8 : 0);
    a.splits = p.splits;
    a.per_split = p.per_split;
    a.ldp = p.ldp;
    if (gated) ga_layout<T, true>(a, akc, bkc, p.tile, s);
    else ga_layout<T, false>(a, akc, bkc, p.tile, s);
    if (p.splits > 1) {
        const i64 mv = (a.m + E - 1) / E;
        const dim3 grid((unsigned)((mv * a.n + 255) / 256), 1, a.mode == GA_PAIR ? 2 : 1);
        if (gated) hipLaunchKernelGGL((gemm_act_join_kernel<T, true>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((gemm_act_join_kernel<T, false>), grid, dim3(256), 0, s, a);
        HIP_LAUNCH_CHECK();
    }
}

}  // namespace slate_hip
