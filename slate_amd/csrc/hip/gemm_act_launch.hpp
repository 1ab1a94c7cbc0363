// Launcher of the fused-epilogue products (one translation unit per type).
#pragma once
#include "gemm_act.hpp"

namespace slate_hip {

namespace {

template <typename T, bool AKC, bool BKC, int BM, int BN, int WVM, int WVN, int KBB, int S, bool GATED, int DMA>
void ga_launch(const GemmActArgs& a, hipStream_t s) {
    constexpr int BMI = GATED ? BM / 2 : BM, LDS = GaEpi<T, BM, BN, WVM, WVN, KBB, S>::LDS;
    auto kern = gemm_act_kernel<T, AKC, BKC, BM, BN, WVM, WVN, KBB, S, GATED, DMA>;
    if constexpr (LDS > 65536)
        HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                      LDS));
    const i64 gx = ((a.m + BMI - 1) / BMI) * ((a.n + BN - 1) / BN);
    hipLaunchKernelGGL(kern, dim3((unsigned)gx, (unsigned)a.splits, a.mode == GA_PAIR ? 2 : 1),
                       dim3(64 * WVM * WVN), LDS, s, a);
    HIP_LAUNCH_CHECK();
}

template <typename T, bool AKC, bool BKC, bool GATED, int DMA>
void ga_tile(const GemmActArgs& a, int tile, hipStream_t s) {
    if constexpr (sizeof(T) == 2 && DMA == 16)
        if (tile == 0) return ga_launch<T, AKC, BKC, 256, 256, 2, 4, 128, 2, GATED, DMA>(a, s);
    if constexpr (sizeof(T) == 2)
        if (tile == 1) return ga_launch<T, AKC, BKC, 128, 128, 2, 2, 128, 2, GATED, DMA>(a, s);
    if (tile <= 2) return ga_launch<T, AKC, BKC, 64, 64, 2, 2, 128, 2, GATED, DMA>(a, s);
    return ga_launch<T, AKC, BKC, 128, 16, 4, 1, 128, 2, GATED, DMA>(a, s);
}

template <typename T, bool GATED, int DMA>
void ga_layout(const GemmActArgs& a, bool akc, bool bkc, int tile, hipStream_t s) {
    if (akc) bkc ? ga_tile<T, true, true, GATED, DMA>(a, tile, s) : ga_tile<T, true, false, GATED, DMA>(a, tile, s);
    else bkc ? ga_tile<T, false, true, GATED, DMA>(a, tile, s) : ga_tile<T, false, false, GATED, DMA>(a, tile, s);
}

template <typename T, int NF> void ga_skinny(const GemmActArgs& a, bool gated, hipStream_t s) {
    constexpr int NW = 8;
    const dim3 grid((unsigned)((a.m + 15) / 16));
    if (gated) hipLaunchKernelGGL((gemm_act_skinny_kernel<T, NF, true, NW>), grid, dim3(64 * NW), 0, s, a);
    else hipLaunchKernelGGL((gemm_act_skinny_kernel<T, NF, false, NW>), grid, dim3(64 * NW), 0, s, a);
    HIP_LAUNCH_CHECK();
}

}  // namespace

template <typename T>
i64 gemm_act(GemmActArgs a, char ta, char tb, hipStream_t s) {
    constexpr int ES = sizeof(T), E = 16 / ES, KB = 128 / ES;
    if (a.m <= 0 || a.n <= 0) return 0;
    const bool gated = a.mode == GA_GATED, akc = ta != 'N', bkc = tb == 'N';
    const int na = a.mode == GA_PLAIN ? 1 : 2, nb = a.mode == GA_SUM || a.mode == GA_PAIR ? 2 : 1;
    // LDS-DMA moves 16 bytes from 16-byte-aligned addresses at 32-bit offsets
    // inside a tile; a slab whose last vector would pass the end of the last
    // column goes through registers, as the ragged end of K does
    bool dma = true, small = true;       // 32-bit offsets: `small`
    a.kfull = a.k / KB * KB;
    auto look = [&](const void* q, i64 ld, bool kc, i64 rows) {
        small = small && (kc ? 256 : KB) * ld * ES < (i64)1 << 31;
        dma = dma && small && (uintptr_t)q % 16 == 0 && (ld * ES) % 16 == 0;
        if (!kc && rows % E && a.k) a.kfull = std::min<i64>(a.kfull, (a.k - 1) / KB * KB);
    };
    for (int i = 0; i < na; ++i) look(a.A[i], a.lda[i], akc, a.m);
    for (int i = 0; i < nb; ++i) look(a.B[i], a.ldb[i], bkc, a.n);
    const GemmActPlan p = gemm_act_plan(ES, a.mode, a.m, a.n, a.k, akc, bkc, dma);
    if (p.bytes && !a.part) return p.bytes;
    if (p.tile < 0) {
        ga_skinny<T, 1>(a, gated, s);
        return 0;
    }
    a.splits = p.splits;
    a.per_split = p.per_split;
    a.ldp = p.ldp;
    a.nsteps = (int)((a.k + KB - 1) / KB);
    if (dma) {
        gated ? ga_layout<T, true, 16>(a, akc, bkc, p.tile, s) : ga_layout<T, false, 16>(a, akc, bkc, p.tile, s);
    } else if (ES >= 4 && small) {
        a.kfull = a.k / KB * KB;           // no access passes an element
        if constexpr (ES >= 4)
            gated ? ga_layout<T, true, 4>(a, akc, bkc, p.tile, s) : ga_layout<T, false, 4>(a, akc, bkc, p.tile, s);
    } else {
        gated ? ga_layout<T, true, 0>(a, akc, bkc, p.tile, s) : ga_layout<T, false, 0>(a, akc, bkc, p.tile, s);
    }
    if (p.splits > 1) {
        constexpr int V = 16 / (int)sizeof(typename ga_traits<T>::acc);
        const dim3 grid((unsigned)(((a.m + V - 1) / V * a.n + 63) / 64), 1, a.mode == GA_PAIR ? 2 : 1);
        if (gated) hipLaunchKernelGGL((gemm_act_join_kernel<T, true>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((gemm_act_join_kernel<T, false>), grid, dim3(256), 0, s, a);
        HIP_LAUNCH_CHECK();
    }
    return 0;
}

}  // namespace slate_hip
