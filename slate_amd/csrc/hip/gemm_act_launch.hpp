// Launcher of the fused-epilogue products (one translation unit per type).
#pragma once
#include "gemm_act.hpp"

namespace slate_hip {

namespace {

template <typename T, bool AKC, bool BKC, int BM, int BN, int WVM, int WVN, int S, bool GATED, int DMA>
void ga_launch(const GemmActArgs& a, hipStream_t s) {
    constexpr int BMI = GATED ? BM / 2 : BM, LDS = GaEpi<T, BM, BN, WVM, WVN, S>::LDS;
    auto kern = gemm_act_kernel<T, AKC, BKC, BM, BN, WVM, WVN, S, GATED, DMA>;
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
        if (tile == 0) return ga_launch<T, AKC, BKC, 256, 256, 2, 4, 2, GATED, DMA>(a, s);
    if constexpr (sizeof(T) == 2 && DMA == 16)
        if (tile == 1) return ga_launch<T, AKC, BKC, 128, 128, 2, 2, 2, GATED, DMA>(a, s);
    if constexpr (sizeof(T) == 2 && DMA == 16)
        if (tile == 4) return ga_launch<T, AKC, BKC, 64, 64, 2, 2, 3, GATED, DMA>(a, s);
    if constexpr (sizeof(T) >= 4)
        if (tile == 5) return ga_launch<T, AKC, BKC, 64, 32, 2, 2, 2, GATED, DMA>(a, s);
    if (tile == 2) return ga_launch<T, AKC, BKC, 64, 64, 2, 2, 2, GATED, DMA>(a, s);
    return ga_launch<T, AKC, BKC, 128, 16, 4, 1, 2, GATED, DMA>(a, s);
}

template <typename T, bool GATED, int DMA>
void ga_layout(const GemmActArgs& a, bool akc, bool bkc, int tile, hipStream_t s) {
    if (akc) bkc ? ga_tile<T, true, true, GATED, DMA>(a, tile, s) : ga_tile<T, true, false, GATED, DMA>(a, tile, s);
    else bkc ? ga_tile<T, false, true, GATED, DMA>(a, tile, s) : ga_tile<T, false, false, GATED, DMA>(a, tile, s);
}

// One operand as it is stored: columns of len elements
struct GaOperand {
    const void** ptr;
    i64* ld;
    i64 len, cols;
    bool kc;                 // columns run along k
    bool bad = false;        // rows not on 16 bytes, or 32-bit offsets too short
    i64 at = -1;             // its place in the workspace
    bool fits(i64 l, int es) const { return (kc ? 256 : 128 / es) * l * es < (i64)1 << 31; }
    i64 whole(int es) const { return (len * es + 15) / 16 * (16 / es); }
};

// can all operands that need it be laid out anew?
inline bool ga_packed(const GaOperand* op, int n, int es) {
    for (int i = 0; i < n; ++i)
        if (op[i].bad && !op[i].fits(op[i].whole(es), es)) return false;
    return true;
}

// their places behind the first `bytes` of the workspace; -> its size.  (Both
// products of a pair often share an operand, which is laid out once.)
inline i64 ga_place(GaOperand* op, int n, int es, i64 bytes) {
    for (int i = 0; i < n; ++i) {
        if (!op[i].bad) continue;
        for (int j = 0; j < i && op[i].at < 0; ++j)
            if (op[j].at >= 0 && *op[j].ptr == *op[i].ptr && *op[j].ld == *op[i].ld && op[j].len == op[i].len &&
                op[j].cols == op[i].cols)
                op[i].at = op[j].at;
        if (op[i].at >= 0) continue;
        op[i].at = bytes;
        bytes += (op[i].whole(es) * op[i].cols * es + 255) / 256 * 256;
    }
    return bytes;
}

template <typename T> void ga_pack(GaOperand* op, int n, char* ws, hipStream_t s) {
    for (int i = 0; i < n; ++i) {
        if (op[i].at < 0) continue;
        T* y = reinterpret_cast<T*>(ws + op[i].at);
        bool done = false;
        for (int j = 0; j < i; ++j) done = done || op[j].at == op[i].at;
        const i64 ld = op[i].whole(sizeof(T)), nv = ld * (i64)sizeof(T) / 16;
        if (!done && nv * op[i].cols)
            hipLaunchKernelGGL((ga_pack_kernel<T>), dim3((unsigned)((nv * op[i].cols + 1023) / 1024)), dim3(256), 0, s,
                               static_cast<const T*>(*op[i].ptr), *op[i].ld, y, op[i].len, op[i].cols);
        HIP_LAUNCH_CHECK();
        *op[i].ptr = y;
        *op[i].ld = ld;
    }
}

template <typename T> void ga_skinny(const GemmActArgs& a, bool gated, hipStream_t s) {
    constexpr int NW = 8;
    const dim3 grid((unsigned)((a.m + 15) / 16));
    if (gated) hipLaunchKernelGGL((gemm_act_skinny_kernel<T, true, NW>), grid, dim3(64 * NW), 0, s, a);
    else hipLaunchKernelGGL((gemm_act_skinny_kernel<T, false, NW>), grid, dim3(64 * NW), 0, s, a);
    HIP_LAUNCH_CHECK();
}

}  // namespace

template <typename T>
i64 gemm_act(GemmActArgs a, char ta, char tb, hipStream_t s) {
    constexpr int ES = sizeof(T), E = 16 / ES, KB = 128 / ES;
    if (a.m <= 0 || a.n <= 0) return 0;
    if (a.mode != GA_SUM) a.terms = 1;
    const bool gated = a.mode == GA_GATED, akc = ta != 'N', bkc = tb == 'N';
    const int na = a.mode == GA_SUM ? a.terms : a.mode == GA_PLAIN ? 1 : 2;
    const int nb = a.mode == GA_SUM ? a.terms : a.mode == GA_PAIR ? 2 : 1;
    // LDS-DMA moves 16 bytes from 16-byte-aligned addresses at 32-bit offsets
    // inside a tile; a slab whose last vector would pass the end of the last
    // column goes through registers, as the ragged end of K does
    bool dma = true, small = true;       // 32-bit offsets: `small`
    GaOperand op[8];
    int nop = 0;
    auto look = [&](const void*& q, i64& ld, bool kc, i64 rows) {
        GaOperand x{&q, &ld, kc ? a.k : rows, kc ? rows : a.k, kc};
        const bool fits = x.fits(ld, ES);
        x.bad = !fits || (uintptr_t)q % 16 != 0 || (ld * ES) % 16 != 0;
        small = small && fits;
        dma = dma && !x.bad;
        op[nop++] = x;
    };
    for (int i = 0; i < na; ++i) look(a.A[i], a.lda[i], akc, a.m);
    for (int i = 0; i < nb; ++i) look(a.B[i], a.ldb[i], bkc, a.n);
    const bool pack = ES == 2 && !dma && gemm_act_pack(a.mode, a.terms, a.m, a.n, a.k) && ga_packed(op, nop, ES);
    const GemmActPlan p = gemm_act_plan(ES, a.mode, a.terms, a.m, a.n, a.k, akc, bkc, dma || pack);
    if (p.tile < 0) {
        if (!a.plan) ga_skinny<T>(a, gated, s);
        return 0;
    }
    const bool regs = !dma && !pack && !(ES >= 4 && small);
    if (regs)            // through registers: columns of 16 bytes or more
        for (int i = 0; i < nop; ++i) op[i].bad = op[i].len < E;
    i64 bytes = (p.bytes + 255) / 256 * 256;
    if (pack || regs) bytes = ga_place(op, nop, ES, bytes);
    if (a.plan || (bytes && !a.part)) return bytes;
    if (pack || regs) ga_pack<T>(op, nop, static_cast<char*>(a.part), s);
    dma = dma || pack;
    a.lenA = op[0].at < 0 ? op[0].len : op[0].whole(ES);
    a.lenB = op[na].at < 0 ? op[na].len : op[na].whole(ES);
    a.kfull = a.k / KB * KB;
    for (int i = 0; i < nop; ++i)
        if (!op[i].kc && op[i].len % E && op[i].at < 0 && a.k) a.kfull = std::min<i64>(a.kfull, (a.k - 1) / KB * KB);
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
