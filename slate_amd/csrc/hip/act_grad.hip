// Gradient through the activation of a feed-forward product, one pass:
//   dZ1 = dC o Z2 o act'(Z1), dZ2 = dC o act(Z1)     (gated)
//   dZ  = dC o act'(Z), db = row (or column) sums of dZ
// Memory bound: each of dC, Z1, Z2 is read once and dZ1, dZ2 written once, in
// 16-byte accesses where rows allow it.  dZ is rounded to the operands' type,
// which the MFMA of the two products that read it takes, and, where the caller
// wants it, what that rounding leaves over as a second matrix of the type; the
// bias gradient sums the unrounded values in 32 (64) bits, per chunk in registers, the
// chunks in order: no atomics, the same result on every run.  4096 x 8192 bf16:
// 49 us plain (4.1 TB/s), 69 us gated (4.9 TB/s).
#include "gemm_act.hpp"

namespace slate_hip {

namespace {

// d less its rounding to T (an infinity or a NaN is whole in the rounded value)
template <typename T, typename R> __device__ inline R ag_rest(R d) {
    const R h = (R)(T)d;
    return fabs(h) < (R)__builtin_huge_val() ? d - h : R(0);
}

// grid.x: blocks of E 2^tx rows (bias_mode 0, 1), grid.y: chunks of columns; the
// 256 threads lie 2^tx along the rows and 256 / 2^tx along the columns, so that
// short columns keep every lane busy (16 x 393 bf16, gelu: 17 us with the lanes
// of a wave along the rows alone).
template <typename T, bool GATED>
__global__ void __launch_bounds__(256) act_grad_rows_kernel(ActGradArgs a, i64 cols, int tx) {
    using R = typename ga_traits<T>::acc;
    constexpr int E = 16 / sizeof(T);
    constexpr bool FAST = sizeof(T) == 2;
    using vE = ga_vec<T, E>;
    const int lane = threadIdx.x & ((1 << tx) - 1), w = threadIdx.x >> tx, ny = 256 >> tx;
    const i64 m = (((i64)blockIdx.x << tx) + lane) * E;
    const int left = (int)max((i64)0, min((i64)E, a.m - m));
    const i64 n0 = (i64)blockIdx.y * cols, n1 = min(a.n, n0 + cols);
    const bool wide = left == E;
    R sum[E];
    #pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = R(0);
    auto get = [&](const void* p, i64 ld, i64 n, T* v) {
        const T* x = static_cast<const T*>(p) + m + n * ld;
        if (a.m >= E) {          // a column's end: its last 16 bytes, shifted down
            typedef unsigned __int128 u128;
            const u128 w = __builtin_bit_cast(u128, *reinterpret_cast<const vE*>(x - (E - left)));
            const vE y = __builtin_bit_cast(vE, w >> ((E - left) * (int)sizeof(T) * 8));
            #pragma unroll
            for (int e = 0; e < E; ++e) v[e] = y[e];
        } else {
            #pragma unroll
            for (int e = 0; e < E; ++e) v[e] = e < left ? x[e] : (T)0;
        }
    };
    auto put = [&](void* p, i64 n, const R* v) {
        T* x = static_cast<T*>(p) + m + n * a.lddz;
        if (wide) {
            vE y;
            #pragma unroll
            for (int e = 0; e < E; ++e) y[e] = (T)v[e];
            *reinterpret_cast<vE*>(x) = y;
        } else {
            #pragma unroll
            for (int e = 0; e < E; ++e) if (e < left) x[e] = (T)v[e];
        }
    };
    // what their rounding leaves over
    auto rest = [&](void* p, i64 n, const R* v) {
        R y[E];
        #pragma unroll
        for (int e = 0; e < E; ++e) y[e] = ag_rest<T>(v[e]);
        put(p, n, y);
    };
    // UN columns' loads are in flight per thread: 4096 x 8192 bf16 48 us with one
    // (two: 51, four: 54), gated 64 us with two (one: 71)
    constexpr int UN = GATED ? 2 : 1;
    auto column = [&](i64 n, const T* c, const T* z1, const T* z2) {
        R d1[E], d2[E], z[E], v[E], d[E];
        #pragma unroll
        for (int e = 0; e < E; ++e) { z[e] = (R)z1[e]; v[e] = R(0); d[e] = R(1); }
        if (a.Z1) ga_act_grad<FAST, E>(a.act, z, v, d);
        #pragma unroll
        for (int e = 0; e < E; ++e) {
            const R g = (R)c[e];
            if constexpr (GATED) { d1[e] = g * (R)z2[e] * d[e]; d2[e] = g * v[e]; }
            else { d1[e] = g * d[e]; d2[e] = R(0); }
            sum[e] += d1[e];
        }
        if (a.dZ1) put(a.dZ1, n, d1);
        if constexpr (GATED) put(a.dZ2, n, d2);
        if constexpr (sizeof(T) == 2) {
            if (a.dL1) rest(a.dL1, n, d1);
            if (GATED && a.dL2) rest(a.dL2, n, d2);
        }
    };
    if (left > 0)
        for (i64 n = n0 + w; n < n1; n += ny * UN) {
            T c[UN][E], z1[UN][E], z2[UN][E];
            #pragma unroll
            for (int u = 0; u < UN; ++u) {
                const i64 nu = min(n + u * ny, n1 - 1);
                get(a.dC, a.lddc, nu, c[u]);
                if (a.Z1) get(a.Z1, a.ldz1, nu, z1[u]);
                if constexpr (GATED) get(a.Z2, a.ldz2, nu, z2[u]);
            }
            #pragma unroll 1
            for (int u = 0; u < UN; ++u) {
                // (one copy of the activations in the code: the vectors are picked by u)
                T cu[E], zu[E], wu[E];
                #pragma unroll
                for (int q = 0; q < UN; ++q)
                    if (q == u)
                        #pragma unroll
                        for (int e = 0; e < E; ++e) { cu[e] = c[q][e]; zu[e] = z1[q][e]; wu[e] = z2[q][e]; }
                if (n + u * ny < n1) column(n + u * ny, cu, zu, wu);
            }
        }
    if (a.bias_mode == 1) {
        __shared__ R red[256 * E];
        #pragma unroll
        for (int e = 0; e < E; ++e) red[threadIdx.x * E + e] = sum[e];
        __syncthreads();
        for (int i = threadIdx.x; i < E << tx; i += 256) {
            R s = red[i];
            for (int q = 1; q < ny; ++q) s += red[(q * E << tx) + i];
            const i64 mm = ((i64)blockIdx.x * E << tx) + i;
            if (mm < a.m) static_cast<R*>(a.part)[blockIdx.y * a.m + mm] = s;
        }
    }
}

// column sums: a wave takes one column's rows [chunk]; grid.x: columns / 4
template <typename T>
__global__ void __launch_bounds__(256) act_grad_cols_kernel(ActGradArgs a, i64 rows) {
    using R = typename ga_traits<T>::acc;
    constexpr bool FAST = sizeof(T) == 2;
    const int lane = threadIdx.x & 63;
    const i64 n = (i64)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (n >= a.n) return;
    const i64 m0 = (i64)blockIdx.y * rows, m1 = min(a.m, m0 + rows);
    R s = R(0);
    for (i64 m = m0 + lane; m < m1; m += 64) {
        R v, d = R(1);
        if (a.Z1) {
            const R z = (R) static_cast<const T*>(a.Z1)[m + n * a.ldz1];
            ga_act_grad<FAST, 1>(a.act, &z, &v, &d);
        }
        const R g = (R) static_cast<const T*>(a.dC)[m + n * a.lddc] * d;
        if (a.dZ1) static_cast<T*>(a.dZ1)[m + n * a.lddz] = (T)g;
        if constexpr (sizeof(T) == 2)
            if (a.dL1) static_cast<T*>(a.dL1)[m + n * a.lddz] = (T)ag_rest<T>(g);
        s += g;
    }
    s = wave_sum(s);
    if (lane == 0) static_cast<R*>(a.part)[blockIdx.y * a.n + n] = s;
}

// 32 sums per workgroup, 8 threads along the chunks of each
template <typename T>
__global__ void __launch_bounds__(256) act_grad_join_kernel(const typename ga_traits<T>::acc* part, i64 len, int chunks,
                                                            void* db, i64 incb, bool wide) {
    using R = typename ga_traits<T>::acc;
    __shared__ R red[8][32];
    const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
    const i64 i = (i64)blockIdx.x * 32 + x;
    R s = R(0);
    if (i < len) {
        #pragma unroll 8
        for (int c = y; c < chunks; c += 8) s += part[c * len + i];
    }
    red[y][x] = s;
    __syncthreads();
    if (y || i >= len) return;
    #pragma unroll
    for (int q = 1; q < 8; ++q) s += red[q][x];
    if (wide) static_cast<R*>(db)[i * incb] = s;
    else static_cast<T*>(db)[i * incb] = (T)s;
}

}  // namespace

// log2 of the threads along the rows
int act_grad_tx(int es, i64 m) {
    int tx = 0;
    while (tx < 6 && (16 / es << tx) < m) ++tx;
    return tx;
}

// Enough blocks for the 256 CUs several times over; none with less than a column
// for each of its threads, or 512 rows of its own.
int act_grad_chunks(int bias_mode, int es, i64 m, i64 n) {
    const int tx = act_grad_tx(es, m);
    const i64 rb = 16 / es << tx, cb = 256 >> tx;
    const i64 other = bias_mode == 2 ? (n + 3) / 4 : (m + rb - 1) / rb;
    const i64 most = bias_mode == 2 ? (m + 511) / 512 : (n + cb - 1) / cb;
    return (int)std::max<i64>(1, std::min<i64>(most, (1024 + other - 1) / std::max<i64>(1, other)));
}

template <typename T> void act_grad(ActGradArgs a, hipStream_t s) {
    if (a.m <= 0 || a.n <= 0) return;
    const int ES = sizeof(T), chunks = act_grad_chunks(a.bias_mode, ES, a.m, a.n);
    if (a.bias_mode == 2) {
        const i64 rows = (a.m + chunks - 1) / chunks;
        hipLaunchKernelGGL((act_grad_cols_kernel<T>), dim3((unsigned)((a.n + 3) / 4), chunks), dim3(256), 0, s, a, rows);
    } else {
        const int tx = act_grad_tx(ES, a.m);
        const i64 cols = (a.n + chunks - 1) / chunks, rb = 16 / ES << tx;
        const dim3 grid((unsigned)((a.m + rb - 1) / rb), chunks);
        if (a.Z2) hipLaunchKernelGGL((act_grad_rows_kernel<T, true>), grid, dim3(256), 0, s, a, cols, tx);
        else hipLaunchKernelGGL((act_grad_rows_kernel<T, false>), grid, dim3(256), 0, s, a, cols, tx);
    }
    HIP_LAUNCH_CHECK();
    if (a.bias_mode) {
        const i64 len = a.bias_mode == 1 ? a.m : a.n;
        hipLaunchKernelGGL((act_grad_join_kernel<T>), dim3((unsigned)((len + 31) / 32)), dim3(256), 0, s,
                           static_cast<const typename ga_traits<T>::acc*>(a.part), len, chunks, a.db, a.incb, a.wide);
        HIP_LAUNCH_CHECK();
    }
}

template void act_grad<__bf16>(ActGradArgs, hipStream_t);
template void act_grad<_Float16>(ActGradArgs, hipStream_t);
template void act_grad<float>(ActGradArgs, hipStream_t);
template void act_grad<double>(ActGradArgs, hipStream_t);

}  // namespace slate_hip
