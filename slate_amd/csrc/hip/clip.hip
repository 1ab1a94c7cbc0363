// The common norm of many matrices, and their scaling to at most a given one:
//   s = sqrt(sum_i |A_i|^2),  B_i = min(1, limit / s) A_i   (B_i = A_i where s
// is not finite).
// Memory bound, and launch bound for many small matrices: one launch takes up
// to CLIP_MATS of them, described in its arguments (no table to copy, so a
// captured call replays by itself).  Squares are summed in 64 bits, which
// neither overflow nor underflow for 16- and 32-bit elements; 64-bit elements
// go to one of three sums by size, the outer two scaled.  The first pass writes
// one partial sum per block; every block of the second adds them all in the
// same order, so that there is no third launch and no atomic, and the result
// is the same on every run.  0.8 G bf16 elements into f32: 299 us for the sums
// (5.4 TB/s), 965 us to scale (5.0 TB/s); 60 matrices of 4.7 M f32: 7 and 10 us.
// In place 0.5 G bf16 take 595 us, 0.13 G f32 287 us, f64 591 us (5.4 to 5.6 TB/s).
#include "ffn.hpp"

namespace slate_hip {

namespace {

constexpr int CLIP_MATS = 72, CLIP_BLOCKS = 1024;
// a unit of work: 32 KiB of a matrix
template <typename T> constexpr int clip_unit() { return 32768 / (int)sizeof(T); }

struct ClipArgs {
    ClipMat v[CLIP_MATS];
    int first[CLIP_MATS + 1];      // units before matrix i
    int count;
    double* part;                  // this launch's first partial
    const double* all;             // every partial (second pass)
    int parts;
    double limit;
    double* norm;
};

template <typename T> __device__ inline void clip_add(double (&s)[3], T x) {
    const double d = (double)x;
    if constexpr (sizeof(T) == 8) {
        const double a = fabs(d);
        // borders: squares of the middle range stay inside the type
        if (a > 1e145) { const double q = d * 0x1p-600; s[2] += q * q; }
        else if (a < 1e-145) { const double q = d * 0x1p600; s[0] += q * q; }
        else s[1] += d * d;                                                 // a NaN lands here
    } else {
        s[1] += d * d;
    }
}

// a block's sum of each entry, in all threads
__device__ inline double clip_block_sum(double x, double* lds) {
    x = wave_sum(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// This thread's share of unit u of an m x n matrix: whole(i, j) for E rows at
// (i, j), one(i, j) for one.  Vectors need no alignment, but cross no column's
// end: the columns are one (flat), or their length is a multiple of E.
template <int E, int UNIT, typename F, typename G>
__device__ inline void clip_walk(i64 m, i64 n, i64 u, bool flat, F&& whole, G&& one) {
    const i64 total = m * n, lo = u * UNIT, hi = min(total, lo + UNIT);
    if (flat) {
        constexpr int N = UNIT / (256 * E), B = N < 4 ? N : 4;
        if (hi - lo == UNIT) {
            #pragma unroll 1
            for (int b = 0; b < N; b += B) whole(lo + (b * 256 + (i64)threadIdx.x) * E, (i64)0, std::integral_constant<int, B>());
            return;
        }
        i64 q = lo + threadIdx.x * E;
        for (; q + E <= hi; q += 256 * E) whole(q, (i64)0, std::integral_constant<int, 1>());
        for (; q < hi; ++q) one(q, (i64)0);
        return;
    }
    const bool vec = m % E == 0;
    const int w = vec ? E : 1;
    i64 q = lo + threadIdx.x * w;
    if (q >= hi) return;
    i64 j = q / m, i = q - j * m;
    const i64 dj = 256 * w / m, di = 256 * w - dj * m;
    for (; q < hi; q += 256 * w) {
        if (vec) whole(i, j, std::integral_constant<int, 1>());
        else one(i, j);
        i += di;
        j += dj;
        if (i >= m) { i -= m; ++j; }
    }
}

__device__ inline int clip_find(const ClipArgs& a, int u) {
    int lo = 0, hi = a.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.first[mid] <= u) lo = mid; else hi = mid;
    }
    return lo;
}

template <typename T>
__global__ void __launch_bounds__(256) clip_sum_kernel(ClipArgs a) {
    constexpr int E = 16 / sizeof(T);
    typedef T vE __attribute__((ext_vector_type(E), aligned(sizeof(T))));
    __shared__ double lds[4];
    double s[3] = {0, 0, 0};
    for (int u = blockIdx.x; u < a.first[a.count]; u += gridDim.x) {
        const int c = clip_find(a, u);
        const ClipMat v = a.v[c];
        const T* A = static_cast<const T*>(v.A);
        const bool flat = v.lda == v.m || v.n == 1;
        const i64 uu = u - a.first[c];
        clip_walk<E, clip_unit<T>()>(v.m, v.n, uu, flat, [&](i64 i, i64 j, auto count) {
            constexpr int B = decltype(count)::value;
            vE x[B];
            #pragma unroll
            for (int b = 0; b < B; ++b) x[b] = *reinterpret_cast<const vE*>(A + i + b * (256 * E) + j * v.lda);
            #pragma unroll
            for (int b = 0; b < B; ++b)
                #pragma unroll
                for (int e = 0; e < E; ++e) clip_add(s, (T)x[b][e]);
        }, [&](i64 i, i64 j) { clip_add(s, A[i + j * v.lda]); });
    }
    #pragma unroll
    for (int h = 0; h < 3; ++h) {
        const double x = clip_block_sum(s[h], lds);
        if (threadIdx.x == 0) a.part[3 * (i64)blockIdx.x + h] = x;
    }
}

// the norm and the factor from all partial sums, in every thread
__device__ inline double clip_norm_of(const ClipArgs& a, double* lds) {
    double s[3] = {0, 0, 0};
    for (int i = threadIdx.x; i < a.parts; i += 256)
        #pragma unroll
        for (int h = 0; h < 3; ++h) s[h] += a.all[3 * (i64)i + h];
    #pragma unroll
    for (int h = 0; h < 3; ++h) s[h] = clip_block_sum(s[h], lds);
    if (s[1] != s[1]) return s[1];
    // the middle sum counts beside the large one only while it is not lost in it
    if (s[2] > 0) return sqrt(s[2] + (s[1] * 0x1p-600) * 0x1p-600) * 0x1p600;
    if (s[1] > 0) return sqrt(s[1] + (s[0] * 0x1p-600) * 0x1p-600);
    return sqrt(s[0]) * 0x1p-600;
}

template <typename TA, typename TB>
__global__ void __launch_bounds__(256) clip_scale_kernel(ClipArgs a) {
    using R = std::conditional_t<sizeof(TA) == 8, double, float>;
    constexpr int E = 16 / sizeof(TA);
    typedef TA vA __attribute__((ext_vector_type(E), aligned(sizeof(TA))));
    typedef TB vB __attribute__((ext_vector_type(E), aligned(sizeof(TB))));
    __shared__ double lds[4];
    const double norm = clip_norm_of(a, lds);
    if (a.norm && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = norm;
    const bool cut = norm > a.limit && norm < __builtin_huge_val();
    // The factor as f 2^e: e is 0 where limit / norm is a normal number of the
    // sums' type; below it would lose bits, or all of them, and ordinary products
    // with it (elements of 2e38, limit 1e-6).  Scaling by 2^e is exact.
    const double q = a.limit / norm;
    R f = (R)q;
    int e = 0, en;
    if (cut && q < (sizeof(R) == 4 ? 0x1p-126 : 0x1p-1022)) {
        const double part = 0.5 * frexp(a.limit, &e);
        f = (R)(part / frexp(norm, &en));          // in [1/4, 1]
        e += 1 - en;
    }
    auto scaled = [&](R x) {
        if constexpr (sizeof(R) == 4) return cut ? __builtin_amdgcn_ldexpf(x * f, e) : x;
        else return cut ? __builtin_amdgcn_ldexp(x * f, e) : x;
    };
    // backwards: what the first pass read last is still in the cache
    for (int u = a.first[a.count] - 1 - (int)blockIdx.x; u >= 0; u -= gridDim.x) {
        const int c = clip_find(a, u);
        const ClipMat v = a.v[c];
        const TA* A = static_cast<const TA*>(v.A);
        TB* B = static_cast<TB*>(v.B);
        if (!cut && v.A == v.B) continue;
        const bool flat = (v.lda == v.m && v.ldb == v.m) || v.n == 1;
        const i64 uu = u - a.first[c];
        clip_walk<E, clip_unit<TA>()>(v.m, v.n, uu, flat, [&](i64 i, i64 j, auto count) {
            constexpr int N = decltype(count)::value;
            vA x[N];
            #pragma unroll
            for (int b = 0; b < N; ++b) x[b] = *reinterpret_cast<const vA*>(A + i + b * (256 * E) + j * v.lda);
            #pragma unroll
            for (int b = 0; b < N; ++b) {
                vB y;
                #pragma unroll
                for (int k = 0; k < E; ++k) y[k] = (TB)scaled((R)x[b][k]);
                *reinterpret_cast<vB*>(B + i + b * (256 * E) + j * v.ldb) = y;
            }
        }, [&](i64 i, i64 j) {
            B[i + j * v.ldb] = (TB)scaled((R)A[i + j * v.lda]);
        });
    }
}

__global__ void __launch_bounds__(256) clip_join_kernel(const double* part, int parts, double* out) {
    __shared__ double lds[4];
    #pragma unroll
    for (int h = 0; h < 3; ++h) {
        double s = 0;
        for (int i = threadIdx.x; i < parts; i += 256) s += part[3 * (i64)i + h];
        s = clip_block_sum(s, lds);
        if (threadIdx.x == 0) out[h] = s;
    }
}

// the matrices [at, at + CLIP_MATS) as one launch's arguments; -> its units
int clip_fill(ClipArgs& a, const ClipMat* v, int count, int at, int unit) {
    a.count = std::max(0, std::min(CLIP_MATS, count - at));
    a.first[0] = 0;
    i64 units = 0;
    for (int i = 0; i < a.count; ++i) {
        a.v[i] = v[at + i];
        units += (a.v[i].m * a.v[i].n + unit - 1) / unit;
        if (units > 0x7fffffff) throw std::invalid_argument("clip_norm: matrices too large for one call");
        a.first[i + 1] = (int)units;
    }
    return a.first[a.count];
}

template <typename TA, typename TB>
void clip_scale_run(const ClipMat* v, int count, double limit, const double* part, int parts, double* norm, hipStream_t s) {
    for (int at = count ? (count - 1) / CLIP_MATS * CLIP_MATS : 0; at >= 0; at -= CLIP_MATS) {
        ClipArgs a;
        const int blocks = std::min(CLIP_BLOCKS, clip_fill(a, v, count, at, clip_unit<TA>()));
        a.limit = limit;
        a.all = part;
        a.parts = parts;
        a.norm = at == 0 ? norm : nullptr;
        hipLaunchKernelGGL((clip_scale_kernel<TA, TB>), dim3(std::max(1, blocks)), dim3(256), 0, s, a);
        HIP_LAUNCH_CHECK();
    }
}

}  // namespace

static int clip_unit_of(char t) { return t == 'd' ? clip_unit<double>() : t == 's' ? clip_unit<float>() : clip_unit<__bf16>(); }

i64 clip_parts(i64 count) { return 3 * CLIP_BLOCKS * ((count + CLIP_MATS - 1) / CLIP_MATS); }

int clip_sum(char ta, const ClipMat* v, int count, double* part, hipStream_t s) {
    int done = 0;
    for (int at = 0; at < count; at += CLIP_MATS) {
        ClipArgs a;
        const int blocks = std::min(CLIP_BLOCKS, clip_fill(a, v, count, at, clip_unit_of(ta)));
        a.part = part + 3 * (i64)done;
        done += blocks;
        if (ta == 'b') hipLaunchKernelGGL((clip_sum_kernel<__bf16>), dim3(blocks), dim3(256), 0, s, a);
        else if (ta == 'h') hipLaunchKernelGGL((clip_sum_kernel<_Float16>), dim3(blocks), dim3(256), 0, s, a);
        else if (ta == 's') hipLaunchKernelGGL((clip_sum_kernel<float>), dim3(blocks), dim3(256), 0, s, a);
        else if (ta == 'd') hipLaunchKernelGGL((clip_sum_kernel<double>), dim3(blocks), dim3(256), 0, s, a);
        else throw std::invalid_argument("clip_norm: bad element type");
        HIP_LAUNCH_CHECK();
    }
    return done;
}

void clip_join(const double* part, int parts, double* out, hipStream_t s) {
    hipLaunchKernelGGL(clip_join_kernel, dim3(1), dim3(256), 0, s, part, parts, out);
    HIP_LAUNCH_CHECK();
}

void clip_scale(char ta, char tb, const ClipMat* v, int count, double limit, const double* part, int parts,
                double* norm, bool scale, hipStream_t s) {
    if (!scale) count = 0;
    if (ta == 'b' && tb == 'b') clip_scale_run<__bf16, __bf16>(v, count, limit, part, parts, norm, s);
    else if (ta == 'b' && tb == 's') clip_scale_run<__bf16, float>(v, count, limit, part, parts, norm, s);
    else if (ta == 'h' && tb == 'h') clip_scale_run<_Float16, _Float16>(v, count, limit, part, parts, norm, s);
    else if (ta == 'h' && tb == 's') clip_scale_run<_Float16, float>(v, count, limit, part, parts, norm, s);
    else if (ta == 's' && tb == 's') clip_scale_run<float, float>(v, count, limit, part, parts, norm, s);
    else if (ta == 'd' && tb == 'd') clip_scale_run<double, double>(v, count, limit, part, parts, norm, s);
    else throw std::invalid_argument("clip_norm: bad element types");
}

}  // namespace slate_hip
