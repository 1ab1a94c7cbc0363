// Matrix products with a fused epilogue for gfx950 (bf16, f16, f32, f64):
//
//   plain   Z = alpha op(A) op(B) + bias,            C = act(Z) + beta R
//   sum     C = alpha sum_p op(A_p) op(B_p)          (two to four products)
//   gated   Z_i = op(A_i) op(B),                     C = act(Z_1) o Z_2
//   pair    C_i = alpha op(A_i) op(B_i)              (two products, one launch)
//
// Sums are kept in 32 bits (64 for f64) in the MFMA accumulators and rounded
// once, when C (and Z) are stored.
//
// Every operand is staged into LDS as slabs of 128 bytes of K per row
// (KB = 64 / 32 / 16 elements) by global_load_lds_dwordx4, 1 KiB per wave and
// instruction, written lane-linear.  The bank swizzle therefore sits on the
// source address and on the read:
//  * KC, source contiguous along k (element (r, k) at X[k + r ld]):
//    image [r][8 chunks of 16 bytes], chunk c of row r at c ^ ((r >> 1) & 7):
//    the 16 rows of a fragment read one chunk column from 16 distinct
//    16-byte slots of the 256-byte bank row.  One ds_read_b128 per fragment.
//  * MN, source contiguous along the tile's rows (X[r + k ld]): image
//    [k][R], the 16-row segment s of row k at s ^ swz(k).  16-bit types read
//    it with ds_read_b64_tr_b16 (a 4 x 16 block arrives transposed: each lane
//    gets four k of its row), 32- and 64-bit types with one read per element.
// A fragment is 16 bytes per lane in either case: lane l holds row l & 15 and
// the E = 8 / 4 / 2 consecutive k of chunk (l >> 4); A and B use the same
// k order, so one, four or two MFMAs multiply it.
//
// Large products are bound by the MFMAs: bf16 8192 columns, 4096 -> 16384,
// gelu_tanh with Z stored 920 us (1195 TFLOP/s), gated 4096 -> 8192 877 us (1254),
// f32 4096^3 990 us (139), f64 2010 us (68).  Few columns are bound by reading
// op(A): f16 33 columns, 8192 -> 2048 9.5 us and 3.5 us to join 16 pieces of K.
#pragma once
#include "ffn.hpp"

namespace slate_hip {

typedef int i4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef _Float16 hf8v __attribute__((ext_vector_type(8)));

// V elements as one access.  Rows need not lie on 16 bytes: the type claims the
// element's alignment only, and the hardware takes such addresses (a vector
// that straddles a cache line costs a second access, not V of them).
template <typename T, int V> struct ga_vec_of { typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T)))); };
template <typename T, int V> using ga_vec = typename ga_vec_of<T, V>::type;

// mma: the u-th of the N MFMAs that multiply two fragments
template <typename T> struct ga_traits;
template <> struct ga_traits<__bf16> {
    using acc = float; using acc4 = f4;
    static constexpr int N = 1;
    __device__ static inline acc4 mma(i4v a, i4v b, acc4 c, int) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, a), __builtin_bit_cast(bf8v, b), c,
                                                       0, 0, 0);
    }
};
template <> struct ga_traits<_Float16> {
    using acc = float; using acc4 = f4;
    static constexpr int N = 1;
    __device__ static inline acc4 mma(i4v a, i4v b, acc4 c, int) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(hf8v, a), __builtin_bit_cast(hf8v, b), c,
                                                      0, 0, 0);
    }
};
template <> struct ga_traits<float> {
    using acc = float; using acc4 = f4;
    static constexpr int N = 4;
    __device__ static inline acc4 mma(i4v a, i4v b, acc4 c, int u) {
        return __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f4, a)[u], __builtin_bit_cast(f4, b)[u], c, 0, 0, 0);
    }
};
template <> struct ga_traits<double> {
    using acc = double; using acc4 = d4;
    static constexpr int N = 2;
    __device__ static inline acc4 mma(i4v a, i4v b, acc4 c, int u) {
        return __builtin_amdgcn_mfma_f64_16x16x4f64(__builtin_bit_cast(d2, a)[u], __builtin_bit_cast(d2, b)[u], c, 0, 0, 0);
    }
};

// ------------------------------------------------------------- activations
// On V values at once, the choice of the function outside: V independent chains
// hide each other's latency.  Results of 16 bits round to 2^-11 at best: their
// exponential and reciprocal are the hardware's (a few 2^-24 of the argument),
// 32- and 64-bit results call exp and divide.
template <bool FAST> __device__ inline float ga_exp(float x) { return FAST ? __expf(x) : expf(x); }
template <bool FAST> __device__ inline double ga_exp(double x) { return exp(x); }
template <bool FAST> __device__ inline float ga_inv(float b) { return FAST ? __builtin_amdgcn_rcpf(b) : 1.f / b; }
template <bool FAST> __device__ inline double ga_inv(double b) { return 1.0 / b; }

// The normal distribution's function P(z) and e = exp(-z^2 / 2).  For 16-bit
// results P(-x sqrt 2) = exp(-x^2) f(1 / (1 + 0.43 x)) / 2 with a polynomial f
// of degree 8 fitted to exp(x^2) erfc(x) on [0, 12] in the relative sense
// (4.4e-7 in 32-bit arithmetic); P(z) = 1 - P(-z).
template <bool FAST, typename R> __device__ inline R ga_phi(R z, R& e) {
    e = ga_exp<FAST>(R(-0.5) * z * z);
    if constexpr (FAST) {
        const R t = ga_inv<FAST>(R(1) + R(0.43 * 0.70710678118654752440) * fabsf(z));
        R f = R(0.0709153654);
        f = f * t - R(0.299052681);
        f = f * t + R(0.364768859);
        f = f * t - R(0.0688474548);
        f = f * t + R(0.238222132);
        f = f * t + R(0.207465912);
        f = f * t + R(0.243989002);
        f = f * t + R(0.242538687);
        f = f * t * e * R(0.5);
        return z < R(0) ? f : R(1) - f;
    } else if constexpr (sizeof(R) == 4) {
        return R(0.5) * erfcf(z * R(-0.70710678118654752440));
    } else {
        return R(0.5) * erfc(z * R(-0.70710678118654752440));
    }
}

// Beyond ga_flat the smooth activations are 0 (left) or z itself (right) in
// their type: arguments are held inside it, which keeps 0 * inf out.
template <typename R> __device__ constexpr R ga_flat() { return sizeof(R) == 4 ? R(120) : R(800); }

template <bool FAST, int V, typename R> __device__ inline void ga_act(int act, const R* z, R* y) {
    constexpr R L = ga_flat<R>();
    if (act == ACT_IDENTITY) {
        #pragma unroll
        for (int r = 0; r < V; ++r) y[r] = z[r];
    } else if (act == ACT_RELU) {
        #pragma unroll
        for (int r = 0; r < V; ++r) y[r] = z[r] < R(0) ? R(0) : z[r];                   // a NaN stays one
    } else if (act == ACT_GELU) {
        #pragma unroll
        for (int r = 0; r < V; ++r) {
            const R x = z[r] < -L ? -L : z[r];
            R e;
            y[r] = x * ga_phi<FAST>(x, e);
        }
    } else if (act == ACT_GELU_TANH) {                                                  // (1 + tanh u) / 2 = 1 / (1 + e^-2u)
        #pragma unroll
        for (int r = 0; r < V; ++r) {
            const R x = z[r] < -L ? -L : z[r], u2 = x * (R(1.59576912160573071176) + R(0.07135481627260024519) * x * x);
            y[r] = x * ga_inv<FAST>(R(1) + ga_exp<FAST>(-u2));
        }
    } else {
        #pragma unroll
        for (int r = 0; r < V; ++r) {
            const R x = z[r] < -L ? -L : z[r];
            y[r] = x * ga_inv<FAST>(R(1) + ga_exp<FAST>(-x));
        }
    }
}
// values and slopes (the backward pass of a gated product needs both)
template <bool FAST, int V, typename R> __device__ inline void ga_act_grad(int act, const R* z, R* v, R* d) {
    constexpr R L = ga_flat<R>();
    // v = x p, d = p + x e
    auto put = [&](int r, R x, R p, R e) {
        v[r] = z[r] > L ? z[r] : x * p;
        d[r] = p + x * e;
    };
    auto in = [&](R x) { return x < -L ? -L : (x > L ? L : x); };
    if (act == ACT_IDENTITY) {
        #pragma unroll
        for (int r = 0; r < V; ++r) { v[r] = z[r]; d[r] = R(1); }
    } else if (act == ACT_RELU) {
        #pragma unroll
        for (int r = 0; r < V; ++r) {
            v[r] = z[r] < R(0) ? R(0) : z[r];
            d[r] = z[r] > R(0) ? R(1) : (z[r] <= R(0) ? R(0) : z[r]);
        }
    } else if (act == ACT_GELU) {
        #pragma unroll
        for (int r = 0; r < V; ++r) {
            const R x = in(z[r]);
            R e;
            const R p = ga_phi<FAST>(x, e);
            put(r, x, p, e * R(0.39894228040143267794));
        }
    } else if (act == ACT_GELU_TANH) {
        #pragma unroll
        for (int r = 0; r < V; ++r) {
            const R x = in(z[r]), u2 = x * (R(1.59576912160573071176) + R(0.07135481627260024519) * x * x);
            const R p = ga_inv<FAST>(R(1) + ga_exp<FAST>(-u2));
            put(r, x, p, p * (R(1) - p) * (R(1.59576912160573071176) + R(0.21406444881780073557) * x * x));
        }
    } else {
        #pragma unroll
        for (int r = 0; r < V; ++r) {
            const R x = in(z[r]), p = ga_inv<FAST>(R(1) + ga_exp<FAST>(-x));
            put(r, x, p, p * (R(1) - p));
        }
    }
}

// V rows of column n: the epilogue on finished sums.  PAST: outputs past the
// caches, which keep the operands instead (256 x 256 tiles: 916 us against 938 for
// 8192 columns, 4096 -> 16384 with Z; smaller outputs are often read next).
template <typename T, int V, bool GATED, bool PAST = false>
__device__ inline void ga_finish(const GemmActArgs& a, int pair, i64 m, i64 n, const typename ga_traits<T>::acc* s1,
                                 const typename ga_traits<T>::acc* s2) {
    using R = typename ga_traits<T>::acc;
    constexpr bool FAST = sizeof(T) == 2;
    using vT = ga_vec<T, V>;
    if (n >= a.n || m >= a.m) return;
    const bool whole = V == 1 || m + V <= a.m;
    const int left = (int)min((i64)V, a.m - m);
    T* C = static_cast<T*>(a.C[pair]) + m + n * a.ldc[pair];
    R z[V], y[V];
    if constexpr (GATED) {
        #pragma unroll
        for (int r = 0; r < V; ++r) z[r] = s1[r];
        ga_act<FAST, V>(a.act, z, y);
        #pragma unroll
        for (int r = 0; r < V; ++r) y[r] *= s2[r];
    } else {
        const R alpha = (R)a.alpha;
        #pragma unroll
        for (int r = 0; r < V; ++r) z[r] = alpha * s1[r];
        if (a.bias_mode == 1) {
            const T* b = static_cast<const T*>(a.bias);
            if (whole && a.incb == 1) {
                const vT x = *reinterpret_cast<const vT*>(b + m);
                #pragma unroll
                for (int r = 0; r < V; ++r) z[r] += (R)x[r];
            } else {
                #pragma unroll
                for (int r = 0; r < V; ++r) if (r < left) z[r] += (R)b[(m + r) * a.incb];
            }
        } else if (a.bias_mode == 2) {
            const R x = (R) static_cast<const T*>(a.bias)[n * a.incb];
            #pragma unroll
            for (int r = 0; r < V; ++r) z[r] += x;
        }
        ga_act<FAST, V>(a.act, z, y);
        if (a.R) {
            const T* X = static_cast<const T*>(a.R) + m + n * a.ldr;
            const R beta = (R)a.beta;
            if (whole) {
                const vT x = *reinterpret_cast<const vT*>(X);
                #pragma unroll
                for (int r = 0; r < V; ++r) y[r] += beta * (R)x[r];
            } else {
                #pragma unroll
                for (int r = 0; r < V; ++r) if (r < left) y[r] += beta * (R)X[r];
            }
        }
    }
    auto put = [&](T* p, const R* v, bool wide) {
        if (wide) {
            vT x;
            #pragma unroll
            for (int r = 0; r < V; ++r) x[r] = (T)v[r];
            if constexpr (PAST) __builtin_nontemporal_store(x, reinterpret_cast<vT*>(p));
            else *reinterpret_cast<vT*>(p) = x;
        } else {
            #pragma unroll
            for (int r = 0; r < V; ++r) if (r < left) p[r] = (T)v[r];
        }
    };
    put(C, y, whole);
    if (a.Z[0]) put(static_cast<T*>(a.Z[0]) + m + n * a.ldz[0], z, whole);
    if constexpr (GATED)
        if (a.Z[1]) put(static_cast<T*>(a.Z[1]) + m + n * a.ldz[1], s2, whole);
}

// W bytes per lane from p to q + W lane (q: of the wave), asynchronously
template <int W> __device__ inline void ga_to_lds(const void* p, void* q) {
    using gptr = const __attribute__((address_space(1))) void*;
    using lptr = __attribute__((address_space(3))) void*;
    if constexpr (W == 4) __builtin_amdgcn_global_load_lds((gptr)p, (lptr)q, 4, 0, 0);
    else __builtin_amdgcn_global_load_lds((gptr)p, (lptr)q, 16, 0, 0);
}

// ------------------------------------------------------------- LDS images
// 16 bytes moved down by `down` bits, zeros behind them
__device__ inline i4v ga_shift(i4v w, int down) {
    typedef unsigned __int128 u128;
    const u128 x = __builtin_bit_cast(u128, w) >> (down & 127);
    return __builtin_bit_cast(i4v, down < 128 ? x : (u128)0);
}

template <typename T, int R, bool KC> struct GaImg {
    static constexpr int ES = sizeof(T), E = 16 / ES, KB = 128 / ES;
    static constexpr int BYTES = R * 128;
    static constexpr int ROWB = R * ES;                       // MN: bytes per k
    static constexpr int SEGB = 16 * ES;                      // MN: bytes of a 16-row segment
    static constexpr int NSEG = R / 16;
    // MN: which segments the k rows that one read touches together go to.  A
    // transposed read of 16 bits takes 32 lanes at a time: 32 bytes of each of the
    // rows k .. k + 3 and k + 8 .. k + 11 (k a multiple of 8, + 4), in 8 slots of
    // the 256-byte bank row; what the row's own place tells apart the segment
    // need not.  (515 x 1024 x 2560 f16 gradients: 45 % of the LDS cycles were
    // conflicts with k & 3 for 64 rows.)
    __device__ static constexpr int swz(int k) {
        if constexpr (ES == 2) {
            if constexpr (NSEG >= 8) return (k & 3) | ((k >> 1) & 4);
            else if constexpr (NSEG == 4) return ((k >> 1) & 1) | ((k >> 2) & 2);
            else return (k >> 3) & (NSEG - 1);
        }
        else if constexpr (ES == 4) return (k >> 2) & 3 & (NSEG - 1);
        else return (k >> 1) & 1 & (NSEG - 1);
    }
    // KC: 16 rows of one chunk column lie in 16 distinct 16-byte slots
    __device__ static constexpr int turn(int r) { return (r >> 1) & 7; }
    // row and k of the first element of 16-byte slot q
    __device__ static inline void src_of(int q, int& r, int& k) {
        if constexpr (KC) {
            r = q / 8;
            k = ((q % 8) ^ turn(r)) * E;
        } else {
            const int p = q * 16;
            k = p / ROWB;
            r = ((p % ROWB) ^ (swz(k) * SEGB)) / ES;
        }
    }
    // this lane's fragment: rows r0..r0+15, chunk half kk
    __device__ static inline i4v frag(const char* img, int r0, int kk, int lane) {
        const int l = lane & 15, g = lane >> 4;
        if constexpr (KC) {
            const int r = r0 + l;
            return *reinterpret_cast<const i4v*>(img + r * 128 + (((kk * 4 + g) ^ turn(r)) << 4));
        } else if constexpr (ES == 2) {
            typedef short s4 __attribute__((ext_vector_type(4)));
            typedef int i2 __attribute__((ext_vector_type(2)));
            const int k = kk * 32 + g * 8 + (l >> 2);
            const char* p = img + k * ROWB + (((r0 >> 4) ^ swz(k)) * SEGB) + (l & 3) * 8;
            using lds_s4 = __attribute__((address_space(3))) s4;
            const i2 x = __builtin_bit_cast(i2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p));
            const i2 y = __builtin_bit_cast(i2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + 4 * ROWB)));
            return i4v{x[0], x[1], y[0], y[1]};
        } else {
            T v[E];
            #pragma unroll
            for (int j = 0; j < E; ++j) {
                const int k = (kk * 4 + g) * E + j;
                v[j] = *reinterpret_cast<const T*>(img + k * ROWB + (((r0 >> 4) ^ swz(k)) * SEGB) + l * ES);
            }
            if constexpr (ES == 4) return __builtin_bit_cast(i4v, f4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]});
            else return __builtin_bit_cast(i4v, d2{(double)v[0], (double)v[1]});
        }
    }
    // bytes from the slab's first element that lane `lane` of piece c (64 accesses
    // of W bytes) stages; rows past the matrix read one that exists and feed no
    // stored output
    template <int W> __device__ static inline uint32_t offset(int c, int lane, i64 ld, i64 rows) {
        const int at = (c * 64 + lane) * W, e = at % 16 / ES, half = W < ES ? at % ES : 0;
        int r, k;
        src_of(at / 16, r, k);
        if constexpr (KC) {
            const i64 rr = r < rows ? r : rows - 1;
            return (uint32_t)((rr * ld + k + e) * ES + half);
        } else {
            const i64 rr = W < 16 ? min((i64)(r + e), rows - 1) : r < rows ? r : 0;
            return (uint32_t)((k * ld + rr) * ES + half);
        }
    }
    // 16-byte slot q of the slab at X, off elements from X, at any alignment; zeros
    // past the matrix in k, anything in rows that do not exist.  A slot that
    // passes the end of its column (of len elements) reads the column's last 16
    // bytes and shifts them down.
    __device__ static inline i64 element(int q, i64 ld, i64 rows) {
        int r, k;
        src_of(q, r, k);
        if constexpr (KC) return (r < rows ? r : rows - 1) * ld + k;
        else return k * ld + r;
    }
    // (the shift, by `down` bits, is left to the caller: it waits for the load)
    __device__ static inline i4v fetch(const T* X, i64 off, int q, i64 ld, i64 len, i64 rows, i64 kleft, bool inside,
                                       int& down) {
        using vE = ga_vec<T, E>;
        down = 0;
        if (inside) return __builtin_bit_cast(i4v, *reinterpret_cast<const vE*>(X + off));
        int r, k;
        src_of(q, r, k);
        const i64 over = max((i64)0, KC ? k + E - kleft : r + E - rows), below = KC ? 0 : max((i64)0, k + 1 - kleft);
        const T* x = X + off - below * ld;
        if (len < E) {                                   // (the whole matrix has shorter columns)
            vE w;
            #pragma unroll
            for (int e = 0; e < E; ++e) w[e] = !below && e + over < E ? x[e] : (T)0;
            return __builtin_bit_cast(i4v, w);
        }
        down = over < E && !below ? (int)over * ES * 8 : 128;
        return __builtin_bit_cast(i4v, *reinterpret_cast<const vE*>(x - over));
    }
    // The same for slabs that all go through registers: what a slot's addresses
    // need, made once, and a load without a branch (the loads of two slabs are in
    // flight, and a load behind a branch would be waited for at once).  avail: the
    // columns' length (MN: from the tile's first row), 16 bytes or more.
    struct Slot { i64 el, el0; int k, cut; };
    __device__ static inline Slot slot(int q, i64 ld, i64 rows, i64 avail) {
        int r, k;
        src_of(q, r, k);
        if constexpr (KC) return {min((i64)r, rows - 1) * ld + k, 0, k, 0};
        else {
            const i64 over = max((i64)0, r + E - avail);
            return {k * ld + r - over, r - over, k, over < E ? (int)over * ES * 8 : 128};
        }
    }
    __device__ static inline i4v load(const T* X, const Slot& t, int kl, int& down) {
        using vE = ga_vec<T, E>;
        if constexpr (KC) {
            const int over = max(0, t.k + E - kl);
            down = over < E ? over * ES * 8 : 128;
            return __builtin_bit_cast(i4v, *reinterpret_cast<const vE*>(X + (t.el - over)));
        } else {
            down = t.k < kl ? t.cut : 128;
            return __builtin_bit_cast(i4v, *reinterpret_cast<const vE*>(X + (t.k < kl ? t.el : t.el0)));
        }
    }
    // A slab with an end of the matrix in it, wave wid of NW.  DMA of 16 bytes:
    // accesses that lie inside go to LDS directly, the others from registers.
    // DMA of 4: all from registers in 16-byte accesses (four times fewer; 452 x 17
    // x 7897 f32, two products: 21 us against 24).
    template <int W, int NW>
    __device__ static inline void stage(const T* X, i64 ld, i64 len, i64 rows, i64 kleft, char* img, int wid, int lane) {
        constexpr int N = BYTES / 1024;
        if constexpr (W == 16) {
            #pragma unroll 1
            for (int c = wid; c < N; c += NW) {
                const int q = c * 64 + lane;
                const i64 off = element(q, ld, rows);
                int r, k;
                src_of(q, r, k);
                if (KC ? k + E <= kleft : k < kleft && r + E <= rows) ga_to_lds<16>(X + off, img + c * 1024);
                else if (k < kleft && (KC || r < rows)) {
                    int down;
                    const i4v w = fetch(X, off, q, ld, len, rows, kleft, false, down);
                    *reinterpret_cast<i4v*>(img + q * 16) = ga_shift(w, down);
                } else *reinterpret_cast<i4v*>(img + q * 16) = i4v{0, 0, 0, 0};
            }
        } else {
            constexpr int C = (N + NW - 1) / NW;
            i4v w[C];
            int down[C];
            #pragma unroll
            for (int i = 0; i < C; ++i) {
                const int q = min(wid + i * NW, N - 1) * 64 + lane;
                w[i] = fetch(X, element(q, ld, rows), q, ld, len, rows, kleft, false, down[i]);
            }
            #pragma unroll
            for (int i = 0; i < C; ++i)
                *reinterpret_cast<i4v*>(img + (min(wid + i * NW, N - 1) * 64 + lane) * 16) = ga_shift(w[i], down[i]);
        }
    }
};

// The epilogue turns the accumulators through LDS, a wave's columns NJ
// fragments at a time, so that stores (and the loads of bias and residual) run
// along the rows in 16-byte accesses and the activation appears in the code
// once: unrolled over the 32 fragments of a wave it is 16 000 instructions.
template <typename T, int BM, int BN, int WVM, int WVN, int S> struct GaEpi {
    static constexpr int AS = sizeof(typename ga_traits<T>::acc), NW = WVM * WVN, NI = BN / WVN / 16;
    static constexpr int LDR = BM / WVM + 16 / AS;                    // rows of a column, and 16 bytes against conflicts
    static constexpr int RING = S * (BM + BN) * 128, MOST = RING > 131071 ? 163840 : (RING > 65535 ? 81920 : RING);
    static constexpr int bytes(int nj) { return NW * LDR * 16 * nj * AS; }
    static constexpr int pick() { int nj = NI; while (nj > 1 && bytes(nj) > MOST) nj /= 2; return nj; }
    static constexpr int NJ = pick();
    static constexpr int LDS = RING > bytes(NJ) ? RING : bytes(NJ);
    static_assert(LDS <= 163840, "tile does not fit the LDS");
};

// ------------------------------------------------------------------ kernel
// DMA: bytes of an LDS-DMA access (the ragged end of K goes through registers).
// 16 where the operands' rows lie on 16 bytes, 4 for 32- and 64-bit elements
// elsewhere: four times the instructions, still asynchronous (1503 x 777 x 1001
// f32: 38 us against 53 us through registers).  0: every slab goes through
// registers, two slabs ahead of its products.
// Two waves a SIMD at least (one workgroup of 512 threads a CU, two of 256): with
// one, the compiler keeps the sums in vector registers between steps and copies
// them to accumulation registers and back in each (f64 4096^3 2230 us against 2010).
template <typename T, bool AKC, bool BKC, int BM, int BN, int WVM, int WVN, int S, bool GATED, int DMA>
__global__ void __launch_bounds__(64 * WVM * WVN, 2) gemm_act_kernel(GemmActArgs a) {
    using TR = ga_traits<T>;
    using acc4 = typename TR::acc4;
    using R = typename TR::acc;
    constexpr int NW = WVM * WVN, NT = 64 * NW, NA = GATED ? 2 : 1, BMI = BM / NA;
    constexpr int WM = BM / WVM, WN = BN / WVN, MI = WM / 16, NI = WN / 16, KB = 128 / (int)sizeof(T);
    using IA = GaImg<T, BMI, AKC>;
    using IB = GaImg<T, BN, BKC>;
    constexpr int SLOT = (BM + BN) * 128;
    constexpr int W = DMA ? DMA : 16, PCA = IA::BYTES / (64 * W), PCB = IB::BYTES / (64 * W);    // pieces of a slab
    constexpr int PA = (PCA + NW - 1) / NW, PB = (PCB + NW - 1) / NW;
    static_assert(MI % NA == 0, "gated tiles pair their fragments");
    static_assert(S == 2 || DMA, "registers hold one slab");
    static_assert(W == 16 || W <= (int)sizeof(T), "an access lies in one element");
    constexpr int LOADS = NA * PA + PB;              // DMA instructions of a wave's slab
    extern __shared__ __align__(16) char smem[];

    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int gm = (int)((a.m + BMI - 1) / BMI), gn = (int)((a.n + BN - 1) / BN), nblk = gm * gn;
    // blocks b and b + 8 share an XCD: consecutive tiles of one group there
    const int lin = xcd_remap(blockIdx.x, nblk);
    const int G = a.group_m, grp = lin / (G * gn), first = grp * G, gsz = min(gm - first, G);
    const int inner = lin - grp * G * gn;
    const i64 m0 = (i64)(first + inner % gsz) * BMI, n0 = (i64)(inner / gsz) * BN;
    const int pair = a.mode == GA_PAIR ? blockIdx.z : 0;
    const int total = a.nsteps * a.terms;
    const int s0 = a.splits > 1 ? (int)blockIdx.y * a.per_split : 0;
    const int s1 = a.splits > 1 ? min(total, s0 + a.per_split) : total;

    const i64 rowsA = a.m - m0, rowsB = a.n - n0;
    const bool sum = a.terms > 1;
    auto slabA = [&](int q, i64 k0) { return static_cast<const T*>(a.A[q]) + (AKC ? m0 * a.lda[q] + k0 : m0 + k0 * a.lda[q]); };
    auto slabB = [&](int q, i64 k0) { return static_cast<const T*>(a.B[q]) + (BKC ? n0 * a.ldb[q] + k0 : n0 + k0 * a.ldb[q]); };

    // LDS-DMA: where the next slab starts, what a step adds, and the lanes' places
    // in it.  (All of it in registers: an argument read again in the loop would
    // cost a scalar load and its wait in every step.)
    const i64 kfull = a.kfull;
    const int nsteps = a.nsteps;
    const char *xa[NA], *xb;
    i64 da[NA], db;
    uint32_t offA[NA][PA], offB[PB];
    auto aim = [&](int p, i64 k0) {
        #pragma unroll
        for (int h = 0; h < NA; ++h) {
            const int q = GATED ? h : p;
            const i64 ld = a.lda[q];
            xa[h] = reinterpret_cast<const char*>(slabA(q, k0));
            da[h] = (AKC ? KB : KB * ld) * (i64)sizeof(T);
            #pragma unroll
            for (int i = 0; i < PA; ++i) offA[h][i] = IA::template offset<W>(min(wid + i * NW, PCA - 1), lane, ld, rowsA);
        }
        const i64 ld = a.ldb[p];
        xb = reinterpret_cast<const char*>(slabB(p, k0));
        db = (BKC ? KB : KB * ld) * (i64)sizeof(T);
        #pragma unroll
        for (int i = 0; i < PB; ++i) offB[i] = IB::template offset<W>(min(wid + i * NW, PCB - 1), lane, ld, rowsB);
    };
    int curp = pair, kt = s0;                             // product, and its step being staged
    while (curp + 1 < a.terms && kt >= nsteps) { kt -= nsteps; ++curp; }
    if constexpr (DMA) aim(curp, (i64)kt * KB);

    // stages one step after the other
    auto issue = [&](char* slot) {
        if (sum && kt == nsteps) { kt = 0; aim(++curp, 0); }
        const i64 k0 = (i64)kt++ * KB;
        if (k0 < kfull) {
            #pragma unroll
            for (int h = 0; h < NA; ++h) {
                #pragma unroll
                for (int i = 0; i < PA; ++i)
                    ga_to_lds<W>(xa[h] + offA[h][i], slot + h * IA::BYTES + min(wid + i * NW, PCA - 1) * (64 * W));
                xa[h] += da[h];
            }
            #pragma unroll
            for (int i = 0; i < PB; ++i)
                ga_to_lds<W>(xb + offB[i], slot + BM * 128 + min(wid + i * NW, PCB - 1) * (64 * W));
            xb += db;
        } else {
            // it may take fewer DMA instructions than the counted wait allows for: the
            // slabs before it have landed first
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            #pragma unroll
            for (int h = 0; h < NA; ++h)
                IA::template stage<W, NW>(slabA(GATED ? h : curp, k0), a.lda[GATED ? h : curp], AKC ? a.k : a.m, rowsA,
                                          a.k - k0, slot + h * IA::BYTES, wid, lane);
            IB::template stage<W, NW>(slabB(curp, k0), a.ldb[curp], BKC ? a.k : a.n, rowsB, a.k - k0, slot + BM * 128,
                                      wid, lane);
        }
    };

    // through registers: slab s + 1 is in one of two sets while slab s is
    // multiplied and slab s + 2 is fetched into the other
    constexpr int QA = IA::BYTES / 16, QB = IB::BYTES / 16, CA = DMA ? 1 : (QA + NT - 1) / NT, CB = DMA ? 1 : (QB + NT - 1) / NT;
    struct Held {
        i4v a[NA][CA], b[CB];
        int sa[NA][CA], sb[CB];
        bool whole;
    };
    typename IA::Slot slotA[NA][CA];
    typename IB::Slot slotB[CB];
    const T *ya[NA], *yb;
    i64 ea[NA], eb;
    const i64 kA = AKC ? a.lenA : a.k, kB = BKC ? a.lenB : a.k, availA = a.lenA - m0, availB = a.lenB - n0;
    int fetched = s0;
    auto point = [&](int p, i64 k0) {
        #pragma unroll
        for (int h = 0; h < NA; ++h) {
            const i64 ld = a.lda[GATED ? h : p];
            ya[h] = slabA(GATED ? h : p, k0);
            ea[h] = AKC ? KB : KB * ld;
            #pragma unroll
            for (int i = 0; i < CA; ++i) slotA[h][i] = IA::slot(min(tid + i * NT, QA - 1), ld, rowsA, availA);
        }
        const i64 ld = a.ldb[p];
        yb = slabB(p, k0);
        eb = BKC ? KB : KB * ld;
        #pragma unroll
        for (int i = 0; i < CB; ++i) slotB[i] = IB::slot(min(tid + i * NT, QB - 1), ld, rowsB, availB);
    };
    if constexpr (!DMA) point(curp, (i64)kt * KB);
    // (after the last slab it reads that one again)
    auto fetch = [&](Held& x) {
        if (sum && kt == nsteps) { kt = 0; point(++curp, 0); }
        const int lA = (int)min(kA - (i64)kt * KB, (i64)KB), lB = (int)min(kB - (i64)kt * KB, (i64)KB);
        x.whole = lA == KB && lB == KB && (AKC || availA >= BMI) && (BKC || availB >= BN);
        #pragma unroll
        for (int h = 0; h < NA; ++h)
            #pragma unroll
            for (int i = 0; i < CA; ++i) x.a[h][i] = IA::load(ya[h], slotA[h][i], lA, x.sa[h][i]);
        #pragma unroll
        for (int i = 0; i < CB; ++i) x.b[i] = IB::load(yb, slotB[i], lB, x.sb[i]);
        if (++fetched < s1) {
            ++kt;
            #pragma unroll
            for (int h = 0; h < NA; ++h) ya[h] += ea[h];
            yb += eb;
        }
    };
    auto write = [&](int s, const Held& x) {
        char* slot = smem + (s % S) * SLOT;
        auto put = [&](auto whole) {
            #pragma unroll
            for (int h = 0; h < NA; ++h)
                #pragma unroll
                for (int i = 0; i < CA; ++i)
                    *reinterpret_cast<i4v*>(slot + h * IA::BYTES + min(tid + i * NT, QA - 1) * 16) =
                        whole ? x.a[h][i] : ga_shift(x.a[h][i], x.sa[h][i]);
            #pragma unroll
            for (int i = 0; i < CB; ++i)
                *reinterpret_cast<i4v*>(slot + BM * 128 + min(tid + i * NT, QB - 1) * 16) =
                    whole ? x.b[i] : ga_shift(x.b[i], x.sb[i]);
        };
        if (x.whole) put(std::true_type());
        else put(std::false_type());
    };
    Held held0, held1;

    const int wm = wid / WVN, wn = wid % WVN;
    acc4 acc[MI][NI];
    #pragma unroll
    for (int i = 0; i < MI; ++i)
        #pragma unroll
        for (int j = 0; j < NI; ++j)
            #pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = R(0);

    if (s0 < s1) {
        if constexpr (DMA) {
            #pragma unroll
            for (int i = 0; i < S - 1; ++i)
                if (s0 + i < s1) issue(smem + (s0 + i) % S * SLOT);
        } else {
            fetch(held0);
            write(s0, held0);
            fetch(held1);
        }
    }
    auto reads = [&](const char* la, int kk, i4v (&fa)[MI], i4v (&fb)[NI]) {
        constexpr int H = MI / NA;
        #pragma unroll
        for (int j = 0; j < NI; ++j) fb[j] = IB::frag(la + BM * 128, wn * WN + j * 16, kk, lane);
        #pragma unroll
        for (int i = 0; i < MI; ++i)
            fa[i] = IA::frag(la + (i / H) * IA::BYTES, wm * (WM / NA) + (i % H) * 16, kk, lane);
    };
    auto products = [&](const i4v (&fa)[MI], const i4v (&fb)[NI]) {
        // (an accumulator's next MFMA comes after all the others')
        #pragma unroll
        for (int u = 0; u < TR::N; ++u)
            #pragma unroll
            for (int i = 0; i < MI; ++i)
                #pragma unroll
                for (int j = 0; j < NI; ++j) {
                    // D's four registers run along the rows of the first operand: rows
                    // of C for f32 sums; for f64 they are 4 apart, and the columns take
                    // them so that lanes run along the rows
                    if constexpr (sizeof(R) == 4) acc[i][j] = TR::mma(fa[i], fb[j], acc[i][j], u);
                    else acc[i][j] = TR::mma(fb[j], fa[i], acc[i][j], u);
                }
    };
    // (In both loops the slab read and the one filled are restrict parameters:
    // different memory, or the compiler waits for the DMA before each transposed
    // read.)
    if constexpr (NW == 8) {
        // Two waves share a SIMD: one reads its fragments while the other's
        // products run, in turns of half a step between barriers.  The second
        // half of the workgroup is one turn behind the first, which costs one
        // barrier at either end.
        const bool late = wid >= 4;
        auto turn = [&]() {
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        };
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        turn();
        if (late) turn();
        for (int s = s0; s < s1; ++s) {
            auto work = [&](const char* __restrict la, char* __restrict fill) __attribute__((always_inline)) {
                #pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    i4v fa[MI], fb[NI];
                    // the slot behind was read to its end a turn ago by the later half
                    if (kk == 0 && s + 1 < s1) issue(fill);
                    reads(la, kk, fa, fb);
                    // the next slab is there when the first half comes to read it:
                    // one turn after this for the later half, two for the first
                    if (kk == 1 && late) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    turn();
                    __builtin_amdgcn_s_setprio(1);
                    products(fa, fb);
                    __builtin_amdgcn_s_setprio(0);
                    if (kk == 1 && !late) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    turn();
                }
            };
            work(smem + s % S * SLOT, smem + (s + S - 1) % S * SLOT);
        }
        if (!late) turn();
    } else {
        auto step = [&](int s, Held& next, Held& spare) __attribute__((always_inline)) {
            // my part of step s has landed (of the steps behind it, LOADS each are in
            // flight, or less where all before that one had landed) ...
            if constexpr (!DMA) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            else if (S > 2 && s + S - 2 < s1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"((S - 2) * LOADS) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            // ... and everyone's, and everyone has read step s - 1's slot
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            auto work = [&](const char* __restrict la, char* __restrict fill) __attribute__((always_inline)) {
                if constexpr (!DMA) fetch(spare);
                else if (s + S - 1 < s1) issue(fill);
                #pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    i4v fa[MI], fb[NI];
                    reads(la, kk, fa, fb);
                    products(fa, fb);
                }
            };
            work(smem + s % S * SLOT, smem + (s + S - 1) % S * SLOT);
            if constexpr (!DMA)
                if (s + 1 < s1) write(s + 1, next);
        };
        if constexpr (DMA) {
            for (int s = s0; s < s1; ++s) step(s, held0, held1);
        } else {
            for (int s = s0; s < s1; s += 2) {
                step(s, held1, held0);
                if (s + 1 < s1) step(s + 1, held0, held1);
            }
        }
    }

    constexpr int H = MI / NA, WH = WM / NA;
    const i64 mw = m0 + wm * WH, nw = n0 + wn * WN;
    // row and column, inside the wave's tile, of register r of fragment (i, j)
    auto row_of = [&](int i, int r) { return i * 16 + (sizeof(R) == 4 ? (lane >> 4) * 4 + r : (lane & 15)); };
    auto col_of = [&](int j, int r) { return j * 16 + (sizeof(R) == 4 ? (lane & 15) : (lane >> 4) + 4 * r); };
    if (a.splits > 1) {
        const int planes = GATED ? 2 : (int)gridDim.z;
        #pragma unroll
        for (int i = 0; i < MI; ++i)
            #pragma unroll
            for (int j = 0; j < NI; ++j) {
                const i64 plane = (i64)blockIdx.y * planes + (GATED ? i / H : pair);
                if constexpr (sizeof(R) == 4) {
                    const i64 m = mw + row_of(i % H, 0), n = nw + col_of(j, 0);
                    if (m < a.m && n < a.n)
                        *reinterpret_cast<f4*>(static_cast<float*>(a.part) + (plane * a.n + n) * a.ldp + m) = acc[i][j];
                } else {
                    #pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const i64 m = mw + row_of(i % H, r), n = nw + col_of(j, r);
                        if (m < a.m && n < a.n) static_cast<R*>(a.part)[(plane * a.n + n) * a.ldp + m] = acc[i][j][r];
                    }
                }
            }
        return;
    }
    using EP = GaEpi<T, BM, BN, WVM, WVN, S>;
    constexpr int NJ = EP::NJ, LDR = EP::LDR, V = 16 / (int)sizeof(T);
    R* img = reinterpret_cast<R*>(smem) + wid * (LDR * 16 * NJ);
    __syncthreads();                                 // every wave has read its last slab
    #pragma unroll 1
    for (int pass = 0; pass < NI / NJ; ++pass) {
        #pragma unroll
        for (int q = 0; q < NI / NJ; ++q)
            if (q == pass) {
                #pragma unroll
                for (int i = 0; i < MI; ++i)
                    #pragma unroll
                    for (int jj = 0; jj < NJ; ++jj)
                        #pragma unroll
                        for (int r = 0; r < 4; ++r)
                            img[col_of(jj, r) * LDR + (i / H) * WH + row_of(i % H, r)] = acc[i][q * NJ + jj][r];
            }
        // a wave reads what it wrote itself: its LDS accesses complete in order
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        #pragma unroll 1
        for (int t = lane; t < (WH / V) * 16 * NJ; t += 64) {
            const int rr = (t % (WH / V)) * V, cc = t / (WH / V);
            R x[V], y[V];
            #pragma unroll
            for (int r = 0; r < V; ++r) {
                x[r] = img[cc * LDR + rr + r];
                if constexpr (GATED) y[r] = img[cc * LDR + WH + rr + r];
            }
            ga_finish<T, V, GATED, BM == 256>(a, pair, mw + rr, nw + pass * (16 * NJ) + cc, x, y);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// ------------------------------------------------------------ few columns
// C of up to 16 columns (tokens), both operands contiguous along k: bound by
// reading op(A) once.  A workgroup takes 16 rows and all of K, its NW waves
// interleaved slabs of 128 bytes per row, fragments straight from memory to
// registers with 2 U of them in flight per wave and operand (no LDS, no
// barrier in the loop); the waves' sums are added in LDS in their order.
// One column: 4096 x 4096 bf16 9.1 us (3.7 TB/s), f64 27 us (5.0 TB/s), two f16
// matrices of 8192 x 4096 29 us (4.6 TB/s).  Columns of 16-bit elements that lie
// across 4 bytes take twice the time (bf16 5120 x 11771 65 us, 11776 32; two f16 of
// 8192 x 4096 57), columns across 16 bytes alone a tenth more (11772: 35; f32
// 4096 x 4095 17.3, 4096 15.5).
template <typename T, bool GATED, int NW>
__global__ void __launch_bounds__(64 * NW) gemm_act_skinny_kernel(GemmActArgs a) {
    using TR = ga_traits<T>;
    using acc4 = typename TR::acc4;
    using R = typename TR::acc;
    constexpr int NA = GATED ? 2 : 1, E = 16 / (int)sizeof(T), KB = 8 * E, U = 4, LD = 16 + 16 / (int)sizeof(R);
    __shared__ __align__(16) R red[NW][NA][16 * LD];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 15, g = lane >> 4;
    const i64 m0 = (i64)xcd_remap(blockIdx.x, gridDim.x) * 16;
    // rows and columns past the matrix read one that exists and are not stored
    const T* pa[NA];
    #pragma unroll
    for (int h = 0; h < NA; ++h) pa[h] = static_cast<const T*>(a.A[h]) + min(m0 + l, a.m - 1) * a.lda[h] + g * E;
    const T* pb = static_cast<const T*>(a.B[0]) + min((i64)l, a.n - 1) * a.ldb[0] + g * E;
    acc4 acc[NA];
    #pragma unroll
    for (int h = 0; h < NA; ++h)
        #pragma unroll
        for (int r = 0; r < 4; ++r) acc[h][r] = R(0);
    auto mul = [&](const i4v (&fa)[NA], i4v fb) {
        #pragma unroll
        for (int u = 0; u < TR::N; ++u)
            #pragma unroll
            for (int h = 0; h < NA; ++h) {
                if constexpr (sizeof(R) == 4) acc[h] = TR::mma(fa[h], fb, acc[h], u);
                else acc[h] = TR::mma(fb, fa[h], acc[h], u);
            }
    };
    const int slabs = (int)(a.k / KB);
    using vE = ga_vec<T, E>;
    auto get = [](const T* p) { return __builtin_bit_cast(i4v, *reinterpret_cast<const vE*>(p)); };
    // the ragged end of K: its loads come first, its products last
    const bool rag = a.k % KB != 0 && slabs % NW == w;
    i4v ra[2][NA], rb[2];
    int down[2] = {0, 0};
    if (rag)
        #pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const i64 k = (i64)slabs * KB + kk * (4 * E), end = a.k - E - g * E;
            const int left = (int)max((i64)0, min((i64)E, a.k - k - g * E));
            auto last = [&](const T* p) {
                if (a.k >= E) return get(p + min(k, end));       // a column's last 16 bytes, to be shifted down
                vE x;
                #pragma unroll
                for (int e = 0; e < E; ++e) x[e] = e < left ? p[k + e] : (T)0;
                return __builtin_bit_cast(i4v, x);
            };
            if (a.k >= E) down[kk] = left ? (E - left) * (int)sizeof(T) * 8 : 128;
            #pragma unroll
            for (int h = 0; h < NA; ++h) ra[kk][h] = last(pa[h]);
            rb[kk] = last(pb);
        }
    // (slabs that do not exist end the loads: guarded one by one, each guard waits
    // for the loads before it, 5120 x 5888 f32 times one column 55 us against 33)
    auto batch = [&](int s, auto whole) __attribute__((always_inline)) {
        i4v fa[2 * U][NA], fb[2 * U];
        #pragma unroll
        for (int u = 0; u < 2 * U; ++u) {
            if (!whole && s + (u >> 1) * NW >= slabs) break;
            const i64 k = (i64)(s + (u >> 1) * NW) * KB + (u & 1) * (4 * E);
            #pragma unroll
            for (int h = 0; h < NA; ++h) fa[u][h] = get(pa[h] + k);
            fb[u] = get(pb + k);
        }
        __builtin_amdgcn_sched_barrier(0);                       // all of them in flight
        #pragma unroll
        for (int u = 0; u < 2 * U; ++u)
            if (whole || s + (u >> 1) * NW < slabs) mul(fa[u], fb[u]);
    };
    int s = w;
    for (; s + (U - 1) * NW < slabs; s += U * NW) batch(s, std::true_type());
    for (; s < slabs; s += U * NW) batch(s, std::false_type());
    if (rag)
        #pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            #pragma unroll
            for (int h = 0; h < NA; ++h) ra[kk][h] = ga_shift(ra[kk][h], down[kk]);
            mul(ra[kk], ga_shift(rb[kk], down[kk]));
        }
    #pragma unroll
    for (int h = 0; h < NA; ++h)
        #pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = sizeof(R) == 4 ? g * 4 + r : l, col = sizeof(R) == 4 ? l : g + 4 * r;
            red[w][h][col * LD + row] = acc[h][r];
        }
    __syncthreads();
    for (int t = threadIdx.x; t < 256; t += 64 * NW) {
        const int col = t >> 4, row = t & 15;
        if (col >= a.n) break;
        R x[NA];
        #pragma unroll
        for (int h = 0; h < NA; ++h) {
            x[h] = red[0][h][col * LD + row];
            #pragma unroll
            for (int q = 1; q < NW; ++q) x[h] += red[q][h][col * LD + row];
        }
        ga_finish<T, 1, GATED>(a, 0, m0 + row, col, &x[0], &x[NA - 1]);
    }
}

// Columns laid out anew on 16 bytes, with zeros behind their ends, so that
// LDS-DMA takes them; a thread moves four 16-byte vectors.  Bound by
// memory: 1636 x 5721 8.7 us (4.3 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) ga_pack_kernel(const T* X, i64 ld, T* Y, i64 len, i64 cols) {
    constexpr int E = 16 / (int)sizeof(T), U = 4;
    using vE = ga_vec<T, E>;
    const i64 nv = (len + E - 1) / E, first = (i64)blockIdx.x * (256 * U), c0 = first / nv;
    const uint32_t r0 = (uint32_t)(first - c0 * nv) + threadIdx.x, nv32 = (uint32_t)nv;
    vE v[U];
    #pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t r = r0 + u * 256, q = r / nv32;
        const i64 c = c0 + q, i = (i64)(r - q * nv32) * E;
        if (c >= cols) continue;
        const T* x = X + c * ld + i;
        if (i + E <= len) v[u] = *reinterpret_cast<const vE*>(x);
        else
            #pragma unroll
            for (int e = 0; e < E; ++e) v[u][e] = i + e < len ? x[e] : (T)0;
    }
    #pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t r = r0 + u * 256, q = r / nv32;
        if (c0 + q < cols) *reinterpret_cast<vE*>(Y + (first + threadIdx.x + u * 256) * E) = v[u];
    }
}

// Adds the partial sums and finishes them: 64 threads along the outputs, 4
// along the pieces of K, so that small outputs (where K is split) keep enough
// loads in flight; the order of the sums depends on the plan alone.  3.5 us for
// 16 pieces of 33 x 2048, 5 us for 2 of 777 x 1001.
template <typename T, bool GATED>
__global__ void __launch_bounds__(256) gemm_act_join_kernel(GemmActArgs a) {
    using R = typename ga_traits<T>::acc;
    constexpr int V = 16 / (int)sizeof(R), NP = GATED ? 2 : 1;
    typedef R vR __attribute__((ext_vector_type(V)));
    __shared__ vR red[3][NP][64];
    const i64 mv = (a.m + V - 1) / V, t = (i64)blockIdx.x * 64 + (threadIdx.x & 63);
    const int y = threadIdx.x >> 6;
    const bool live = t < mv * a.n;
    const i64 n = live ? t / mv : 0, m = live ? (t - n * mv) * V : 0;
    const int planes = a.mode == GA_PAIR || GATED ? 2 : 1, pair = GATED ? 0 : (int)blockIdx.z;
    const i64 plane = a.n * a.ldp;
    vR x[NP];
    #pragma unroll
    for (int h = 0; h < NP; ++h) {
        #pragma unroll
        for (int r = 0; r < V; ++r) x[h][r] = R(0);
        const R* P = static_cast<const R*>(a.part) + (GATED ? h : pair) * plane + n * a.ldp + m;
        #pragma unroll 4
        for (int s = y; s < a.splits; s += 4) x[h] += *reinterpret_cast<const vR*>(P + (i64)s * planes * plane);
        if (y) red[y - 1][h][threadIdx.x & 63] = x[h];
    }
    __syncthreads();
    if (y || !live) return;
    R z[2][V];
    #pragma unroll
    for (int h = 0; h < NP; ++h) {
        #pragma unroll
        for (int q = 0; q < 3; ++q) x[h] += red[q][h][threadIdx.x];
        #pragma unroll
        for (int r = 0; r < V; ++r) z[h][r] = x[h][r];
    }
    ga_finish<T, V, GATED>(a, pair, m, n, z[0], z[NP - 1]);
}

}  // namespace slate_hip
