// Host path of the fused feed-forward products, their gradients, the common
// norm of many matrices, and copies to and from the 16-bit element types.
// Same arguments as the gfx950 entry points (csrc/hip/bindings_ffn.hip); sums
// in 64 bits, one rounding per stored element.
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>

#include <cmath>
#include <cstdint>
#include <cstring>
#include <limits>
#include <stdexcept>
#include <vector>

#include "clip_apart.hpp"

namespace py = pybind11;

namespace slate_host {

namespace {

using i64 = int64_t;

struct bf16 {
    uint16_t u;
    operator double() const {
        const uint32_t w = (uint32_t)u << 16;
        float f;
        std::memcpy(&f, &w, 4);
        return f;
    }
    static bf16 from(double d) {
        // to nearest even, from 64 bits at once (via float it would round twice)
        float f = (float)d;
        if (f != f) return {0x7fc0};
        uint32_t w;
        std::memcpy(&w, &f, 4);
        const uint32_t low = w & 0xffff;
        uint32_t up = w >> 16;
        const double back = (double)f;
        const bool more = std::fabs(back) < std::fabs(d), less = std::fabs(back) > std::fabs(d);
        if (low > 0x8000 || (low == 0x8000 && (more || (!less && (up & 1))))) ++up;
        return {(uint16_t)up};
    }
};

struct f16 {
    uint16_t u;
    operator double() const {
        const int s = u >> 15, e = (u >> 10) & 31, f = u & 1023;
        double v;
        if (e == 0) v = std::ldexp((double)f, -24);
        else if (e == 31) v = f ? std::numeric_limits<double>::quiet_NaN() : std::numeric_limits<double>::infinity();
        else v = std::ldexp((double)(1024 + f), e - 25);
        return s ? -v : v;
    }
    static f16 from(double d) {
        const uint16_t s = std::signbit(d) ? 0x8000 : 0;
        if (d != d) return {(uint16_t)(s | 0x7e00)};
        const double a = std::fabs(d);
        if (a >= 65520.0) return {(uint16_t)(s | 0x7c00)};
        int e;
        std::frexp(a, &e);                                   // a = f 2^e, f in [0.5, 1)
        if (a == 0.0) return {s};
        const int q = std::max(e - 11, -24);                 // exponent of the last place
        const i64 n = (i64)std::nearbyint(std::ldexp(a, -q));
        if (q == -24) return {(uint16_t)(s | (uint16_t)n)};  // subnormal, or carried into the first normal
        // n in [1024, 2048]; the carry runs into the exponent by itself
        return {(uint16_t)(s | (uint16_t)(((i64)(q + 24) << 10) + n))};
    }
};

template <typename T> inline T put(double v) {
    if constexpr (std::is_same<T, bf16>::value || std::is_same<T, f16>::value) return T::from(v);
    else return (T)v;
}

template <typename F> void real_dispatch(char dt, F&& f) {
    switch (dt) {
        case 'b': f(bf16()); break;
        case 'h': f(f16()); break;
        case 's': f(float()); break;
        case 'd': f(double()); break;
        default: throw std::invalid_argument("element type must be bfloat16, float16, float32 or float64");
    }
}

enum { IDENTITY, RELU, GELU, GELU_TANH, SILU };
enum { PLAIN, GATED, SUM, PAIR };

void act_grad_at(int act, double z, double& v, double& d) {
    const double x = z < -800 ? -800 : (z > 800 ? 800 : z);  // beyond, the smooth ones are 0 or z
    double p, e;
    switch (act) {
        case RELU: v = z < 0 ? 0 : z; d = z > 0 ? 1 : (z <= 0 ? 0 : z); return;
        case GELU:
            p = 0.5 * std::erfc(-x * M_SQRT1_2);
            e = 0.39894228040143267794 * std::exp(-0.5 * x * x);
            break;
        case GELU_TANH: {
            p = 1 / (1 + std::exp(-1.59576912160573071176 * (x + 0.044715 * x * x * x)));
            e = p * (1 - p) * 1.59576912160573071176 * (1 + 0.134145 * x * x);
            break;
        }
        case SILU: p = 1 / (1 + std::exp(-x)); e = p * (1 - p); break;
        default: v = z; d = 1; return;
    }
    v = z > 800 ? z : x * p;
    d = p + x * e;
}
double act_at(int act, double z) {
    double v, d;
    act_grad_at(act, z, v, d);
    return v;
}

template <typename T> T* ptr(uintptr_t p) { return reinterpret_cast<T*>(p); }

// op(A) as doubles, rows x cols column-major
template <typename T> std::vector<double> dense(uintptr_t A, i64 ld, bool t, i64 rows, i64 cols) {
    std::vector<double> D((size_t)(rows * cols));
    const T* a = ptr<const T>(A);
    for (i64 j = 0; j < cols; ++j)
        for (i64 i = 0; i < rows; ++i) D[(size_t)(i + j * rows)] = (double)(t ? a[j + i * ld] : a[i + j * ld]);
    return D;
}

// D += op(A) op(B)
void multiply(i64 m, i64 n, i64 k, const std::vector<double>& A, const std::vector<double>& B, std::vector<double>& D) {
#pragma omp parallel for schedule(static)
    for (i64 j = 0; j < n; ++j)
        for (i64 l = 0; l < k; ++l) {
            const double b = B[(size_t)(l + j * k)];
            const double* a = A.data() + l * m;
            double* d = D.data() + j * m;
            for (i64 i = 0; i < m; ++i) d[i] += a[i] * b;
        }
}

void clip_sum(char ta, const std::vector<i64>& v, double* s) {
    s[0] = s[1] = s[2] = 0;
    real_dispatch(ta, [&](auto z) {
        using T = decltype(z);
        for (size_t q = 0; q + 5 < v.size(); q += 6)
            for (i64 j = 0; j < v[q + 5]; ++j)
                for (i64 i = 0; i < v[q + 4]; ++i) {
                    const double x = (double)ptr<const T>((uintptr_t)v[q])[i + j * v[q + 1]], a = std::fabs(x);
                    if (a > 1e145) { const double w = x * 0x1p-600; s[2] += w * w; }
                    else if (a < 1e-145) { const double w = x * 0x1p600; s[0] += w * w; }
                    else s[1] += x * x;
                }
    });
}

void clip_scale(char ta, char tb, const std::vector<i64>& v, double limit, const double* s, double* norm_out, bool scale) {
    double norm;
    if (s[1] != s[1]) norm = s[1];
    else if (s[2] > 0) norm = std::sqrt(s[2] + (s[1] * 0x1p-600) * 0x1p-600) * 0x1p600;
    else if (s[1] > 0) norm = std::sqrt(s[1] + (s[0] * 0x1p-600) * 0x1p-600);
    else norm = std::sqrt(s[0]) * 0x1p-600;
    *norm_out = norm;
    if (!scale) return;
    const bool cut = norm > limit && norm < std::numeric_limits<double>::infinity();
    // the factor as f 2^e: beyond the normal numbers limit / norm has lost bits
    double f = cut ? limit / norm : 1.0;
    int e = 0, en;
    if (f < std::numeric_limits<double>::min()) {
        f = 0.5 * std::frexp(limit, &e);
        f /= std::frexp(norm, &en);                // in (1/4, 1)
        e += 1 - en;
    }
    real_dispatch(ta, [&](auto za) { real_dispatch(tb, [&](auto zb) {
        using TA = decltype(za); using TB = decltype(zb);
        for (size_t q = 0; q + 5 < v.size(); q += 6) {
            if (!cut && v[q] == v[q + 2]) continue;
            const TA* A = ptr<const TA>((uintptr_t)v[q]);
            TB* B = ptr<TB>((uintptr_t)v[q + 2]);
            for (i64 j = 0; j < v[q + 5]; ++j)
                for (i64 i = 0; i < v[q + 4]; ++i)
                    B[i + j * v[q + 3]] = put<TB>(std::ldexp((double)A[i + j * v[q + 1]] * f, e));
        }
    }); });
}

}  // namespace

void register_ffn(py::module& m) {
    m.def("gemm_act", [](char dt, int mode, char ta, char tb, i64 m, i64 n, i64 k, double alpha,
                         uintptr_t A0, i64 lda0, uintptr_t A1, i64 lda1, uintptr_t B0, i64 ldb0, uintptr_t B1, i64 ldb1,
                         uintptr_t C0, i64 ldc0, uintptr_t C1, i64 ldc1, uintptr_t bias, i64 incb, int bias_mode,
                         int act, double beta, uintptr_t R, i64 ldr, uintptr_t Z0, i64 ldz0, uintptr_t Z1, i64 ldz1,
                         const std::vector<i64>& more, uintptr_t, uintptr_t) {
        if (more.size() % 4 || (mode != SUM && !more.empty())) throw std::invalid_argument("gemm_act: bad terms of a sum");
        real_dispatch(dt, [&](auto z) {
            using T = decltype(z);
            std::vector<uintptr_t> A = {A0, A1}, B = {B0, B1};
            std::vector<i64> lda = {lda0, lda1}, ldb = {ldb0, ldb1};
            for (size_t i = 0; i < more.size(); i += 4) {
                A.push_back((uintptr_t)more[i]); lda.push_back(more[i + 1]);
                B.push_back((uintptr_t)more[i + 2]); ldb.push_back(more[i + 3]);
            }
            const uintptr_t C[2] = {C0, C1}, Z[2] = {Z0, Z1};
            const i64 ldc[2] = {ldc0, ldc1}, ldz[2] = {ldz0, ldz1};
            std::vector<double> D[2];
            const int outs = mode == GATED || mode == PAIR ? 2 : 1, sums = mode == SUM ? (int)A.size() : 1;
            for (int h = 0; h < outs; ++h) {
                D[h].assign((size_t)(m * n), 0.0);
                for (int p = 0; p < sums; ++p) {
                    const int ia = h + p, ib = mode == GATED ? 0 : h + p;
                    multiply(m, n, k, dense<T>(A[ia], lda[ia], ta != 'N', m, k),
                             dense<T>(B[ib], ldb[ib], tb != 'N', k, n), D[h]);
                }
            }
            for (i64 j = 0; j < n; ++j)
                for (i64 i = 0; i < m; ++i) {
                    const size_t at = (size_t)(i + j * m);
                    if (mode == GATED) {
                        if (Z0) ptr<T>(Z0)[i + j * ldz0] = put<T>(D[0][at]);
                        if (Z1) ptr<T>(Z1)[i + j * ldz1] = put<T>(D[1][at]);
                        ptr<T>(C0)[i + j * ldc0] = put<T>(act_at(act, D[0][at]) * D[1][at]);
                        continue;
                    }
                    for (int h = 0; h < outs; ++h) {
                        double v = alpha * D[h][at];
                        if (bias_mode) v += (double)ptr<const T>(bias)[(bias_mode == 1 ? i : j) * incb];
                        if (Z[h]) ptr<T>(Z[h])[i + j * ldz[h]] = put<T>(v);
                        v = act_at(act, v);
                        if (R) v += beta * (double)ptr<const T>(R)[i + j * ldr];
                        ptr<T>(C[h])[i + j * ldc[h]] = put<T>(v);
                    }
                }
        });
        return (i64)0;                      // no workspace is wanted
    });
    m.def("act_grad_ws", [](char, int, i64, i64) { return (i64)0; });
    m.def("act_grad", [](char dt, i64 m, i64 n, int act, uintptr_t dC, i64 lddc, uintptr_t Z1, i64 ldz1, uintptr_t Z2,
                         i64 ldz2, uintptr_t dZ1, uintptr_t dZ2, uintptr_t dL1, uintptr_t dL2, i64 lddz, uintptr_t db, i64 incb, int bias_mode,
                         bool wide, uintptr_t, uintptr_t) {
        real_dispatch(dt, [&](auto z) {
            using T = decltype(z);
            std::vector<double> sum((size_t)(bias_mode == 1 ? m : bias_mode == 2 ? n : 0), 0.0);
            for (i64 j = 0; j < n; ++j)
                for (i64 i = 0; i < m; ++i) {
                    double v = 0, d = 1;
                    if (Z1) act_grad_at(act, (double)ptr<const T>(Z1)[i + j * ldz1], v, d);
                    const double g = (double)ptr<const T>(dC)[i + j * lddc];
                    const double d1 = Z2 ? g * (double)ptr<const T>(Z2)[i + j * ldz2] * d : g * d;
                    if (dZ1) ptr<T>(dZ1)[i + j * lddz] = put<T>(d1);
                    if (dZ2) ptr<T>(dZ2)[i + j * lddz] = put<T>(g * v);
                    // what their rounding leaves over (nothing of an infinity or a NaN)
                    auto rest = [](double d) { const double h = (double)put<T>(d); return put<T>(std::isfinite(h) ? d - h : 0.0); };
                    if (dL1) ptr<T>(dL1)[i + j * lddz] = rest(d1);
                    if (dL2) ptr<T>(dL2)[i + j * lddz] = rest(g * v);
                    if (bias_mode) sum[(size_t)(bias_mode == 1 ? i : j)] += d1;
                }
            for (size_t i = 0; i < sum.size(); ++i) {
                if (!wide) ptr<T>(db)[(i64)i * incb] = put<T>(sum[i]);
                else if constexpr (sizeof(T) == 8) ptr<double>(db)[(i64)i * incb] = sum[i];
                else ptr<float>(db)[(i64)i * incb] = (float)sum[i];
            }
        });
    });
    // matrices: A, lda, B, ldb, rows, columns one after the other; the sums of
    // squares of small, ordinary and large elements (see csrc/hip/clip.hip)
    m.def("clip_parts", [](i64) { return (i64)3; });
    m.def("clip_sum", [](char ta, const std::vector<i64>& v, uintptr_t part, uintptr_t) {
        clip_sum(ta, v, ptr<double>(part));
        return (i64)1;
    });
    m.def("clip_join", [](uintptr_t part, i64, uintptr_t out, uintptr_t) {
        std::memcpy(ptr<void>(out), ptr<const void>(part), 3 * sizeof(double));
    });
    m.def("clip_scale", [](char ta, char tb, const std::vector<i64>& v, double limit, uintptr_t part, i64,
                           uintptr_t norm, bool scale, uintptr_t) {
        clip_scale(ta, tb, v, limit, ptr<const double>(part), ptr<double>(norm), scale);
    });
    m.def("clip_norm", [](char ta, char tb, const std::vector<i64>& v, double limit, uintptr_t part, uintptr_t norm,
                          bool scale, bool look, uintptr_t) {
        auto es = [](char t) { return t == 'd' ? 8 : t == 's' ? 4 : 2; };
        if (v.size() % 6) throw std::invalid_argument("clip: six integers per matrix are wanted");
        if (scale && look && !clip_apart(v.data(), v.size() / 6, es(ta), es(tb))) return false;
        clip_sum(ta, v, ptr<double>(part));
        clip_scale(ta, tb, v, limit, ptr<const double>(part), ptr<double>(norm), scale);
        return true;
    });
    m.def("gecopy16", [](char ds, char dd, char uplo, char trans, i64 mm, i64 n, uintptr_t A, i64 lda, uintptr_t B,
                         i64 ldb, uintptr_t) {
        real_dispatch(ds, [&](auto zs) { real_dispatch(dd, [&](auto zd) {
            using Ts = decltype(zs); using Td = decltype(zd);
            for (i64 j = 0; j < n; ++j)
                for (i64 i = 0; i < mm; ++i) {
                    if ((uplo == 'L' && i < j) || (uplo == 'U' && i > j)) continue;
                    const Ts x = trans == 'N' ? ptr<const Ts>(A)[i + j * lda] : ptr<const Ts>(A)[j + i * lda];
                    if constexpr (std::is_same<Ts, Td>::value) ptr<Td>(B)[i + j * ldb] = x;
                    else ptr<Td>(B)[i + j * ldb] = put<Td>((double)x);
                }
        }); });
    });
}

}  // namespace slate_host
