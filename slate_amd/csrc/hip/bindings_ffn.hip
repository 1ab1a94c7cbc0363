// pybind11 entry points of the fused feed-forward products, their gradients,
// gradient clipping, and copies to and from the 16-bit element types.
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include "ffn.hpp"
#include "clip_apart.hpp"

namespace py = pybind11;
using namespace slate_hip;

namespace {

inline hipStream_t S(uintptr_t s) { return reinterpret_cast<hipStream_t>(s); }
inline const void* P(uintptr_t p) { return reinterpret_cast<const void*>(p); }
inline void* W(uintptr_t p) { return reinterpret_cast<void*>(p); }

template <typename F> void real_dispatch(char dt, F&& f) {
    switch (dt) {
        case 'b': f(__bf16()); break;
        case 'h': f(_Float16()); break;
        case 's': f(float()); break;
        case 'd': f(double()); break;
        default: throw std::invalid_argument("element type must be bfloat16, float16, float32 or float64");
    }
}

std::vector<i64> ints(const py::list& v) {
    const Py_ssize_t n = PyList_GET_SIZE(v.ptr());
    std::vector<i64> x(n);
    for (Py_ssize_t i = 0; i < n; ++i) x[i] = PyLong_AsLongLong(PyList_GET_ITEM(v.ptr(), i));
    if (PyErr_Occurred()) throw py::error_already_set();
    return x;
}
// six integers per matrix: A, lda, B, ldb, rows, columns
std::vector<ClipMat> mats(const std::vector<i64>& v) {
    if (v.size() % 6) throw std::invalid_argument("clip: six integers per matrix are wanted");
    std::vector<ClipMat> c;
    c.reserve(v.size() / 6);
    for (size_t i = 0; i < v.size(); i += 6) {
        const i64* x = &v[i];
        if (x[4] > 0 && x[5] > 0) c.push_back({P((uintptr_t)x[0]), W((uintptr_t)x[2]), x[4], x[5], x[1], x[3]});
    }
    return c;
}
int bytes_of(char t) { return t == 'd' ? 8 : t == 's' ? 4 : 2; }

// A backward pass: dZ (and the bias gradient), then the products that read it.
// v: rows, columns, act, dC, ldc, Z1, ldz1, Z2, ldz2, db, incb, bias_mode, how many
// dZ are made, whether with what their rounding leaves over, and T; then 10 + 4 T
// integers for each product: mode, op(A) and op(B) transposed, m, n, k and address
// and leading dimension of T matrices A, T matrices B, C and C2, where the address
// -1 - i is the i-th dZ made here (the rests behind them).  The workspace holds them, the bias
// gradient's partial sums, and behind them what one product after the other wants.
// -> its size; without one nothing is launched.
template <typename T> i64 ffn_grad(double alpha, const std::vector<i64>& v, char* ws, hipStream_t s) {
    constexpr size_t HEAD = 15;
    const int nt = v.size() < HEAD ? 0 : (int)v[14];
    const size_t PER = 10 + 4 * nt;
    if (nt < 2 || nt > 4 || (v.size() - HEAD) % PER)
        throw std::invalid_argument("ffn_grad: 15 + (10 + 4 T) n integers are wanted, T 2 to 4");
    auto round = [](i64 x, i64 to) { return (x + to - 1) / to * to; };
    ActGradArgs g;
    g.m = v[0]; g.n = v[1]; g.act = (int)v[2];
    g.dC = P((uintptr_t)v[3]); g.lddc = v[4];
    g.Z1 = P((uintptr_t)v[5]); g.ldz1 = v[6];
    g.Z2 = P((uintptr_t)v[7]); g.ldz2 = v[8];
    g.db = W((uintptr_t)v[9]); g.incb = v[10]; g.bias_mode = (int)v[11];
    const int made = (int)v[12], ndz = v[13] ? 2 * made : made;
    g.lddz = round(std::max<i64>(g.m, 1), g.m >= 64 ? 64 : 8);
    const i64 dz = round(g.lddz * g.n * (i64)sizeof(T), 256);
    const i64 sums = g.bias_mode ? (i64)act_grad_chunks(g.bias_mode, sizeof(T), g.m, g.n) * (g.bias_mode == 1 ? g.m : g.n) *
                                       (sizeof(T) == 8 ? 8 : 4) : 0;
    const i64 rest = round(ndz * dz + sums, 256);
    // (an address to plan with: as aligned as the workspace's)
    char* base = ws ? ws : reinterpret_cast<char*>(4096);
    if (ws && (ndz || g.bias_mode)) {
        if (made > 0) g.dZ1 = base;
        if (made > 1) g.dZ2 = base + dz;
        if (ndz > made) g.dL1 = base + made * dz;
        if (ndz > made && made > 1) g.dL2 = base + 3 * dz;
        g.part = base + ndz * dz;
        act_grad<T>(g, s);
    }
    i64 most = 0;
    for (size_t i = HEAD; i < v.size(); i += PER) {
        const i64* x = &v[i];
        GemmActArgs a;
        a.alpha = alpha;
        a.mode = (int)x[0];
        a.m = x[3]; a.n = x[4]; a.k = x[5];
        auto at = [&](int j, i64& ld) -> void* {
            ld = x[j + 1];
            if (x[j] >= 0 || x[j] < -ndz) return W((uintptr_t)x[j]);
            ld = g.lddz;
            return base + (-1 - x[j]) * dz;
        };
        for (int j = 0; j < nt; ++j) {
            a.A[j] = at(6 + 2 * j, a.lda[j]);
            a.B[j] = at(6 + 2 * nt + 2 * j, a.ldb[j]);
            if (x[6 + 2 * j]) a.terms = j + 1;
        }
        for (int j = 0; j < 2; ++j) {
            a.C[j] = W((uintptr_t)x[6 + 4 * nt + 2 * j]);
            a.ldc[j] = x[7 + 4 * nt + 2 * j];
        }
        a.part = base + rest;
        a.plan = !ws;
        most = std::max(most, gemm_act<T>(a, x[1] ? 'T' : 'N', x[2] ? 'T' : 'N', s));
    }
    return rest + most;
}

}  // namespace

void register_ffn(py::module& m) {
    // Launches and returns 0, or returns the bytes of workspace that the call
    // wants where ws is 0 (nothing is launched then).
    m.def("gemm_act", [](char dt, int mode, char ta, char tb, i64 mm, i64 n, i64 k, double alpha,
                         uintptr_t A0, i64 lda0, uintptr_t A1, i64 lda1, uintptr_t B0, i64 ldb0, uintptr_t B1, i64 ldb1,
                         uintptr_t C0, i64 ldc0, uintptr_t C1, i64 ldc1, uintptr_t bias, i64 incb, int bias_mode,
                         int act, double beta, uintptr_t R, i64 ldr, uintptr_t Z0, i64 ldz0, uintptr_t Z1, i64 ldz1,
                         const py::list& more, uintptr_t ws, uintptr_t st) {
        GemmActArgs a;
        a.m = mm; a.n = n; a.k = k;
        a.mode = mode; a.alpha = alpha; a.beta = beta; a.act = act;
        a.A[0] = P(A0); a.lda[0] = lda0; a.A[1] = P(A1); a.lda[1] = lda1;
        a.B[0] = P(B0); a.ldb[0] = ldb0; a.B[1] = P(B1); a.ldb[1] = ldb1;
        a.terms = mode == GA_SUM ? 2 : 1;
        if (PyList_GET_SIZE(more.ptr())) {          // a sum's third and fourth product: A, lda, B, ldb each
            const auto x = ints(more);
            if (mode != GA_SUM || x.size() % 4 || x.size() > 8) throw std::invalid_argument("gemm_act: a sum has up to four products");
            for (size_t i = 0; i < x.size(); i += 4, ++a.terms) {
                a.A[a.terms] = P((uintptr_t)x[i]); a.lda[a.terms] = x[i + 1];
                a.B[a.terms] = P((uintptr_t)x[i + 2]); a.ldb[a.terms] = x[i + 3];
            }
        }
        a.C[0] = W(C0); a.ldc[0] = ldc0; a.C[1] = W(C1); a.ldc[1] = ldc1;
        a.Z[0] = W(Z0); a.ldz[0] = ldz0; a.Z[1] = W(Z1); a.ldz[1] = ldz1;
        a.bias = P(bias); a.incb = incb; a.bias_mode = bias_mode;
        a.R = P(R); a.ldr = ldr;
        a.part = W(ws);
        i64 bytes = 0;
        real_dispatch(dt, [&](auto z) {
            using T = decltype(z);
            bytes = gemm_act<T>(a, ta, tb, S(st));
        });
        return bytes;
    });
    m.def("act_grad_ws", [](char dt, int bias_mode, i64 mm, i64 n) {
        i64 bytes = 0;
        real_dispatch(dt, [&](auto z) {
            const int es = sizeof(z);
            if (bias_mode) bytes = (i64)act_grad_chunks(bias_mode, es, mm, n) * (bias_mode == 1 ? mm : n) * (es == 8 ? 8 : 4);
        });
        return bytes;
    });
    m.def("act_grad", [](char dt, i64 mm, i64 n, int act, uintptr_t dC, i64 lddc, uintptr_t Z1, i64 ldz1, uintptr_t Z2,
                         i64 ldz2, uintptr_t dZ1, uintptr_t dZ2, uintptr_t dL1, uintptr_t dL2, i64 lddz, uintptr_t db, i64 incb, int bias_mode,
                         bool wide, uintptr_t ws, uintptr_t st) {
        ActGradArgs a;
        a.m = mm; a.n = n; a.act = act;
        a.dC = P(dC); a.lddc = lddc; a.Z1 = P(Z1); a.ldz1 = ldz1; a.Z2 = P(Z2); a.ldz2 = ldz2;
        a.dZ1 = W(dZ1); a.dZ2 = W(dZ2); a.dL1 = W(dL1); a.dL2 = W(dL2); a.lddz = lddz;
        a.db = W(db); a.incb = incb; a.bias_mode = bias_mode; a.wide = wide;
        a.part = W(ws);
        if (bias_mode && !ws) throw std::invalid_argument("act_grad: workspace missing");
        real_dispatch(dt, [&](auto z) { act_grad<decltype(z)>(a, S(st)); });
    });
    m.def("ffn_grad", [](char dt, double alpha, const py::list& v, uintptr_t ws, uintptr_t st) {
        const auto x = ints(v);
        i64 bytes = 0;
        real_dispatch(dt, [&](auto z) { bytes = ffn_grad<decltype(z)>(alpha, x, (char*)W(ws), S(st)); });
        return bytes;
    });
    m.def("clip_parts", [](i64 count) { return clip_parts(count); });
    // false, and nothing launched, where `look` is set and address ranges of the call overlap
    m.def("clip_norm", [](char ta, char tb, const py::list& v, double limit, uintptr_t part, uintptr_t norm, bool scale,
                          bool look, uintptr_t st) {
        const auto x = ints(v);
        const auto c = mats(x);
        if (scale && look && !clip_apart(x.data(), x.size() / 6, bytes_of(ta), bytes_of(tb))) return false;
        const int n = clip_sum(ta, c.data(), (int)c.size(), (double*)W(part), S(st));
        clip_scale(ta, tb, c.data(), (int)c.size(), limit, (const double*)P(part), n, (double*)W(norm), scale, S(st));
        return true;
    });
    m.def("clip_sum", [](char ta, const py::list& v, uintptr_t part, uintptr_t st) {
        const auto c = mats(ints(v));
        return (i64)clip_sum(ta, c.data(), (int)c.size(), (double*)W(part), S(st));
    });
    m.def("clip_join", [](uintptr_t part, i64 parts, uintptr_t out, uintptr_t st) {
        clip_join((const double*)P(part), (int)parts, (double*)W(out), S(st));
    });
    m.def("clip_scale", [](char ta, char tb, const py::list& v, double limit, uintptr_t part, i64 parts, uintptr_t norm,
                           bool scale, uintptr_t st) {
        const auto c = mats(ints(v));
        clip_scale(ta, tb, c.data(), (int)c.size(), limit, (const double*)P(part), (int)parts, (double*)W(norm), scale,
                   S(st));
    });
    m.def("gecopy16", [](char ds, char dd, char uplo, char trans, i64 mm, i64 n, uintptr_t A, i64 lda, uintptr_t B,
                         i64 ldb, uintptr_t st) {
        real_dispatch(ds, [&](auto zs) { real_dispatch(dd, [&](auto zd) {
            using Ts = decltype(zs); using Td = decltype(zd);
            gecopy16<Ts, Td>(uplo, trans, mm, n, static_cast<const Ts*>(P(A)), lda, static_cast<Td*>(W(B)), ldb, S(st));
        }); });
    });
}
