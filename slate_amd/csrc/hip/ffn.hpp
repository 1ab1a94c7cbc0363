// Feed-forward products with fused epilogues, their backward passes, and the
// clipping of many gradients by their common norm: types and launchers.
#pragma once
#include "common.hpp"

namespace slate_hip {

enum : int { ACT_IDENTITY = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_GELU_TANH = 3, ACT_SILU = 4 };
enum : int { GA_PLAIN = 0, GA_GATED = 1, GA_SUM = 2, GA_PAIR = 3 };

// ---------------------------------------------------------------- arguments
struct GemmActArgs {
    i64 m = 0, n = 0, k = 0;
    const void* A[4] = {};
    const void* B[4] = {};
    void* C[2] = {nullptr, nullptr};
    void* Z[2] = {nullptr, nullptr};
    i64 lda[4] = {}, ldb[4] = {}, ldc[2] = {0, 0}, ldz[2] = {0, 0};
    const void* bias = nullptr;
    const void* R = nullptr;
    i64 incb = 1, ldr = 0;
    double alpha = 1, beta = 0;
    int mode = GA_PLAIN;
    int terms = 1;          // GA_SUM: how many products are added (2 to 4)
    int bias_mode = 0;      // 0 none, 1 one value per row of C, 2 one per column
    int act = ACT_IDENTITY;
    // filled by the launcher
    i64 kfull = 0;          // first k that LDS-DMA does not stage
    i64 lenA = 0, lenB = 0; // length of the operands' columns, 16 bytes or more where they go through registers
    int nsteps = 0;         // K steps per product
    int group_m = 8;
    int splits = 1, per_split = 0;
    void* part = nullptr;   // splits > 1: partial sums, plane (split, i) of n columns of ldp
    i64 ldp = 0;
    bool plan = false;      // only the workspace wanted is returned, nothing launched
};

// Which kernel, and in how many pieces K: from sizes, types and alignment alone.
// tile -1: the kernel for few columns; bytes: workspace.
struct GemmActPlan { int tile = 0, splits = 1, per_split = 0; i64 ldp = 0, bytes = 0; };
GemmActPlan gemm_act_plan(int es, int mode, int terms, i64 m, i64 n, i64 k, bool akc, bool bkc, bool dma);
bool gemm_act_pack(int mode, int terms, i64 m, i64 n, i64 k);    // lay operands whose rows lie across 16 bytes out anew?
// Launches and returns 0, or returns the workspace wanted where part is null.
template <typename T> i64 gemm_act(GemmActArgs a, char ta, char tb, hipStream_t s);

// dZ = dC o act'(Z) (dZ1 = dC o Z2 o act'(Z1), dZ2 = dC o act(Z1) where Z2 is
// given), and the sums of dZ over the columns (bias_mode 1) or rows (2).  Where
// dL1 (dL2) is given, 16-bit types: what the rounding of dZ left over, rounded
struct ActGradArgs {
    i64 m = 0, n = 0;
    const void *dC = nullptr, *Z1 = nullptr, *Z2 = nullptr;
    void *dZ1 = nullptr, *dZ2 = nullptr, *dL1 = nullptr, *dL2 = nullptr;
    i64 lddc = 0, ldz1 = 0, ldz2 = 0, lddz = 0;
    void* db = nullptr;
    i64 incb = 1;
    int bias_mode = 0, act = 0;
    bool wide = false;        // db in the sums' type, not T
    void* part = nullptr;     // bias_mode 1: chunks x m (2: x n) sums
};
int act_grad_chunks(int bias_mode, int es, i64 m, i64 n);
template <typename T> void act_grad(ActGradArgs a, hipStream_t s);

// clip.hip: s = sqrt(sum_i |A_i|^2), B_i = min(1, limit / s) A_i, over any
// number of matrices.  part: clip_parts() doubles, three (sums of squares of
// small, ordinary and large elements) per block of the first pass.
struct ClipMat { const void* A; void* B; i64 m, n, lda, ldb; };
i64 clip_parts(i64 count);
int clip_sum(char ta, const ClipMat* v, int count, double* part, hipStream_t s);          // -> partial sums written
void clip_join(const double* part, int parts, double* out, hipStream_t s);                // all of them as one
void clip_scale(char ta, char tb, const ClipMat* v, int count, double limit, const double* part, int parts,
                double* norm, bool scale, hipStream_t s);

// B (m x n) = op(A) where either has 16-bit elements, rounded to nearest even
template <typename Ts, typename Td>
void gecopy16(char uplo, char trans, i64 m, i64 n, const Ts* A, i64 lda, Td* B, i64 ldb, hipStream_t s);

}  // namespace slate_hip
