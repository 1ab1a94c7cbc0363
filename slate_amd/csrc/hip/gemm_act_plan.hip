// Which kernel, which tile and how many pieces of K a fused product takes: from
// its sizes, types, layouts and alignment alone.
#include "ffn.hpp"

namespace slate_hip {

GemmActPlan gemm_act_plan(int es, int mode, i64 m, i64 n, i64 k, bool akc, bool bkc, bool dma) {
    GemmActPlan p;
    // Up to 16 columns and both operands along k: 4096 x 4096 bf16 times one
    // column 9.2 us against 14.9 us of the tiles with K split (16 columns of
    // 8192 x 2048: 12.0 against 14.6; 33 of 2048 x 8192 would be 29.6 against
    // 19.0).  Below 1024 rows it fills too few CUs.
    if (mode <= GA_GATED && akc && bkc && n <= 16 && m >= 1024) {
        p.tile = -1;
        return p;
    }
    const i64 rows = mode == GA_GATED ? 2 * m : m, pairs = mode == GA_PAIR ? 2 : 1;
    const int steps = (int)((k * es + 127) / 128) * (mode == GA_SUM ? 2 : 1);
    auto tiles = [&](i64 bm, i64 bn) { return ((rows + bm - 1) / bm) * ((n + bn - 1) / bn) * pairs; };
    // A larger tile reads less per flop, a smaller one fills the CUs with
    // several workgroups whose loads and epilogues overlap.  Measured at
    // 2000^3 bf16: 41 us with 64 x 64, 49 us with 128 x 128; at 4096^3 245, 163
    // and 138 us with 256 x 256.  32- and 64-bit products wait for the MFMAs,
    // not for what a larger tile saves: f32 133 us at 2000^3 (128 x 128: 143 in
    // two pieces), 992 at 4096^3 (967 to 1010), f64 290 (350) and 2220 (2720).
    i64 t;
    if (n <= 16) { p.tile = 3; t = tiles(128, 16); }
    else if (es == 2 && dma && k >= 192 && tiles(256, 256) >= 192) { p.tile = 0; t = tiles(256, 256); }
    else if (es == 2 && tiles(128, 128) >= 768) { p.tile = 1; t = tiles(128, 128); }
    else { p.tile = 2; t = tiles(64, 64); }
    // Few tiles: K in pieces of at least 4 steps, up to two workgroups per CU
    // (64 columns, 1024 x 4096 bf16: 13 us in 16 pieces, 20 us in 4).
    const i64 want = p.tile == 3 ? 1024 : 512;
    if (t < want / 2 && steps >= 8) p.splits = (int)std::min<i64>(steps / 4, want / t);
    if (p.splits > 1) {
        p.per_split = (steps + p.splits - 1) / p.splits;
        p.splits = (steps + p.per_split - 1) / p.per_split;
    }
    if (p.splits > 1) {
        p.ldp = (m + 7) / 8 * 8;
        p.bytes = (i64)p.splits * (mode == GA_GATED || mode == GA_PAIR ? 2 : 1) * n * p.ldp * (es == 8 ? 8 : 4);
    }
    return p;
}

}  // namespace slate_hip
