// Which kernel, which tile and how many pieces of K a fused product takes: from
// its sizes, types, layouts and alignment alone.
#include "ffn.hpp"

namespace slate_hip {

// Laying misaligned 16-bit operands out anew costs a pass over them and two
// launches; the products gain LDS-DMA and with it the larger tiles: 4096^3 144
// against 362 us, 512 x 4096 x 4096 47 against 61, 2000^3 51 against 52; where
// the operands are long for what is computed, or small, it loses: 4096 x 128 x
// 4096 35 against 28 us, 1000^3 20 against 15.
bool gemm_act_pack(int mode, int terms, i64 m, i64 n, i64 k) {
    return (mode == GA_PLAIN ? 1 : mode == GA_SUM ? terms : 2) * m * n * k >= 8000000000 && m * n >= 256 * (m + n);
}

namespace {

// Microseconds that a tile takes, by how many of its workgroups a CU
// holds at once (256 CUs): per step of K (128 bytes), and for its start and
// epilogue; measured on outputs of 256 to 8192 rows and columns, K of 256 to
// 11456.  A larger tile reads less per flop, a smaller one fills the CUs and
// overlaps one workgroup's epilogue with another's products.  bf16: 4096^3 127
// us with 256 x 256 (128: 149, 64: 218), 4096 x 2048 x 4096 71 with 128 x 128
// (101, 97), 4096 x 512 x 4096 31 with 64 x 64 and three slots (256: 95, 128: 52,
// two slots 39), 2048 x 2048 x 4096 51 with two slots (99, 53, three slots 60: a
// CU holds four workgroups of the one, three of the other).  32- and 64-bit
// products wait for the MFMAs, not for what a larger tile would save: 64 x 64
// f32 134 us at 2000^3 (128 x 128: 142 in two pieces), 989 at 4096^3 (966), f64
// 256 (275) and 2020 (1943); 64 x 32 where columns are few or tiles do not fill
// the CUs: f32 32 x 4096 x 4096 20 us (64 x 64: 27), 130 x 1000 x 3000 20 (23),
// 1024^3 26 (30), f64 32 x 4096 x 4096 38 (50); 2000^3 276 (257), f32 440 x 5716 x
// 6329 297 (274).  16-bit operands that go through registers: 1024 x 4096 x 1024
// 31 us, 2048 x 4096 x 512 33 (128 x 128: 39).
enum { HALF_DMA, HALF_REGS, SINGLE, DOUBLE };
struct GaCost { int kind, tile, rows, cols, per_cu; double step[6], ends[6]; };
const GaCost ga_costs[] = {
    {HALF_DMA, 0, 256, 256, 1, {1.72}, {11}},
    {HALF_DMA, 1, 128, 128, 2, {0.70, 0.95}, {4, 7}},
    {HALF_DMA, 2, 64, 64, 4, {0.515, 0.54, 0.60, 0.68}, {1, 2, 3, 3}},
    {HALF_DMA, 4, 64, 64, 3, {0.36, 0.45, 0.60}, {1, 2, 3}},
    {HALF_REGS, 2, 64, 64, 4, {0.55, 0.78, 1.10, 1.50}, {1, 2, 3, 3}},
    {SINGLE, 2, 64, 64, 4, {0.72, 1.10, 1.50, 2.00}, {1, 2, 3, 3}},
    {SINGLE, 5, 64, 32, 6, {0.50, 0.61, 0.88, 1.09, 1.45, 1.75}, {1, 2, 3, 3, 3, 3}},
    {DOUBLE, 2, 64, 64, 4, {0.72, 1.15, 1.50, 2.00}, {1, 2, 3, 3}},
    {DOUBLE, 5, 64, 32, 6, {0.60, 0.68, 0.90, 1.12, 1.45, 1.75}, {1, 2, 3, 3, 3, 3}},
};
double ga_time(const GaCost& c, i64 wgs, int steps) {
    const i64 full = wgs / (256 * c.per_cu), rest = wgs - full * 256 * c.per_cu;
    auto turn = [&](int held, double step) { return steps * step + c.ends[held - 1]; };
    double t = 4 + full * turn(c.per_cu, c.step[c.per_cu - 1]);
    if (rest) {
        const int held = (int)((rest + 255) / 256);
        // (with a fifth of the CUs idle the others' 256 x 256 tiles run faster)
        t += turn(held, c.tile == 0 && rest <= 208 ? 1.45 : c.step[held - 1]);
    }
    return t;
}

}  // namespace

GemmActPlan gemm_act_plan(int es, int mode, int terms, i64 m, i64 n, i64 k, bool akc, bool bkc, bool dma) {
    GemmActPlan p;
    // Up to 16 columns and both operands along k: 4096 x 4096 bf16 times one
    // column 8.6 us against 14.9 us of the tiles with K split (16 columns of
    // 8192 x 2048: 10.6 against 14.6; 33 of 2048 x 8192 would be 29.6 against
    // 19.0).  Below 1024 rows it fills too few CUs; and a CU with two of its
    // workgroups takes twice as long, so that where many have one less than
    // others, rows are long and columns more than a few, K is split instead (15
    // columns: f32 5120 x 5888 32 us against 45, 4096 x 5888 28 against 27; one
    // column: bf16 5120 x 5888 19 against 18).
    const i64 groups = (m + 15) / 16, turns = (groups + 255) / 256 * 256;
    const bool uneven = groups > 256 && 10 * turns >= 13 * groups && n > 8 && k * es >= 8192;
    if (mode <= GA_GATED && akc && bkc && n <= 16 && m >= 1024 && !uneven) {
        p.tile = -1;
        return p;
    }
    const i64 rows = mode == GA_GATED ? 2 * m : m, pairs = mode == GA_PAIR ? 2 : 1;
    const int steps = std::max<int>(1, (int)((k * es + 127) / 128) * terms);
    auto tiles = [&](i64 bm, i64 bn) { return ((rows + bm - 1) / bm) * ((n + bn - 1) / bn) * pairs; };
    if (n > 16) {
        // The tile and the pieces of K (4 steps or more) with the least time by
        // the costs above.  What the operands take from memory bounds them all;
        // partial sums go there and back.
        const int kind = es == 2 ? (dma ? HALF_DMA : HALF_REGS) : es == 4 ? SINGLE : DOUBLE;
        const double outs = 1e-6 * std::max(es, 4) * (mode == GA_GATED || mode == GA_PAIR ? 2 : 1) * m * n;     // MB
        const double mem = es * (double)k * pairs * (rows + n) / 4.4e6;
        double best = 0;
        for (const GaCost& c : ga_costs) {
            if (c.kind != kind) continue;
            const i64 t = tiles(c.rows, c.cols);
            for (int want = 1; want == 1 || (want <= steps / 4 && t * want <= 1024); ++want) {
                const int per = (steps + want - 1) / want, sp = (steps + per - 1) / per;
                if (sp != want) continue;
                const double x = std::max(ga_time(c, t * sp, per), mem) + (sp > 1 ? 2 + 0.45 * outs * sp : 0);
                if (best == 0 || x < best) { best = x; p.tile = c.tile; p.splits = sp; }
            }
        }
    } else {
        // K in pieces of at least 4 steps, up to four workgroups per CU (16
        // columns, 4096 x 4096 bf16: 15 us in 16 pieces, 21 us in 4)
        p.tile = 3;
        const i64 t = tiles(128, 16);
        if (t < 512 && steps >= 8) p.splits = (int)std::min<i64>(steps / 4, 1024 / t);
    }
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
