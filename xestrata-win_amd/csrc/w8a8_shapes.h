// xestrata-win_amd/csrc/w8a8_shapes.h - the shapes of the int8 products' work-groups and the rule that takes one for a call
// (w8a8.hip's launches; plain C++).
#pragma once

#include <cstdint>

namespace xs {

// The kernels' shapes and what a work-group of each costs, in ns: a step of 128 bytes of k `alone`, with up to as many on the
// chip as CUs, `each` for every one of a CU where several share it (0: they do not, and go in rounds), and what is `fixed` beside
// the steps, the start and the outputs.  Fitted to measurements at 48 to 8192 inputs; a step goes by the rows that a shape reads
// (tokens + weights).
struct Shape {
    int tokens, rows;   // of a work-group; GATED: rows / 2 outputs
    int alone, each, fixed;
};
constexpr Shape kShapes[] = {
    {16, 16, 80, 105, 1000},     // w8a8_ring_kernel (GATED: 16 gate and 16 up rows)
    {32, 32, 130, 125, 1200},
    {64, 32, 185, 225, 1600},
    {64, 64, 250, 0, 2700},
    {64, 64, 347, 242, 1100},    // w8a8_tile_kernel
    {64, 128, 384, 0, 2400},
    {128, 128, 600, 530, 2700},
    {128, 256, 1037, 0, 6000},
    {256, 256, 1790, 0, 8500},
};
constexpr int kShapeCount = sizeof kShapes / sizeof kShapes[0];

// The shape that costs a call least: over 240 calls of 18 to 4096 tokens, 128 to 8192 outputs and 48 to 8192 inputs it takes
// 1.016 times the best shape's time in the mean, 1.23 at worst (a 5 us call); over 69 of 24 to 4096 tokens, 512 to 4096 outputs and
// 12288 to 65536 inputs 1.008, 1.15 at worst (a gated 64 x 512 x 65536: 32 x 32 43 us, 16 x 16 38).  E.g. (tokens x outputs x inputs, us: it / another):
// 24 x 2048 x 4096: 16 x 16 5.0 / 32 x 32 7.0; 37 x 2050 x 7168: 32 x 32 8.4 / 64 x 32 10.3; 64 x 8192 x 4096: 64 x 32 12.2 / 32 x
// 32 12.8; 200 x 4096 x 4096: 64 x 64 ring 11.1 / 64 x 32 13.8; 300 x 2594 x 4208: 64 x 64 tile 14.8 / ring 17.0; 512 x 4096 x
// 4096: 64 x 128 17.3 / 64 x 64 18.0; 4096 x 2048 x 256: 128 x 128 9.6 / 128 x 256 10.1; 1024 x 4096 x 4096: 128 x 128 24 / 64 x 64
// 28; 2048 x 4096 x 7168: 128 x 256 55 / 128 x 128 60; 4096 x 8192 x 7168: 256 x 256 190 / 128 x 128 227.
// Up to 16 tokens every work-group reads the same few lines of x and its own weights once, and many small ones keep the most
// of memory's requests in flight: 16 x 16 (1 x 4096 x 4096 5.6 / 32 rows 6.6; 1 x 8192 x 8192 14.3 / 17).
inline int pick_shape(int n_tok, int n_in, int n_out, bool gated) {
    if (n_tok <= 16) return 0;
    int best = -1;
    double least = 0;
    const double steps = (n_in + 127) / 128;
    for (int i = 0; i < kShapeCount; ++i) {
        const Shape& s = kShapes[i];
        const int outputs = !gated ? s.rows : i == 0 ? 16 : s.rows / 2;
        const int64_t n = (int64_t)((n_tok + s.tokens - 1) / s.tokens) * ((n_out + outputs - 1) / outputs);
        const double alone = gated && i == 0 ? 1.5 * s.alone : s.alone, each = gated && i == 0 ? 2.0 * s.each : s.each;
        const double rounds = (double)((n + 255) / 256);
        const double step = !s.each ? rounds * alone : rounds * each > alone ? rounds * each : alone;
        const double cost = steps * step + rounds * s.fixed;
        if (best < 0 || cost < least) best = i, least = cost;
    }
    return best;
}

}  // namespace xs
