// linear_i8_plan.hpp -- which kernel a product of 8-bit codes takes: host
// arithmetic on its sizes.
#pragma once

#include <stdint.h>

namespace vvli {

enum I8Kind { kI8Stream, kI8Tile };

// A kernel, and what a call of it takes, in us:
//   base + turn * turns + round * rounds * work + fill * blocks / CUs * work + w * (W in MB) + y * (Y in MB) + part * (parts in MB)
// rounds: blocks that a CU gets. Streams: work is what a block copies, in units of
// 1024 copies, turns the chunks that a wave takes one after the other. Tiles: work
// is the steps of a block, turns the rounds.
//
// The numbers are fits (nonnegative, of relative errors, sizes where the kernel is
// near the fastest weighing most) to 365 sizes, M = 1 to 4096 with (N, K) of nine
// projections, W in no cache, before results of more than 128 MiB passed the caches
// (4096 x 9728 x 896: 64.8 by the fit, 55 measured). On the geometric mean, choosing
// by them cost 0.3 % over the fastest kernel here and 1.2 % over that of 126
// measured variants then; 15 % where it cost most (448 x 3584 x 18944: 58 us, in
// parts by 128 x 128 tiles of four stages 51). Sides of 192 fill the CUs where those
// of 128 and 256 leave a third of them idle (us without and with them: 2048 x 4608 x
// 3584 49 and 41, 1536 x 16384 x 2048 72 and 65, 896 x 9728 x 896 20.9 and 18.5, 131
// x 37888 x 3584 48 and 43).
struct I8Kernel {
    I8Kind kind;
    uint8_t r, m, stages, waves;  // stream: tiles of 16 rows of W, groups of 8 of X; tile: 64s of rows of either
    bool split;                   // tile: K in parts
    float base, turn, round, fill, w, y, part;
};
constexpr I8Kernel kI8Kernels[] = {
    {kI8Stream, 1, 1, 2, 8, false, 3.28f, 0.f, 10.8f, 0.607f, 0.0681f, 0.f, 0.f},
    {kI8Stream, 1, 2, 2, 8, false, 3.32f, 0.f, 9.32f, 3.76f, 0.0481f, 0.f, 0.f},
    {kI8Stream, 1, 4, 2, 8, false, 3.13f, 0.561f, 0.f, 1.65f, 0.0355f, 0.f, 0.f},
    {kI8Stream, 1, 6, 2, 8, false, 3.f, 0.856f, 0.f, 0.824f, 0.0326f, 0.f, 0.f},
    {kI8Stream, 2, 1, 2, 4, false, 3.17f, 0.0757f, 11.2f, 0.f, 0.0711f, 0.f, 0.f},
    {kI8Stream, 2, 2, 2, 4, false, 3.09f, 0.0625f, 12.5f, 1.45f, 0.0484f, 0.f, 0.f},
    {kI8Stream, 2, 4, 2, 4, false, 3.12f, 0.0114f, 13.6f, 1.13f, 0.0477f, 0.f, 0.f},
    {kI8Stream, 2, 6, 2, 4, false, 3.79f, 0.f, 11.8f, 2.63f, 0.0542f, 0.f, 0.f},
    {kI8Stream, 2, 8, 1, 8, false, 3.35f, 0.689f, 3.24f, 4.12f, 0.081f, 0.f, 0.f},
    {kI8Tile, 1, 1, 4, 4, false, 3.34f, 0.f, 0.144f, 0.0667f, 0.0843f, 0.168f, 0.f},
    {kI8Tile, 2, 1, 3, 4, false, 1.53f, 1.73f, 0.248f, 0.119f, 0.0851f, 0.0917f, 0.f},
    {kI8Tile, 2, 2, 2, 4, false, 3.59f, 2.36f, 0.126f, 0.343f, 0.0931f, 0.0322f, 0.f},
    {kI8Tile, 2, 2, 4, 4, false, 2.83f, 0.f, 0.395f, 0.157f, 0.109f, 0.183f, 0.f},
    {kI8Tile, 3, 2, 2, 4, false, 2.98f, 0.f, 0.521f, 0.194f, 0.08f, 0.199f, 0.f},
    {kI8Tile, 4, 2, 2, 4, false, 4.06f, 0.f, 0.581f, 0.31f, 0.0694f, 0.192f, 0.f},
    {kI8Tile, 3, 4, 2, 4, false, 3.32f, 1.64f, 0.696f, 0.452f, 0.0435f, 0.19f, 0.f},
    {kI8Tile, 4, 3, 2, 4, false, 2.47f, 1.7f, 0.768f, 0.379f, 0.0577f, 0.19f, 0.f},
    {kI8Tile, 4, 4, 2, 4, false, 3.4f, 2.62f, 0.832f, 0.591f, 0.0438f, 0.192f, 0.f},
    {kI8Tile, 1, 1, 4, 4, true, 5.88f, 0.f, 0.144f, 0.0408f, 0.102f, 0.f, 0.484f},
    {kI8Tile, 2, 2, 2, 4, true, 7.09f, 0.f, 0.275f, 0.258f, 0.094f, 0.241f, 0.192f},
    {kI8Tile, 4, 4, 2, 4, true, 7.04f, 3.19f, 0.63f, 0.899f, 0.0267f, 0.0752f, 0.261f},
};
constexpr uint32_t kI8KernelCount = sizeof(kI8Kernels) / sizeof(kI8Kernels[0]);
constexpr uint32_t kI8Largest = 17;  // tiles of 256 x 256, the fastest a product where they fill the CUs
static_assert(kI8Kernels[kI8Largest].r == 4 && kI8Kernels[kI8Largest].m == 4 && !kI8Kernels[kI8Largest].split, "256 x 256");

constexpr uint32_t kI8MostSplits = 8, kI8SplitCodes = 512, kI8SplitTiles = 128;  // parts of K, codes of a part at least, tiles at most
constexpr uint64_t kI8PartBytes = uint64_t{64} << 20;                           // of all parts together
constexpr uint64_t kI8TileBytes = uint64_t{1} << 30;                            // 256 rows of W, X or Y for a tile kernel

// Bytes of parts that calls of up to M rows may take (it does not fall where M, N or K grow).
inline uint64_t i8_part_bytes(uint64_t M, uint64_t N, uint64_t K) {
    if (M <= 32 || K < 2 * kI8SplitCodes) return 0;
    return M * N >= kI8PartBytes / 4 / kI8MostSplits ? kI8PartBytes : M * N * 4 * kI8MostSplits;
}

struct I8Plan {
    uint32_t kernel, splits;  // of kI8Kernels
    uint64_t blocks;
    uint64_t cut;  // columns of Y of this launch (0: all); a call of the others follows
};

inline uint64_t i8_up(uint64_t n, uint64_t d) { return (n + d - 1) / d; }

// Blocks of a call without a split.
inline uint64_t i8_blocks(const I8Kernel& k, uint64_t M, uint64_t N) {
    return k.kind == kI8Stream ? i8_up(i8_up(N, 16 * k.r), 8) * 8 * i8_up(M, 8 * k.m) : i8_up(N, 64 * k.r) * i8_up(M, 64 * k.m);
}

inline double i8_time(const I8Kernel& k, uint64_t M, uint64_t N, uint64_t K, uint64_t splits, uint32_t cus) {
    const uint64_t steps = i8_up(K, 128);
    const double w = static_cast<double>(N) * K / 1e6, y = 4.0 * M * N / 1e6;
    if (k.kind == kI8Stream) {
        const uint64_t blocks = i8_up(N, 16 * k.r) * i8_up(M, 8 * k.m), copies = 2 * k.r + k.m;
        const uint64_t fit = 160 / (k.waves * k.stages * copies);  // of a CU's LDS
        const double work = static_cast<double>(copies) * steps / 1024.0;
        return k.base + k.turn * i8_up(blocks, cus * (fit ? fit : 1)) * i8_up(steps, k.waves) + k.round * i8_up(blocks, cus) * work +
               k.fill * work * blocks / cus + k.w * w + k.y * y;
    }
    const uint64_t blocks = i8_blocks(k, M, N) * splits, work = i8_up(steps, splits), rounds = i8_up(blocks, cus);
    return k.base + k.turn * rounds + k.round * rounds * work + k.fill * static_cast<double>(blocks) * work / cus + k.w * w + k.y * y +
           k.part * splits * y;
}

// Whether k takes the call at all: streams hold whatever they are given, but are slow from a few groups of X on; tiles are
// for more rows than a stream's group, and their rows have to fit a buffer's 32-bit offsets (ld: of W, X, Y in bytes, the
// largest).
inline bool i8_takes(const I8Kernel& k, uint64_t M, uint64_t N, uint64_t K, uint64_t ld, uint32_t cus) {
    const bool tiles = M > 32 && ld * 256 <= kI8TileBytes;
    if (k.kind == kI8Stream) return M > 32 && !tiles ? k.m == 8 : i8_up(M, 8 * k.m) <= (k.m == 1 ? 4u : 8u) && (k.m == 1 || 4u * k.m < M + 8);
    if (!tiles) return false;
    const uint64_t blocks = i8_blocks(k, M, N);
    if (k.split) return blocks <= kI8SplitTiles && K >= 2 * kI8SplitCodes;
    // 128 x 128: two blocks of a CU where there are as many, else deeper stages.
    return !(k.r == 2 && k.m == 2) || (blocks <= cus) == (k.stages == 4);
}

// The kernel that takes least, and what it takes.
inline I8Plan i8_one(uint64_t M, uint64_t N, uint64_t K, uint64_t ld, uint32_t cus, double& least) {
    I8Plan best{0, 1, 0, 0};
    for (uint32_t i = 0; i < kI8KernelCount; ++i) {
        const I8Kernel& k = kI8Kernels[i];
        if (!i8_takes(k, M, N, K, ld, cus)) continue;
        for (uint64_t s = k.split ? 2 : 1; s <= (k.split ? kI8MostSplits : 1); ++s) {
            if (k.split && (K < s * kI8SplitCodes || s * M * N * 4 > kI8PartBytes)) break;
            const double t = i8_time(k, M, N, K, s, cus);
            if (best.blocks == 0 || t < least) least = t, best = I8Plan{i, static_cast<uint32_t>(s), i8_blocks(k, M, N) * s, 0};
        }
    }
    return best;
}

// Where 256 x 256 tiles leave a last round that few CUs have a tile of, the whole rounds are a launch of their own and the
// other columns one of smaller tiles (us, all in one launch and so, 256 CUs: 4096 x 4608 x 3584 83 -> 73, 1024 x 37888 x
// 3584 158 -> 145, 4096 x 37888 x 3584 529 -> 516, 4096 x 6144 x 2048 64.7 -> 62.4). The fits' `base` stands for what the
// second launch costs.
inline I8Plan i8_plan(uint64_t M, uint64_t N, uint64_t K, uint64_t ld, uint32_t cus) {
    double least = 0;
    I8Plan best = i8_one(M, N, K, ld, cus, least);
    const I8Kernel& k = kI8Kernels[kI8Largest];
    if (!i8_takes(k, M, N, K, ld, cus)) return best;
    const uint64_t tm = i8_up(M, 64 * k.m), tiles = i8_blocks(k, M, N), first = tiles / cus * cus / tm * 64 * k.r;
    if (tiles <= cus || first == 0 || first >= N) return best;
    double rest = 0;
    i8_one(M, N - first, K, ld, cus, rest);
    if (i8_time(k, M, first, K, 1, cus) + rest < least) best = I8Plan{kI8Largest, 1, first / (64 * k.r) * tm, first};
    return best;
}

constexpr uint64_t kI8MostBlocks = (uint64_t{1} << 32) / 512;  // a launch has fewer than 2^32 threads

// The launches of a call, in order: f(plan, m0, M, n0, N) for the rows m0 .. m0 + M - 1 and columns n0 .. n0 + N - 1 of Y of
// each, until one returns false. A launch with too many blocks is two of half the longer side.
template <typename F>
bool i8_launches(uint64_t M, uint64_t N, uint64_t K, uint64_t ld, uint32_t cus, F& f, uint64_t m0 = 0, uint64_t n0 = 0) {
    const I8Plan plan = i8_plan(M, N, K, ld, cus);
    if (plan.blocks < kI8MostBlocks) {
        if (!plan.cut) return f(plan, m0, M, n0, N);
        return f(plan, m0, M, n0, plan.cut) && i8_launches(M, N - plan.cut, K, ld, cus, f, m0, n0 + plan.cut);
    }
    const uint64_t half = i8_up((M >= N ? M : N) / 2, 256) * 256;
    if (M >= N) return i8_launches(half, N, K, ld, cus, f, m0, n0) && i8_launches(M - half, N, K, ld, cus, f, m0 + half, n0);
    return i8_launches(M, half, K, ld, cus, f, m0, n0) && i8_launches(M, N - half, K, ld, cus, f, m0, n0 + half);
}

}  // namespace vvli
