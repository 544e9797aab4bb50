// int8_choice.cpp -- which kernel a product in 8-bit integers takes, by its sizes alone.
//
// Every kernel gives the same bits; times go by the shape of a weight, the share of its
// blocks that is stored and the number of tokens.
#include "int8.hpp"

namespace xspmm {
namespace detail {

namespace {

int64_t groups_of(int64_t n, int64_t each) { return (n + each - 1) / each; }

// us of lists, measured at 14336 x 4096, 4096 x 14336 and 2048 x 2048 with 64 to 2048 tokens
// and 5 to 40 % stored (within a tenth): a window's loads, one after the other, and its
// blocks, in rounds of two workgroups a CU, a last one of one.
double lists_us(int weights, int64_t Mb, int64_t Kb, int64_t N, double share)
{
    const int64_t items = groups_of(Mb, kInt8ListRows / weights) * groups_of(N, kInt8ListTokens), rest = items % 512;
    const double full = 2.7 + 7.5 * share, last = rest == 0 ? 0.0 : rest <= 256 ? 1.75 + 5.5 * share : full;
    return 6.0 + (double)groups_of(Kb, kInt8ListColumns) * ((double)(items / 512) * full + last);
}

// us of tiles: a step of four block-columns, whose loads take most of it whatever is stored.
double tiles_us(int weights, int64_t Mb, int64_t Kb, int64_t N, double share)
{
    const int64_t items = groups_of(Mb, kInt8TileRows / weights) * groups_of(N, kInt8TileTokens), rest = items % 512;
    const double full = 0.6 + 0.3 * share, last = rest == 0 ? 0.0 : rest <= 256 ? 0.42 + 0.2 * share : full;
    return 8.0 + (double)groups_of(Kb, kInt8TileColumns) * ((double)(items / 512) * full + last);
}

}  // namespace

// One token, and more where every workgroup's rounding them anew costs less than a launch:
// us with and without, bf16, 16384 x 1024 30 % stored 16 tokens 10.4 and 11.1, 48 tokens 15.7
// and 10.9; gate and up of 14336 x 4096 25 % stored one token 10.0 and 12.6, two 16.9 and
// 13.6; 4096 x 4096 10 % stored four tokens 8.5 and 11.1.
bool int8_rounds_itself(int weights, int64_t M, int64_t K, int64_t N)
{
    const int64_t Mb = (M + 15) / 16, Kb = (K + 15) / 16;
    if (N == 1) return Kb <= 2 * kInt8FewPieces;
    const int64_t tokens = N < kInt8FewTokens ? N : kInt8FewTokens;
    return Kb * tokens <= kInt8FewPieces && weights * Mb * groups_of(N, kInt8FewTokens) <= 1024;
}

Int8Choice int8_choice(int weights, int64_t M, int64_t K, const int64_t* blocks, int64_t N, bool rounds)
{
    const int64_t Mb = (M + 15) / 16, Kb = (K + 15) / 16, all = blocks[0] + (weights == 2 ? blocks[1] : 0);
    if (rounds) {
        // Sixteen waves to a block-row while there are no more than two workgroups a CU
        // (16 waves each), half and a quarter of them beyond (us of one and two rows a
        // workgroup: fp16 4096 x 14336, 25 % stored, one token 6.7 and 7.8; bf16 gate and
        // up of 14336 x 4096 13.0 and 10.1, of four rows 10.3).
        const int64_t groups = Mb * groups_of(N, kInt8FewTokens);
        return {Int8Kernel::kFew, groups <= 512 ? 1 : groups <= 1024 ? 2 : 4, N > 1 || Kb <= kInt8FewPieces ? 1 : 2};
    }
    // Lists and tiles look their blocks up in a map of the grid, and load them, and their
    // windows of x, by offsets of 31 bits.
    bool windows = N <= (1 << 21);
    for (int l = 0; l < weights; ++l)
        windows = windows && has_block_map(Mb, Kb, blocks[l]) && narrow_bytes(blocks[l], 256, 1) >= 0;
    if (windows) {
        // The walk by blocks, whose x comes through L1, and results: 14336 x 4096 and 2048
        // tokens 48 us at 5 % stored, 117 at 25 %, 370 with all.  The others have a chain of
        // loads for every window of x: they pay where there are tokens enough, lists up to
        // some 45 % stored (90 us at 40 %, tiles 103), tiles from there on (119; lists
        // of 4096 x 14336 114 at 40 %, tiles 118).
        const double share = (double)all / ((double)weights * (double)Mb * (double)Kb);
        const double walk = 5.0 + 7.4e-7 * (double)all * (double)N + 7e-7 * (double)weights * (double)M * (double)N;
        const double lists = lists_us(weights, Mb, Kb, N, share), tiles = tiles_us(weights, Mb, Kb, N, share);
        // so that four times as many blocks are more than a row has in most windows
        if (lists < walk && lists <= tiles) return {Int8Kernel::kLists, share < 0.06 ? 1 : share < 0.15 ? 2 : 3, 0};
        if (tiles < walk) return {Int8Kernel::kTiles, 0, 0};
    }
    // us by (tiles of 16 tokens a wave, waves to a block-row):
    //   sizes, stored, tokens              1, 4   1, 16   4, 1   4, 4
    //   14336 x 4096,  3 %, 64              5.7   13.3     7.3    4.6
    //   2048 x 2048,   6 %, 96, gated       3.9    6.2     9.7    4.9
    //   1024 x 1024,  10 %, 300, gated      4.4    8.3     9.7    5.2
    //   4096 x 14336, 20 %, 33             11.1   10.8    18.5    7.1
    //   4096 x 14336, 30 %, 24, gated      21.9   14.4    73.0   22.0
    //   512 x 8192,   80 %, 300            16.4   12.1    55.9   17.2
    //   4096 x 14336, 10 %, 1100, gated   124    152      80.3   65.1
    //   14336 x 4096,  3 %, 2048           93.4  365      42.0   54.4
    //   50000 x 300,   6 %, 24, gated       9.1   28.0     7.1   10.8
    // Four tiles of tokens read a block and its column once for 64, and pay as soon as there
    // are two workgroups of them a CU, with long rows one.  Four waves to a row have a
    // quarter of the chain of loads, and sums to join: they pay until there are waves enough
    // without that, the sooner the shorter the rows.  Where there are few workgroups of
    // one tile, long rows are split over sixteen waves.
    auto waves = [&](int tiles) { return Mb * groups_of(N, 16 * tiles); };
    const int64_t each = Mb > 0 ? all / Mb : 0, four = waves(4), one = waves(1);
    if (N > 16 && (four >= 512 || (each >= 128 && four >= (N > 32 ? 256 : 257))))
        return {Int8Kernel::kWalk, 4, four < 8192 && four < 2048 + 64 * each ? 4 : 1};
    return {Int8Kernel::kWalk, 1, (one <= 512 && each >= 64) || (one <= 1024 && each >= 192) ? 16 : 4};
}

}  // namespace detail
}  // namespace xspmm
