// int8_choice.cpp -- which kernel a product in 8-bit integers takes, by its sizes alone.
//
// Every kernel gives the same bits; times go by the shape of a weight, the share of its
// blocks that is stored and the number of tokens.
#include "int8.hpp"

namespace xspmm {
namespace detail {

namespace {

int64_t groups_of(int64_t n, int64_t each) { return (n + each - 1) / each; }

// us of a kernel with x in LDS: `steps` of a workgroup's windows one after the other, in rounds
// of two workgroups a CU, of which the last may be one or less; what is stored adds to a
// step; results in fp32 are written at 3 TB/s more of them.
struct Steps {
    double launch, two[2], one[2];  // of a step: none stored, and what all stored adds
};
double steps_us(const Steps& t, int64_t items, int64_t steps, double share, double more_bytes)
{
    const int64_t rest = items % 512;
    const double two = t.two[0] + t.two[1] * share, one = t.one[0] + t.one[1] * share;
    const double last = rest == 0 ? 0.0 : rest <= 256 ? one : one + (two - one) * (double)(rest - 256) / 256.0;
    return t.launch + (double)steps * ((double)(items / 512) * two + last) + more_bytes * 3e-7;
}

}  // namespace

// One token, and more where every workgroup's rounding them anew costs less than a launch
// and the walk behind it: us with (its fastest) and without, bf16, 14336 x 4096 25 % stored, gate and
// up, one token 9.8 and 11.8, two 13.9 and 13.2, four 13.0 and 14.1; 5 % stored, one
// weight, four tokens 8.7 and 10.2; 16384 x 1024 25 % stored, gate and up, eight tokens 7.2
// and 9.3, sixteen 8.2 and 9.5, 32 11.1 and 11.2, 64 23.5 and 12.5.
bool int8_rounds_itself(int64_t M, int64_t K, int64_t N)
{
    const int64_t Mb = (M + 15) / 16, Kb = (K + 15) / 16;
    if (N == 1) return Kb <= 2 * kInt8FewPieces;
    const int64_t tokens = N < kInt8FewTokens ? N : kInt8FewTokens;
    return Kb * tokens <= kInt8FewPieces && Mb * groups_of(N, kInt8FewTokens) <= 1024;
}

Int8Choice int8_choice(int weights, int64_t M, int64_t K, const int64_t* blocks, int64_t N, int size, bool rounds)
{
    const int64_t Mb = (M + 15) / 16, Kb = (K + 15) / 16, all = blocks[0] + (weights == 2 ? blocks[1] : 0);
    if (rounds) {
        // Sixteen waves to a block-row while there is a workgroup a CU, half of them up to twice
        // that.  Beyond, half or a quarter: by how much the blocks of a row take beside
        // rounding the tokens once more.  us of one, two and four rows a workgroup, bf16:
        //   4096 x 14336,  25 %, 1 token            8.1    8.9   10.4
        //   8192 x 4096,    5 %, 1                  6.8    6.1    6.2
        //   8192 x 4096,    5 %, 4                 12.3    8.7    8.6
        //   14336 x 4096,  25 %, 1, gate and up    14.5    9.7   11.0
        //   14336 x 4096,   5 %, 2                 22.5   13.0    9.5
        //   16384 x 1024,  25 %, 16, gate and up   19.8   11.2    8.4
        //   16384 x 1024,  80 %, 2, gate and up    15.7   10.3   10.3
        //   5000 x 30000,  80 %, 1                 39.1   31.0   49.8
        const int64_t groups = Mb * groups_of(N, kInt8FewTokens), pieces = Kb * (N < kInt8FewTokens ? N : kInt8FewTokens);
        const int rows = groups <= 256 ? 1 : groups <= 512 ? 2 : 4 * all <= (128 + pieces) * Mb ? 4 : 2;
        return {Int8Kernel::kFew, rows, N > 1 || Kb <= kInt8FewPieces ? 1 : 2};
    }
    // Lists and tiles look their blocks up in a map of the grid, and load them, and their
    // windows of x, by offsets of 31 bits.  Few tokens leave most of a workgroup's without work
    // (70000 x 1024, 70 % stored, 31 tokens: walk 17.4 us, lists 26.0, tiles 28.9).
    bool windows = N > 32 && N <= (1 << 21);
    for (int l = 0; l < weights; ++l)
        windows = windows && has_block_map(Mb, Kb, blocks[l]) && narrow_bytes(blocks[l], 256, 1) >= 0;
    if (windows) {
        // Times (us) fitted to 1584 measured products of eight shapes, 2 to 100 % stored, 64 to
        // 2048 tokens, one weight and two, 16 and 32 bits, of a sample in
        // profiles/int8_kernel_choice.txt: within 14 % of them (one standard deviation), and
        // what they choose is 0.4 % slower than the fastest in the mean.  Measured at 14336
        // x 4096, 2048 tokens, bf16:
        //   stored      4 %    10 %   18 %   25 %   35 %   50 %   100 %
        //   walk        45     69     97     126    160    216    378
        //   lists       50     58     62      75     90    110    178
        //   tiles       78     83     91     100    106    111    123
        // The walk goes by blocks, whose x comes through L1, and results; lists and tiles have a
        // chain of loads for every window of x.
        const int64_t rows = groups_of(N, 64) * 64;
        const double share = (double)all / ((double)weights * (double)Mb * (double)Kb);
        const double more = size == 4 ? 2.0 * (double)M * (double)N : 0.0;
        const double walk = 4.5 + 9.8e-7 * (double)all * (double)rows + 9e-7 * (double)weights * (double)M * (double)rows;
        const double lists = steps_us({7.3, {2.65, 8.4}, {1.3, 7.7}},
                                      groups_of(Mb, kInt8ListRows / weights) * groups_of(N, kInt8ListTokens),
                                      groups_of(Kb, kInt8ListColumns), share, more);
        const double tiles = steps_us({11.0, {0.6, 0.47}, {0.41, 0.21}},
                                      groups_of(Mb, kInt8TileRows / weights) * groups_of(N, kInt8TileTokens),
                                      groups_of(Kb, kInt8TileColumns), share, more);
        // Four times as many blocks are more than a row has in most windows (us of one, two
        // and three fours, 14336 x 4096, gate and up, 2048 tokens: 6 % stored 84, 92 and
        // 122, 10 % 96, 97 and 126, 22 % 135, 118 and 135, 40 % 202, 171 and 171; 4096 x
        // 14336 at 30 % 131, 102 and 93).
        if (lists < walk && lists <= tiles) return {Int8Kernel::kLists, share < 0.08 ? 1 : share < 0.26 ? 2 : 3, 0};
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
