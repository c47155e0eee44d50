// Where the loads of the loss's matrix products read (MatPath), gone through on the host for every tile size and layout: each
// load lies inside its operand or is refused by the range check, which sees a lane's register and nothing else, and
// what is inside arrives once; of rows that lie as a caller has them nothing behind a row's end is read.
#include "../../butterfly_amd/csrc/matmul.hpp"

#include <cstdio>
#include <vector>

using namespace bf;

static int failures = 0;

static void fail(const char *what, int size, int waves, int64_t rows, int64_t cols, int64_t stride, int first, int64_t step)
{
    if (++failures < 20)
        printf("%s: %d by %d wavefronts, %lld x %lld stride %lld, first %d, step %lld\n", what, size, waves, (long long)rows,
               (long long)cols, (long long)stride, first, (long long)step);
}

// An operand of rows x cols 16-bit elements, its last row cut behind cols; rows and cols from (first, step) on.
template <MatLayout LAYOUT, int SIZE, bool SPREAD, int WAVES>
static void walk(int64_t rows, int64_t cols, int64_t stride)
{
    using Path = MatPath<LAYOUT, SIZE, SPREAD, WAVES>;
    MatOperand o = {nullptr, 0, stride * 2, ((rows - 1) * stride + cols) * 2, cols % kMatK ? (int)(cols % kMatK) * 2 : kWholeTail};
    // the row and 16-byte unit of its tile that a load brings, from rows that are far apart
    constexpr int per = LAYOUT == kRows ? 8 : SIZE / 8, far = 1 << 21;
    std::vector<int> place(64 * WAVES * Path::kLoads);
    for (int t = 0; t < 64 * WAVES; ++t) {
        Path p;
        int all;
        p.init(far, t / 64, t % 64);
        p.start({nullptr, 0, far, (int64_t)1 << 40, kWholeTail}, 0, 0, false, all);
        for (int j = 0; j < Path::kLoads; ++j) place[t * Path::kLoads + j] = p.offset(j) / far * per + p.offset(j) % far / 16;
    }
    const int64_t m = LAYOUT == kRows ? rows : cols, k = LAYOUT == kRows ? cols : rows, steps = (k + kMatK - 1) / kMatK;
    for (int first = 0; first < m; first += SIZE) {
        for (int64_t from = 0; from < steps; from += 3) {
            // the base moves at `from`; two steps behind the operand's end, and loads of nothing
            for (int nothing = 0; nothing < 2; ++nothing) {
                std::vector<Path> lanes(64 * WAVES);
                std::vector<int> left(64 * WAVES);
                int64_t skip = 0;
                for (int t = 0; t < 64 * WAVES; ++t) {
                    lanes[t].init(o.stride, t / 64, t % 64);
                    skip = lanes[t].start(o, first, from, nothing, left[t]);
                }
                for (int64_t step = from; step < steps + 2; ++step) {
                    std::vector<int> seen(SIZE * 8);
                    if (step == steps - 1)
                        for (int t = 0; t < 64 * WAVES; ++t) lanes[t].cut(o, t % 64);
                    for (int t = 0; t < 64 * WAVES; ++t) {
                        for (int j = 0; j < Path::kLoads; ++j) {
                            const int64_t sum = (int64_t)lanes[t].lane_offset[Path::variant(j)] + lanes[t].load_offset[j];
                            const int at = lanes[t].offset(j);
                            const bool cut = lanes[t].lane_offset[Path::variant(j)] < 0;
                            if (sum != at || (at < 0 && !cut)) fail("offset", SIZE, WAVES, rows, cols, stride, first, step);
                            if ((unsigned)at + 16 > (unsigned)left[t]) continue;   // refused: zeros
                            const int64_t byte = skip + at;
                            if (nothing || byte < 0 || byte + 16 > o.bytes) fail("outside", SIZE, WAVES, rows, cols, stride, first, step);
                            const int i = place[t * Path::kLoads + j];
                            const int64_t row = i / per + (LAYOUT == kRows ? first : step * kMatK);
                            const int64_t unit = i % per + (LAYOUT == kRows ? step * 8 : first / 8);
                            if (byte != row * o.stride + unit * 16) fail("elsewhere", SIZE, WAVES, rows, cols, stride, first, step);
                            if (LAYOUT == kRows && step < steps && unit * 8 >= cols) fail("behind a row", SIZE, WAVES, rows, cols, stride, first, step);
                            ++seen[i];
                        }
                        lanes[t].advance();
                    }
                    if (nothing) continue;
                    for (int i = 0; i < SIZE * 8; ++i) {
                        const int64_t row = i / per + (LAYOUT == kRows ? first : step * kMatK);
                        const int64_t col = 8 * (i % per + (LAYOUT == kRows ? step * 8 : first / 8));
                        if (row < rows && col < cols && seen[i] != 1) fail("not once", SIZE, WAVES, rows, cols, stride, first, step);
                    }
                }
            }
        }
    }
}

template <int SIZE, int WAVES>
static void walk_all(int64_t rows, int64_t cols, int64_t stride)
{
    walk<kRows, SIZE, true, WAVES>(rows, cols, stride);
    walk<kRows, SIZE, false, WAVES>(rows, cols, stride);
    walk<kCols, SIZE, false, WAVES>(rows, cols, stride);
}

int main()
{
    for (int64_t rows : {1, 63, 64, 65, 127, 129, 200, 256, 300, 515})
        for (int64_t cols : {8, 40, 64, 72, 200, 264, 520})
            for (int64_t gap : {0, 8, 96}) {
                walk_all<256, 8>(rows, cols, cols + gap);
                walk_all<128, 4>(rows, cols, cols + gap);
                walk_all<128, 8>(rows, cols, cols + gap);
            }
    // rows far apart: the base moves every few steps of a kCols operand, and no offset passes 2^31
    walk_all<256, 8>(300, 264, 1 << 20);
    walk_all<128, 4>(300, 264, 1 << 20);
    if (failures == 0) printf("all loads ok\n");
    return failures != 0;
}
