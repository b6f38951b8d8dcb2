// Host-only checks of how the layer products deal their tiles (compiled here for the CPU).
#include <cstdio>
#include <cstring>
#include <vector>

#include "kernel/product_cut.hpp"

using namespace rocm_wmma_gemm::device;

static int fail(const char* what, int tiles, int workgroups, int most, int rows, int slice)
{
    std::printf("FAIL: %s: %d tiles, %d workgroups, K up to %d, %d rows, slice %d\n", what, tiles, workgroups, most, rows,
                slice);
    return 1;
}

// The slices of a launch whose sums have `rows` terms, of at most `most`: each has a K tile, none ends
// behind the last, and together they are all of them.  A kernel's loads move on by K tiles until a slice's
// count is used up, so one without a K tile would run past its operands.
static int check_slices(product_kind kind, int tiles, int workgroups, int most, int rows)
{
    constexpr int  bk  = 64;
    const tail_cut cut = cut_tail(tiles, workgroups, summed_tiles(kind, most, rows, bk), true);
    if(cut.whole + cut.cut != tiles)
        return fail("tiles lost", tiles, workgroups, most, rows, -1);
    if(cut.cut == 0)
        return cut.slices == 1 ? 0 : fail("slices of nothing", tiles, workgroups, most, rows, -1);
    if(cut.cut * cut.slices > workgroups)
        return fail("more slices than room for their parts", tiles, workgroups, most, rows, -1);
    const int k       = kind == product_kind::sum ? rows : most;
    const int k_tiles = k > bk ? (k + bk - 1) / bk : 1;
    int       at      = 0;
    for(int s = 0; s < cut.slices; ++s)
    {
        const tile_run run = run_of_slice(cut, s, k_tiles);
        if(run.count < 1 || run.from != at || run.from + run.count > k_tiles)
            return fail("a slice outside the sum", tiles, workgroups, most, rows, s);
        at += run.count;
    }
    return at == k_tiles ? 0 : fail("K tiles lost", tiles, workgroups, most, rows, cut.slices);
}

static int check_cuts()
{
    const int workgroups[] = {1, 2, 8, 64, 256, 512};
    const int most[]       = {1, 63, 64, 65, 256, 512, 777, 1024, 3904, 4099, 16384};
    for(int w : workgroups)
        for(int tiles = 0; tiles <= 2 * w + 3; tiles += tiles < 40 ? 1 : 17)
            for(int m : most)
            {
                if(check_slices(product_kind::rows, tiles, w, m, 0) || check_slices(product_kind::batch, tiles, w, m, 0))
                    return 1;
                for(int rows = 0; rows <= m; rows += rows < 130 || m - rows < 130 ? 1 : 61)
                    if(check_slices(product_kind::sum, tiles, w, m, rows))
                        return 1;
            }
    return 0;
}

// A symmetric product of g x g tiles: every tile of the square is written once, by itself or as the mirror of
// the one above the diagonal.
static int check_triangle()
{
    for(int g = 1; g <= 60; ++g)
    {
        std::vector<int> written(g * g, 0);
        for(int local = 0; local < g * (g + 1) / 2; ++local)
        {
            const tile_coord t = triangle_tile(local, g);
            if(t.m < 0 || t.n < t.m || t.n >= g)
                return fail("a tile outside the triangle", g, t.m, t.n, local, -1);
            ++written[t.m * g + t.n];
            written[t.n * g + t.m] += has_mirror(t.m * 128, t.n * 128);
        }
        for(int i = 0; i < g * g; ++i)
            if(written[i] != 1)
                return fail("a tile not written once", g, i / g, i % g, written[i], -1);
    }
    return 0;
}

int main(int argc, char** argv)
{
    if(argc == 2 && !std::strcmp(argv[1], "cuts"))
        return check_cuts();
    if(argc == 2 && !std::strcmp(argv[1], "triangle"))
        return check_triangle();
    return 2;
}
