// How the tiles of a layer product's launch are dealt to its persistent workgroups: whole tiles round by
// round, and where the last round has tiles for at most half of them, each of those in slices along K that
// another kernel adds up; and which tiles a symmetric product has.  Integer arithmetic alone, so that the host
// can check it.
#ifndef ROCM_WMMA_GEMM_PRODUCT_CUT_HPP
#define ROCM_WMMA_GEMM_PRODUCT_CUT_HPP

#include "tile_map.hpp"

namespace rocm_wmma_gemm
{
namespace device
{

enum class product_kind
{
    batch = 0,
    rows  = 1,
    sum   = 2
};

struct tail_cut
{
    int whole; // tiles before the cut ones
    int cut; // tiles that are cut
    int slices, each; // each of them in `slices` runs of `each` K tiles, the last perhaps shorter
    RWG_HD int positions() const
    {
        return whole + cut * slices;
    }
};

// A slice shorter than this many K tiles costs more to write and add up than it saves.
constexpr int least_slice = 4, most_slices = 16;

RWG_HD inline tail_cut cut_tail(int tiles, int workgroups, int k_tiles, bool may_cut)
{
    const int rest   = tiles % workgroups;
    int       slices = may_cut && rest > 0 ? workgroups / rest : 1;
    slices           = slices < most_slices ? slices : most_slices;
    slices           = slices < k_tiles / least_slice ? slices : k_tiles / least_slice;
    if(slices < 2)
    {
        return {tiles, 0, 1, k_tiles};
    }
    const int each = (k_tiles + slices - 1) / slices;
    return {tiles - rest, rest, (k_tiles + each - 1) / each, each};
}

// K tiles of `bk` that a tile's sum has.  A sum over the rows of a group has as many rows as the group,
// which only the device knows: cut by the most it can have, K, it would leave slices behind its end.
RWG_HD inline int summed_tiles(product_kind kind, int K, int group_rows, int bk)
{
    const int k = kind == product_kind::sum ? group_rows : K;
    return k > 0 ? (k - 1) / bk + 1 : 0;
}

// The run of K tiles of slice `slice`, of `k_tiles` (at least one).
struct tile_run
{
    int from, count;
};

RWG_HD inline tile_run run_of_slice(const tail_cut& cut, int slice, int k_tiles)
{
    const int from = slice * cut.each;
    return {from, k_tiles - from < cut.each ? k_tiles - from : cut.each};
}

// Tile `local` of the tiles on and above the diagonal of g x g: rows r and g - 1 - r of the triangle
// together have g + 1 tiles.
RWG_HD inline tile_coord triangle_tile(int local, int g)
{
    const int r = local / (g + 1), c = local - r * (g + 1), m = c < g - r ? r : g - 1 - r;
    return {m, c < g - r ? r + c : m + c - (g - r)};
}

// Whether a tile of the triangle, corner (row0, col0), is written a second time, transposed, below the
// diagonal.  A tile on the diagonal is not: it holds both halves, and two waves would store each of its
// elements in no order (the matrix cores' sums for (i, j) and (j, i) may differ in their last bits).
RWG_HD inline bool has_mirror(int row0, int col0)
{
    return row0 != col0;
}

} // namespace device
} // namespace rocm_wmma_gemm

#endif // ROCM_WMMA_GEMM_PRODUCT_CUT_HPP
