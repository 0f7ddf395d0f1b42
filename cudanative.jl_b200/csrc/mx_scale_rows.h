// Which rows of B's scale tiles a tile of columns needs.
#pragma once

#ifdef __CUDACC__
#define B200_HOST_DEVICE __host__ __device__
#else
#define B200_HOST_DEVICE
#endif

namespace b200 {

// Scale tiles hold 128 columns, counted from their group's first one; `group_row` is the group's first row of tiles.  A tile of
// `cols` columns from the group's column `col` on takes `count` rows from `first` on: those of its own columns, so that
// no copy reads a row that no group uses, whether or not the buffer of the scales has it.
struct ScaleRows {
    int first, count;
};
B200_HOST_DEVICE inline ScaleRows scale_rows(int group_row, int col, int cols) {
    return {group_row + col / 128, (col % 128 + cols + 127) / 128};
}

}  // namespace b200
