// Where a label's blocks of 32 dims stand in MX4 codes and scales (mx4.hpp), as arithmetic on label, block and width: the kernels take it from here,
// and tests/test_label_layout.py goes through it on the host.  Plain C++, nothing of the GPU.
#pragma once
#include <stdint.h>

namespace xfc {

constexpr int MX_BLOCK = 32, MX_UNIT = 64, MX_STEP = 128;  // dims of a block, labels of a unit, dims of a step
constexpr int MX_TILES = MX_UNIT / 16;

constexpr int mx_blocks(int64_t d) { return (int)((d + MX_BLOCK - 1) / MX_BLOCK); }
constexpr int mx_steps(int64_t d) { return (int)((d + MX_STEP - 1) / MX_STEP); }
// bytes of a unit
constexpr int64_t mx_code_bytes(int64_t d) { return (int64_t)MX_UNIT * MX_BLOCK / 2 * mx_blocks(d); }
constexpr int64_t mx_scale_bytes(int64_t d) { return (int64_t)MX_UNIT * 4 * mx_steps(d); }
// ... before a step: they pass 32 bits from 2^26 and 2^30 dims on
constexpr int64_t mx_step_codes(int step) { return (int64_t)step * 4096; }
constexpr int64_t mx_step_scales(int step) { return (int64_t)step * 256; }
// blocks of a step: four, fewer in the last one
constexpr int mx_wide(int step, int blocks) { return blocks - 4 * step < 4 ? blocks - 4 * step : 4; }

// The label of a unit that row i of tile t is, and back.
constexpr int mx_label(int t, int i) { return 32 * (t >> 1) + 8 * (i >> 2) + 4 * (t & 1) + (i & 3); }
constexpr int mx_tile(int label) { return 2 * (label >> 5) + ((label >> 2) & 1); }
constexpr int mx_row(int label) { return 4 * ((label >> 3) & 3) + (label & 3); }

// Where in its unit a label's block stands: codes (16 bytes), scale.  For up to 2^26 dims, more than any call of those that use it takes.
constexpr int mx_code_at(int tile, int row, int block, int blocks) {
  return (int)mx_step_codes(block >> 2) + ((tile * 16 + row) * mx_wide(block >> 2, blocks) + (block & 3)) * 16;
}
constexpr int mx_scale_at(int tile, int row, int block) { return (int)mx_step_scales(block >> 2) + (block & 3) * 64 + row * 4 + tile; }

}  // namespace xfc
