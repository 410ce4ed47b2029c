// Grids of many blocks (host; no HIP in here, so that their sizes can be checked without a device).
#pragma once

namespace vte {

// A launch's dimension holds fewer than 2^32 threads: `blocks` of up to 1024 of them as x times y, x as a kernel without a
// second dimension would have it while it may be.  y * x may be up to x - 1 more than `blocks`.
struct BlockGrid {
    unsigned x, y;
};
constexpr BlockGrid block_grid(long long blocks) {
    const long long most = 1 << 20, y = (blocks + most - 1) / most;
    return BlockGrid{(unsigned)(y > 1 ? most : blocks), (unsigned)y};
}

// Heads that a block of 256 threads of the norm and rotation of rows takes: two 16-byte runs a thread, or a wave each.
constexpr int qk_norm_heads(bool wide, int head_dim, int size) { return wide ? 8192 / (head_dim * size) : 4; }

}  // namespace vte
