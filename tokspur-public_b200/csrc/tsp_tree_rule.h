// Which of the two kernels of tsp_tree_attention a call gets. Plain C++: the rule is tested without a GPU.
#pragma once

#include <stdint.h>

namespace tsp {

// Registers a thread that the hand-over between the warpgroups of tree_mma_kernel starts from. __launch_bounds__ caps the count, ptxas may choose another: the
// hand-over would then wait for registers that nobody gives.
constexpr int kTmLaunchRegs = 128;

// Tiles of 128 binary16 rows on the tensor memory's MMAs once more than six narrow tiles would read the cache: 6 sequences over 6000 slots, 48 rows a kv
// head 43 us (these tiles) against 41 (narrow ones), 64 rows 44 against 46; one over 8000 slots, 128 rows 34 against 48. rows: the most that the call allows a
// sequence, times the heads of a group: a batch goes by its widest draft (63 single tokens and one draft of 12 rows x 4 heads over up to 8192 slots 136 us, of 13 rows 382:
// tiles of 128 rows for every single token). registers: that kernel's, as compiled; the narrow tiles serve everything where they do not fit.
constexpr bool wide_tiles(uint32_t head_dim, bool binary16, uint64_t rows, int registers) {
    return head_dim < 256 && binary16 && rows > 48 && registers == kTmLaunchRegs;
}

}  // namespace tsp
