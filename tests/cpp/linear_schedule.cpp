// The steps that linear attention's kernels make between their products (csrc/linscan.h) are
// each made once, in order and inside their arrays, whatever the numbers. Compiled only.
#include "linscan.h"

using namespace snhip;

constexpr bool each_once(int all, int steps) {
    int made = 0;
    for (int m = 0; m < all; m++)
        if (lin_due(m, all, steps)) {
            if (lin_step_at(m, all, steps) != made) return false;
            made++;
        }
    return made == steps;
}
constexpr bool all_once(int all) {
    for (int steps = 1; steps <= all; steps++)
        if (!each_once(all, steps)) return false;
    return true;
}

// Products of a step (plane pairs, row tiles, column tiles) and the pairs of values to make for
// each column tile.
static_assert(each_once(3 * 4 * 1, 4) && each_once(3 * 4 * 2, 8), "one plane");
static_assert(each_once(5 * 2 * 1, 4) && each_once(5 * 2 * 2, 8), "two planes: the numbers do not divide");
static_assert(each_once(6 * 2 * 1, 4) && each_once(6 * 2 * 2, 8), "three planes");
static_assert(each_once(3 * 8 * 2, 8) && each_once(5 * 8 * 2, 8) && each_once(6 * 8 * 2, 8), "the state's products");
static_assert(all_once(7) && all_once(24) && all_once(61), "others");
