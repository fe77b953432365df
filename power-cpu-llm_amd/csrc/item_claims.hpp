// Which items of a launch a workgroup takes: the rule alone, over counters in memory
// that `add` counts up (returning the count before) and `read` looks at.
//
// Items lie in rounds of one for every workgroup of the grid; an XCD has the
// workgroups of its turn, and of every round the items of its part, side by side. Each
// part has a counter of the items taken of it.
#pragma once

#include <cstdint>

namespace pcl {

constexpr uint32_t kItemParts = 8; // XCDs

struct ItemClaims {
    uint32_t items, grid;
    uint32_t each; // items of a part in a round
    bool others;   // whether workgroups go on to other parts' items behind their own

    // The place of item n of a part.
    constexpr uint32_t place(uint32_t of, uint32_t n) const
    {
        return n / each * grid + of * each + n % each;
    }

    // Item n, taken from `part`, or where that is past the last one an item of the
    // first part behind it that has one left, from which the workgroup then goes on
    // taking: those that run out of items at the end spread over the others, and no
    // counter is counted up in vain but where two come for the last item.
    template <typename Read, typename Add>
    constexpr uint32_t settle(uint32_t n, uint32_t &part, Read read, Add add) const
    {
        if (n < items || !others)
            return n;
        const uint32_t mine = part;
        uint32_t taken[kItemParts - 1] = {};
#pragma unroll
        for (uint32_t i = 0; i < kItemParts - 1; ++i)
            taken[i] = read((mine + 1 + i) % kItemParts);
#pragma unroll
        for (uint32_t i = 0; i < kItemParts - 1; ++i) {
            const uint32_t of = (mine + 1 + i) % kItemParts;
            if (n < items || place(of, taken[i]) >= items)
                continue;
            n = place(of, add(of));
            part = n < items ? of : part;
        }
        return n;
    }
};

} // namespace pcl
