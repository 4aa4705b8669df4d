// i4d_ring.h -- a warp's ring of asynchronous copies, each slot with a barrier
// whose phase ends when its copy has landed.  Host and device: the order of
// copies and waits is tested without a GPU.
#pragma once

#include "i4d_seq.h"

namespace i4d_ops {

struct Ring {
    // Bit s: parity of the next phase of slot s.  Bit 31: a wait ran out;
    // nothing is copied or used any more.
    uint32_t bits = 0;
    I4D_HD uint32_t parity(int slot) const { return bits >> slot & 1; }
    I4D_HD void passed(int slot) { bits ^= 1u << slot; }
    I4D_HD bool gave_up() const { return bits >> 31; }
    I4D_HD void give_up() { bits |= 1u << 31; }
};

// The copies that come before the first wait: those of the first SLOTS - 1 of
// items first, first + step, ... below n.  issue(item, slot) starts one.
template <int SLOTS, typename Issue>
I4D_HD void ring_fill(const Ring& ring, int first, int step, Issue&& issue) {
    if (ring.gave_up()) return;
    for (int k = 0; k < SLOTS - 1; ++k) issue(first + k * step, k);
}

// Uses the items in turn, the slots in turn from 0 on, a copy started into the
// slot of the item used last (after free_slot()) before each wait.
// wait(slot, parity): whether this thread saw the phase end.  use(item, slot,
// landed): false, in all threads alike, if one of them did not.  That ends the
// walk, this one and all later ones, behind a wait each for the copies still
// in flight, so that none is left behind; whether they landed changes nothing.
template <int SLOTS, typename Issue, typename Wait, typename Free, typename Use>
I4D_HD void ring_walk(Ring& ring, int first, int step, int n, Issue&& issue, Wait&& wait, Free&& free_slot, Use&& use) {
    if (ring.gave_up()) return;
    int slot = 0;
    for (int i = first; i < n; i += step) {
        free_slot();
        issue(i + (SLOTS - 1) * step, slot == 0 ? SLOTS - 1 : slot - 1);
        if (!use(i, slot, wait(slot, ring.parity(slot)))) {
            ring.give_up();
            for (int k = 0, s = slot; k < SLOTS && i + k * step < n; ++k, s = s == SLOTS - 1 ? 0 : s + 1) wait(s, ring.parity(s));
            return;
        }
        ring.passed(slot);
        slot = slot == SLOTS - 1 ? 0 : slot + 1;
    }
}

}  // namespace i4d_ops
