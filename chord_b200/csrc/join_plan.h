// Which parts of a row of paged_attention are joined, where they lie and where the joins go: plain C++, so that a
// host without a GPU can check it too.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define CHORD_JOIN_FN __host__ __device__ __forceinline__
#else
#define CHORD_JOIN_FN inline
#endif

namespace chord {

// Parts of a row that one CTA joins at once: up to kAtOnce of them; more than that by groups of half as many
// neighbours or, where that would leave more than as many groups, of kFan.
constexpr int kAtOnce = 16, kFan = 24;

// Slots of a lot, a part each: of the row that the lot begins inside of, of the one that it ends inside of (the
// former where it lies within one row), and of the join of the group that it is the first of.
enum LotSlot : int32_t { kSlotInside = 0, kSlotFirst = 1, kSlotGroup = 2, kSlots = 3 };

struct PartPlace {
  int32_t lot, slot;
};

// The joins of a row that `lots` lots from first_lot on have parts of.  A lot can be the last of a row and the first
// of the next one, which then both have parts in it.  So a group of a single lot is not joined by itself: its part
// stands where the lot left it, and a lot's group slot and the group field of its lock word are one row's alone.
struct RowJoin {
  int32_t first_lot, lots, fan;  // fan: lots of a group, one where all are joined at once
  CHORD_JOIN_FN RowJoin(int32_t first, int32_t count)
      : first_lot(first), lots(count), fan(count <= kAtOnce ? 1 : count <= kAtOnce * kAtOnce / 4 ? kAtOnce / 2 : kFan) {}
  CHORD_JOIN_FN int32_t groups() const { return (lots + fan - 1) / fan; }
  // The first of the lot's group, counted in the row's lots, and the lots of a group.
  CHORD_JOIN_FN int32_t group_of(int32_t lot) const { return (lot - first_lot) / fan * fan; }
  CHORD_JOIN_FN int32_t group_lots(int32_t begin) const { return lots - begin < fan ? lots - begin : fan; }
  // The j-th part of a group, and the j-th of what the row's last join takes.
  CHORD_JOIN_FN PartPlace part(int32_t begin, int32_t j) const {
    return {first_lot + begin + j, begin + j == 0 ? kSlotFirst : kSlotInside};
  }
  CHORD_JOIN_FN PartPlace joined(int32_t j) const {
    const int32_t begin = j * fan;
    if (group_lots(begin) == 1) return part(begin, 0);
    return {first_lot + begin, kSlotGroup};
  }
};

}  // namespace chord
