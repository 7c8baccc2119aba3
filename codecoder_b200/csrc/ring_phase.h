// Phases of a ring of mbarriers, one per slot, as plain arithmetic (host and device): use k of the ring takes slot
// k % stages and is that slot's phase k / stages.
#pragma once
#include <cstdint>

namespace bpc {

// the parity to wait for until use k is complete
constexpr uint32_t ring_parity(int k, int stages) { return static_cast<uint32_t>(k / stages) & 1u; }

// the last use of `slot` among the first `issued` ones (slot < issued): the one whose copies may be under way
constexpr int ring_last_use(int issued, int slot, int stages) { return slot + (issued - 1 - slot) / stages * stages; }

}  // namespace bpc
