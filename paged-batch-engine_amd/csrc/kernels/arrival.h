// Arrival tickets of workgroups that each finish a part of one result: the last
// to arrive combines the parts. Words in a workspace that may hold anything.
#pragma once
#include "decode_device.h"

namespace pbe {
namespace {

// Arrival tickets. A word holds tag << kTicketBits | arrivals of launch `tag`;
// anything else in it (a workspace may hold anything) counts as none. The last
// arrival leaves 0, so a replayed launch, which has the same tag, starts anew.
constexpr int kTicketBits = 11;
// Makes a word that is 0 ready for arrivals; nothing waits for it.
__device__ __forceinline__ void open_ticket(gptr<uint64_t> word, uint64_t tag) {
  uint64_t none = 0;
  (void)__hip_atomic_compare_exchange_strong(word, &none, tag << kTicketBits, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                             __HIP_MEMORY_SCOPE_AGENT);
}
// Whether this is the last of `members` arrivals: one round trip where the
// word was opened; a word that held something else is claimed by exchange.
__device__ __forceinline__ bool last_arrival(gptr<uint64_t> word, uint64_t tag, uint32_t members) {
  uint64_t now = __hip_atomic_fetch_add(word, (uint64_t)1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
  if ((now >> kTicketBits) != tag) {
    uint64_t seen = now;
    do {
      now = (seen >> kTicketBits) == tag ? seen + 1 : (tag << kTicketBits) | 1u;
    } while (!__hip_atomic_compare_exchange_strong(word, &seen, now, __ATOMIC_RELAXED, __ATOMIC_RELAXED,
                                                   __HIP_MEMORY_SCOPE_AGENT));
  }
  if ((now & ((1u << kTicketBits) - 1)) != members) return false;
  __hip_atomic_store(word, (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return true;
}

}  // namespace
}  // namespace pbe
