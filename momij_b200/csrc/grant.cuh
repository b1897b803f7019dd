// grant.cuh -- a limit of a kernel that calls raise to what they need, from any
// host thread (host only, no CUDA in it).
#pragma once

#include <mutex>

namespace momij {

// Makes `granted` at least `size` by set(size), which says whether it took; the
// check, the setting and the record are one step under a lock, so that the limit
// never falls behind what `granted` says.
template <typename Set>
bool grant_at_least(int& granted, int size, Set&& set) {
    if (__atomic_load_n(&granted, __ATOMIC_ACQUIRE) >= size) return true;
    static std::mutex mu;
    std::lock_guard<std::mutex> hold(mu);
    if (granted >= size) return true;
    if (!set(size)) return false;
    __atomic_store_n(&granted, size, __ATOMIC_RELEASE);
    return true;
}

}  // namespace momij
