// sequences.hpp -- what the operators with a state per sequence share: which
// state a batch entry has and how many of its tokens are there.
#pragma once

#include "common.hpp"

namespace genllm {

// A padded batch over a pool of states.  ids == nullptr: entry b has state b.
// lens == nullptr: every entry has all S tokens.
struct Sequences {
    const int32_t* ids = nullptr;
    const int32_t* lens = nullptr;
    int32_t n_states = 0;
    int32_t S = 0;
};

constexpr int kEntryEmpty = -1;  // no sequence here: nothing is read or written
constexpr int kEntryBad = -2;    // no such state, or that of an earlier entry with tokens: NaN results, no state is touched

// The state of entry b.  Every lane of the wave calls it with the same b; the
// result is uniform.  Two entries with one state would race on it, so that the
// later one is bad.  An entry without tokens leaves its state alone, and so does not
// count: a server's idle rows may keep the ids they had.
__device__ __forceinline__ int entry_state(const Sequences& s, int b) {
    if (!s.ids) return b;
    const int id = s.ids[b];
    if (id < 0) return kEntryEmpty;
    bool bad = id >= s.n_states;
    for (int i = int(threadIdx.x & 63); i < b; i += 64)
        if (s.ids[i] == id && (!s.lens || s.lens[i] > 0)) bad = true;
    return __ballot(bad) != 0 ? kEntryBad : __builtin_amdgcn_readfirstlane(id);
}

__device__ __forceinline__ int entry_len(const Sequences& s, int b) {
    if (!s.lens) return s.S;
    const int n = __builtin_amdgcn_readfirstlane(s.lens[b]);
    return n < 0 ? 0 : n > s.S ? s.S : n;
}

inline bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace genllm
