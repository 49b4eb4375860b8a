// Selective scan: how threads and channels, tokens and states belong together, and where in a tile a thread reads.  Plain numbers, which hold on the host as on
// the device.
#pragma once

#include <stdint.h>

#include <type_traits>

constexpr int kScanTile = 32;      // tokens
constexpr int kScanThreads = 256;

// An offset that is no tensor's: windows of the tensors are 2^31 - 1 bytes, and a read past their end is a zero, a write is none.
constexpr uint32_t kNowhere = 0x80000000u;

// Channels have L lanes of S states each.
template <int L, int S>
struct scan_form {
    static constexpr int THREADS = kScanThreads, CH = THREADS / L, WAVES = THREADS / 64, NP = L * S;
    static constexpr int ROWS = THREADS / CH, EACH = kScanTile / ROWS;      // tokens at once, and of a thread, where threads lie along the channels
    static constexpr int SHARED = (kScanTile * NP + THREADS - 1) / THREADS;      // values of B of a thread
    static constexpr int BC = THREADS / NP;      // tokens of B at once

    // Along the channels: thread t has channel channel(t) of the tokens row(t), row(t) + ROWS and so on.
    static constexpr int channel(int thread) { return thread % CH; }
    static constexpr int row(int thread) { return thread / CH; }
    // B and C: thread t has state shared_state(t) of the tokens shared_token(t), shared_token(t) + BC and so on.
    static constexpr int shared_state(int thread) { return thread % NP; }
    static constexpr int shared_token(int thread) { return thread / NP; }

    // Where a thread's first value lies, in bytes from where the workgroup's channels (the group's states) of the tile's first token begin: values of `size` bytes,
    // tokens `token` bytes apart.  Up to four states have more threads than a tile has values: the others read nowhere, not the tokens after it, which may be
    // past the tensor.
    static constexpr uint32_t channel_offset(int thread, bool there, uint32_t size, uint32_t token) {
        return ((uint32_t)channel(thread) * size | (there ? 0u : kNowhere)) + (uint32_t)row(thread) * token;
    }
    static constexpr uint32_t shared_offset(int thread, int states, uint32_t size, uint32_t token) {
        const bool there = shared_state(thread) < states && shared_token(thread) < kScanTile;
        return there ? (uint32_t)shared_state(thread) * size + (uint32_t)shared_token(thread) * token : kNowhere;
    }
};

// Lanes of a channel and states of a lane for more than 8 states.
template <class F>
void with_many_states(int N, F launch) {
    using std::integral_constant;
    if (N <= 16) launch(integral_constant<int, 4>(), integral_constant<int, 4>());
    else if (N <= 32) launch(integral_constant<int, 8>(), integral_constant<int, 4>());
    else launch(integral_constant<int, 16>(), integral_constant<int, 4>());
}

// Of tiles: four lanes at least, so that a thread has few tokens along the channels.  4 states, bf16, 22 x 4031 tokens of 192 channels 102 us with four lanes, 108 with
// two and 192 with one; 2 x 157 of 196 23.1, 31.0 and 54.3; 8 states, 2 x 14926 of 2432 444 with four and 434 with two, 8 x 2048 of 1024 107 and 116.
template <class F>
void with_lanes(int N, F launch) {
    using std::integral_constant;
    if (N <= 4) launch(integral_constant<int, 4>(), integral_constant<int, 1>());
    else if (N <= 8) launch(integral_constant<int, 4>(), integral_constant<int, 2>());
    else with_many_states(N, launch);
}

// Of single tokens: whole accesses of states.
template <class F>
void with_step_lanes(int N, F launch) {
    using std::integral_constant;
    if (N <= 4) launch(integral_constant<int, 1>(), integral_constant<int, 4>());
    else if (N <= 8) launch(integral_constant<int, 2>(), integral_constant<int, 4>());
    else with_many_states(N, launch);
}

static inline int fc_scan_channels(int N) {      // of a workgroup
    int channels = 0;
    with_lanes(N, [&](auto lanes, auto) { channels = kScanThreads / decltype(lanes)::value; });
    return channels;
}
