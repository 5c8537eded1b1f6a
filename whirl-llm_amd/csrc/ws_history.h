// The sequences' token histories on the device (ws_history), and what a call over them reports (WS_ACCEPT_*).
#pragma once

#include <stdint.h>

namespace ws {

// A sequence's text on the device: tokens[base .. base + len) are what the model holds, tokens[base + len] is the token
// that goes in next, behind it the drafts of the running cycle (placed there by history_stage_kernel).
struct HistoryRef {
    int32_t* tokens;        // nullptr: no device history
    uint32_t* len;          // per slot
    uint64_t* n_gen;        // per slot or nullptr: output tokens so far
    const uint32_t* slot;   // per sequence: its slot
    uint32_t cap;           // tokens per slot
};

constexpr uint32_t kAcceptHost = 1u, kAcceptNearTypical = 2u, kAcceptHistoryFull = 4u, kAcceptPathFull = 8u;

}  // namespace ws
