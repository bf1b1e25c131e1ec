// What the entry points (token_api.hip) hand to scan.hip: the gated recurrence.
#pragma once

#include "token_common.h"

namespace dcih {

// Where sequences stand among the tokens: kRows one in each row of tokens; kFlat several of one length in each row (the last
// row may have fewer); kPacked one behind the other between offsets.
enum ScanForm { kRows, kFlat, kPacked };

struct ScanArgs {
    const void *x, *gates;             // token t of row b at b * *_row + t * *_step (elements); shared gates: [dim]
    int64_t x_row, x_step, g_row, g_step;
    int64_t rows, length;              // rows of tokens, tokens of a row
    int64_t sequences;
    int64_t each, total;               // (kFlat) tokens of a sequence, tokens of all rows
    int dim;
    ScanForm form;
    bool decay, shared;
    const float* state;                // [sequences][dim], null: zeros
    const void* bounds;                // lengths [sequences], offsets [sequences + 1] (kPacked), or null
    bool wide_bounds;
    void* h;                           // [rows][length][dim]
    float* last;                       // [sequences][dim], null: not asked for
    float* states;                     // the state before each tile, for the gradient; null: not asked for
    // gradient
    const void* dh;                    // [rows][length][dim], null: zeros
    const float* dlast;                // [sequences][dim], null: zeros
    void *dx, *dgates;                 // null: not asked for; contiguous, dgates [dim] where gates are shared
    float* dstate;
    void* work;
};

int64_t scan_state_floats(int64_t rows, int64_t length, int dim, int dtype);
int64_t scan_work_bytes(int64_t rows, int64_t length, int dim, int dtype);       // of either direction, whatever the gates
bool scan_is_short(const ScanArgs& a, int dtype);      // one thread has a channel of a sequence from the first token to the last
int scan(const ScanArgs& a, int dtype, hipStream_t s);
int scan_grad(const ScanArgs& a, int dtype, hipStream_t s);
int scan_copy(const float* from, float* to, int64_t n, hipStream_t s);

}  // namespace dcih
