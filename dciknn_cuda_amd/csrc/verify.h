// What the entry points (token_api.hip) hand to verify.hip: drafted tokens against the model's probabilities.
#pragma once

#include "token_common.h"

namespace dcih {

constexpr int kMaxDrafts = 256;

struct VerifyArgs {
    const void* z;                // logits: row i of sequence b at z + (b * (drafts + 1) + i) * stride (elements)
    int64_t n, stride;            // sequences
    int drafts, vocab;
    double c2;                    // log2(e) / temperature
    const void* ids;              // [n][drafts]
    bool wide_ids;
    const float* uniforms;        // [n][drafts + 1]
    const void* slot_ids;         // [n][drafts][slots], null: drafts are named for certain
    bool wide_slots;
    const void* teacher;
    int teacher_dtype, slots;
    int32_t *tokens, *accepted;   // [n][drafts + 1], [n]
    float* logprobs;              // [n][drafts + 1]
    void* work;
};

int64_t verify_work_bytes(int64_t rows, int vocab, int dtype);
int verify(const VerifyArgs& a, int dtype, hipStream_t s);

}  // namespace dcih
