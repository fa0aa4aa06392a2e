/*
 * bsgdraft_slots.h — C ABI: the verification of bsgdraft.h for a batch in which some sequences take no part, as the
 * calls of bsgdraft.h and bsgserve.h that are given slots leave them out.
 */
#ifndef BSGDRAFT_SLOTS_H
#define BSGDRAFT_SLOTS_H

#include "bsgdraft.h"

#ifdef __cplusplus
extern "C" {
#endif

/* bsg_verify_drafts, where a sequence whose entry of `slots` (int32 [rows], or NULL: none) is below 0 takes no part: none of
 * its rows is looked at, and its answer is that of a sequence without nodes. */
int bsg_verify_drafts_slots(const void* logits, int64_t logits_stride, const void* draft_logits, int64_t draft_stride,
                            int64_t tokens, int64_t vocab, const int32_t* token_ids, const float* uniforms,
                            const int32_t* parents, const int32_t* cu, const int32_t* slots, int32_t rows, int32_t max_new,
                            float temperature, const float* temperatures, int32_t* accepted, int32_t* path,
                            int32_t* out_tokens, int dtype, void* ws, int64_t ws_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* BSGDRAFT_SLOTS_H */
