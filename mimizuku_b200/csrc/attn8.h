// The arguments of the attention over the 8-bit key/value cache (attn8.cu).
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

namespace mmz {

struct Attn8 {
    const __half* q;             // [batch][rows][q_heads][64], strides in values
    long q_seq, q_row, q_head;
    const uint8_t *k8, *v8;      // [batch][kv_heads][cap][64] codes, strides in bytes
    const float *ks, *vs;        // [batch][kv_heads][ceil(cap / block)] scales
    long c_seq, c_head, s_seq, s_head;
    const int* lens;             // [batch], null: cap
    __half* out;                 // as q
    long o_seq, o_row, o_head;
    __half* probs;               // [batch][slots][rows][cap], null: none
    const int* pslot;            // [q_heads] slot of a head's probabilities, -1: none
    int batch, rows, q_heads, kv_heads, cap, block, causal, slots;
    float scale;
    // the engine's decoding step: finished sequences (done[b] != 0) count as empty and their probabilities are left as
    // they are; a sequence's probabilities lie at p_seq * b + p_step * *pctr (null: 0)
    const int* done = nullptr;
    long p_seq = 0, p_step = 0;
    const int* pctr = nullptr;
};

}  // namespace mmz
