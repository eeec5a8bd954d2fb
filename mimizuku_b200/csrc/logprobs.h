// The outputs of the log-probability operators (logprobs.cu, linear_logprobs.cu).
#pragma once

namespace mmz {

constexpr int TOP_MAX = 8;  // alternatives of a row

// Row r's target and outputs lie at index r * ld + *col (col null: 0), so that a captured decoding step can move
// along the sequences; an alternative's at that index times `top`. A null output is not written.
struct LogpOut {
    const int* target;
    float *logp, *entropy, *lse;
    int* top_id;
    float* top_logp;
    long ld;
    const int* col;
    int top;
};

// The engine's decoding step: where the outputs' column is `col`, the ids id[0] and id[1] (-1: none) are left out too, as
// they are of the choice of the first token after a prompt.
struct Begin {
    int col = -1, id[2] = {-1, -1};
};

}  // namespace mmz
