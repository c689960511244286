// Arguments that the vocabulary kernels (vocab.hip) share with their torch
// binding.
#pragma once

#include <hip/hip_runtime.h>

#define VOCAB_MAX_K 256  // top alternatives, or a teacher's entries, per row

#define VOCAB_MAX_TOP_V 524288  // vocabulary, where top alternatives are asked

enum { VOCAB_BF16 = 0, VOCAB_FP16 = 1, VOCAB_FP32 = 2 };

// rows of V logits, contiguous within a row; row r = o * inner + i starts at
// base + o * stride_o + i * stride_i (in elements)
struct VocabRows {
    const void *base;
    long V, stride_o, stride_i;
    int rows, inner, nseg;  // nseg: stretches per row
    unsigned line;          // 127: stretches begin at cache lines; 0: at rows
};

struct VocabLogprobs {
    const long *tokens;  // [rows] or null
    long ignore;
    int K;
    double temperature;
    float *part;  // [rows, nseg, 4] workspace
    void *gmax;   // [rows, nseg, segment / group] of the logits' type:
                  // workspace, where K > 0
    float *logprobs, *entropy, *top_lp;
    long *top_ids;
    float *stat;  // [rows, 4]
};

struct VocabDistill {
    const float *teacher_lp;  // [rows, K]
    const long *ids;          // [rows, K]
    int K, bucket;
    double temperature;
    float *part, *loss, *stat;
    int *entry;  // [rows, K, 2]: id or -1, and its gradient's bits
};

struct VocabGrad {
    const float *stat;  // [rows, 4]
    float c, inv_t;
    const float *d_row;      // of the log probabilities, or of the loss
    const float *d_entropy;  // null where none
    const float *d_top;      // [rows, K], null where none
    const int *entry;        // [rows, K, 2], the teacher's
    const long *ids;         // [rows, K]
    int K;
    const long *tokens;  // [rows] or null
    long ignore;
};
