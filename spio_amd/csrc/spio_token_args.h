// Arguments of the kernels over sequences of tokens, as the host hands them over and the device reads them: one structure
// a kernel family, of fields of eight bytes each (kernels/*_kernel.py list them in this order).  A pointer that a
// kernel does not use, or an input that is absent, is null.
#ifndef SPIO_TOKEN_ARGS_H
#define SPIO_TOKEN_ARGS_H

// Rows of u, delta, gate, B and C are `*_row` values apart (all tokens of all sequences follow each other); those of the
// other tensors follow each other without gaps.
struct SpioScanArgs {
    const void *u, *delta, *B, *C, *gate, *dout;  // [sequences][tokens][channels], B and C [sequences][tokens][states]
    const float *A, *D, *bias;                    // [channels][states], [channels], [channels]
    const float* before;                          // [sequences][channels][states]
    void* out;
    float* after;
    float* kept;          // states before every tile of tokens: [sequences][tiles][states][channels]
    float* ends;          // [sequences][chunks][states + 1][channels], the last row the sum of the time steps
    void *du, *ddelta, *dgate;
    float* token_sums;    // [sequences][tokens][blocks of 64 channels][dB, dC]
    float* channel_sums;  // [sequences][chunks][states + 2][channels]: dA, dD, dbias
    void *dB, *dC;
    float *dA, *dD, *dbias;  // [channels][states], [channels], [channels]
    long long tokens, channels, chunk, sequences;
    long long u_row, delta_row, gate_row, b_row, c_row;
};

struct SpioConv1dArgs {
    const void *x, *weight, *bias, *dy;  // [sequences][tokens][channels] (x's rows x_row apart), [channels][width], [channels]
    const void* before;                  // [sequences][width - 1][channels]: the inputs before the first token
    void *out, *after, *dx;
    float* partials;                     // [sequences][slices][width + 1][channels]: dweight, dbias
    float *dweight, *dbias;              // [channels][width], [channels]
    long long tokens, channels, sequences, slice, x_row;
};

// Rows (tokens) of q are q_row, its heads q_head values apart, and so k's; the outputs have no gaps.
struct SpioRotaryArgs {
    const void *q, *k, *dq, *dk;             // [tokens][heads][D]; dq, dk the gradients of the outputs
    const float *q_weight, *k_weight;        // [D]
    const void* positions;                   // [tokens] of a sequence, or of all
    const double* frequencies;               // [pairs]: radians a position
    void *q_out, *k_out;                     // (backward: the gradients of q and k)
    float* partials;                         // [workgroups][2][D]
    float *dq_weight, *dk_weight;            // [D]
    long long tokens, q_heads, k_heads, parts, pairs;
    long long q_row, q_head, k_row, k_head;
    long long position_tokens;               // positions repeat after as many
    long long wide_positions;                // int64, else int32
    double eps, scale;
};

#endif
