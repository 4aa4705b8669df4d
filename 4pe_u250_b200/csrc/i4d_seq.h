// i4d_seq.h -- what the operators accept of the arrays that say where the
// tokens of a batch are.  Host and device: the device cannot return an error
// for values that it alone sees, so it skips what these refuse.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define I4D_HD __host__ __device__ __forceinline__
#else
#define I4D_HD inline
#endif

namespace i4d_ops {

constexpr int kMaxTokens = 1 << 30;  // of one sequence, so that a block's end is an int

// Rows [q0, q1) of `tokens`, at most max_q, the last of `len` tokens in a table row of table_blocks blocks.
I4D_HD bool seq_ok(int q0, int q1, int len, int tokens, int max_q, int table_blocks, int block_tokens) {
    return q0 >= 0 && q1 >= q0 && q1 <= tokens && q1 - q0 <= max_q && len >= q1 - q0 &&
           len <= static_cast<int64_t>(table_blocks) * block_tokens && len <= kMaxTokens;
}

I4D_HD bool block_ok(int id, int blocks) { return static_cast<unsigned>(id) < static_cast<unsigned>(blocks); }

// Blocks that the new tokens of one sequence can touch: it has no more of them
// than its call allows, has rows, or can have.
I4D_HD int touched_blocks(int max_q, int tokens, int block_tokens) {
    const int most = max_q < tokens ? max_q : tokens, n = most < kMaxTokens ? most : kMaxTokens;
    return n <= 0 ? 0 : (n - 1 + block_tokens - 1) / block_tokens + 1;
}

// Block j of those that the tokens [first, len) of a sequence lie in, or -1.
// (Blocks are compared, not tokens: the last one's end may pass 32 bits.)
I4D_HD int touched_block(int first, int len, int block_tokens, int j) {
    const int at = first / block_tokens + j;
    return first < len && at <= (len - 1) / block_tokens ? at : -1;
}

// Length of a sequence that eviction reads.
I4D_HD bool length_ok(int len, int max_length) { return len >= 0 && len <= max_length; }

}  // namespace i4d_ops
