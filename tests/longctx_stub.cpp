// Host side of the long-context operators without a GPU: a context whose
// device does not exist, so that a call that passes every check stops at the
// first CUDA call (I4D_ERR_CUDA) and one that does not says why.
#include <cstdarg>
#include <cstdio>

#include "i4d_internal.h"
#include "i4d_seq.h"

namespace {
char g_message[512];
}

namespace i4d_ops {
OpContext op_context(const i4d_ctx*) { return {-1, 148, nullptr, nullptr}; }
i4d_status op_fail(i4d_ctx*, i4d_status st, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(g_message, sizeof(g_message), fmt, ap);
    va_end(ap);
    return st;
}
}  // namespace i4d_ops

extern "C" {
const char* stub_message() { return g_message; }
int stub_seq_ok(int q0, int q1, int len, int tokens, int max_q, int table_blocks, int block_tokens) {
    return i4d_ops::seq_ok(q0, q1, len, tokens, max_q, table_blocks, block_tokens);
}
int stub_block_ok(int id, int blocks) { return i4d_ops::block_ok(id, blocks); }
int stub_length_ok(int len, int max_length) { return i4d_ops::length_ok(len, max_length); }
}
