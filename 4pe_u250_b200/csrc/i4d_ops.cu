// i4d_ops.cu -- host side of the long-context serving operators (see
// include/i4d.h): checks of arguments, launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <initializer_list>

#include "i4d.h"
#include "i4d_internal.h"
#include "i4d_kv8_attn.cuh"
#include "i4d_kv8_cache.cuh"
#include "i4d_kv8_prompt.cuh"
#include "i4d_logits.cuh"
#include "i4d_rope.cuh"

using namespace i4d_ops;

namespace {

// Takes the error word and leaves zero in one step: what an operator on another
// stream reports meanwhile is either taken or still there for the next call.
__global__ void k_take_errors(unsigned* err, unsigned* taken) { *taken = atomicExch(err, 0u); }

// The context's device for the length of a call; the caller's is put back.
class DeviceScope {
  public:
    explicit DeviceScope(int device) {
        err_ = cudaGetDevice(&before_);
        if (err_ == cudaSuccess && before_ != device) {
            err_ = cudaSetDevice(device);
            changed_ = err_ == cudaSuccess;
        }
    }
    ~DeviceScope() {
        if (changed_) cudaSetDevice(before_);
    }
    cudaError_t error() const { return err_; }

  private:
    int before_ = 0;
    bool changed_ = false;
    cudaError_t err_;
};

#define OP_ARG(cond, ...)                                                \
    do {                                                                 \
        if (!(cond)) return op_fail(ctx, I4D_ERR_ARG, __VA_ARGS__);      \
    } while (0)

#define OP_CK(call)                                                                                  \
    do {                                                                                             \
        const cudaError_t e_ = (call);                                                               \
        if (e_ != cudaSuccess) return op_fail(ctx, I4D_ERR_CUDA, "%s failed: %s", #call, cudaGetErrorString(e_)); \
    } while (0)

int dtype_bytes(int t) { return t == I4D_F32 ? 4 : 2; }
bool is_dtype(int t) { return t == I4D_F32 || t == I4D_BF16 || t == I4D_F16; }
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// The stream of an operator that is about to be enqueued.
cudaStream_t stream_of(const OpContext& o, void* stream) {
    if (o.used) *o.used = true;
    return stream ? static_cast<cudaStream_t>(stream) : o.stream;
}

// Bytes [lo, hi) that `n` rows of `heads` heads touch.
struct Span {
    const char* name;
    uintptr_t lo, hi;
};
Span span_of(const char* name, const void* p, int64_t n, int64_t stride, int64_t heads, int64_t head_stride, int64_t inner, int64_t bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    if (!p || n <= 0 || heads <= 0) return {name, at, at};
    return {name, at, at + static_cast<uintptr_t>(((n - 1) * stride + (heads - 1) * head_stride + inner) * bytes)};
}
Span span_of(const char* name, const void* p, int64_t n, int64_t bytes) { return span_of(name, p, 1, 0, 1, 0, n, bytes); }
bool overlap(const Span& a, const Span& b) { return a.lo < b.hi && b.lo < a.hi; }

// What a call writes must not lie in what else it reads or writes.
i4d_status check_apart(i4d_ctx* ctx, std::initializer_list<Span> writes, std::initializer_list<Span> reads) {
    for (const Span* w = writes.begin(); w != writes.end(); ++w) {
        for (const Span* x = w + 1; x != writes.end(); ++x) OP_ARG(!overlap(*w, *x), "%s overlaps %s", w->name, x->name);
        for (const Span& r : reads) OP_ARG(!overlap(*w, r), "%s overlaps %s", w->name, r.name);
    }
    return I4D_OK;
}

// Rows of heads in one buffer, as [tokens][heads][dim] with strides.
struct View {
    const char* name;
    const void* p;
    int64_t n, stride, heads, head_stride, inner;
    int bytes;
    Span span() const { return span_of(name, p, n, stride, heads, head_stride, inner, bytes); }
    bool same(const View& o) const { return p == o.p && stride == o.stride && head_stride == o.head_stride; }
};

// False where no element of one view is one of the other: apart in memory, or
// parts of one buffer's rows (the q, k and v of a fused projection), which lie
// apart in each period of a stride that all their steps are multiples of.
bool overlap(const View& a, const View& b) {
    if (!overlap(a.span(), b.span())) return false;
    for (const int64_t period : {a.stride, a.head_stride, b.stride, b.head_stride}) {
        if (period <= 0) continue;
        const auto extent = [&](const View& v) {
            return v.inner + (v.stride % period ? (v.n - 1) * v.stride : 0) + (v.head_stride % period ? (v.heads - 1) * v.head_stride : 0);
        };
        const int64_t from = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b.p) - reinterpret_cast<uintptr_t>(a.p)) / a.bytes % period;
        const int64_t delta = from < 0 ? from + period : from;
        if (extent(a) <= delta && delta + extent(b) <= period) return false;
    }
    return true;
}

// Every element has a place of its own.
bool rows_apart(const View& v) {
    if (v.n == 1) return v.heads == 1 || v.head_stride >= v.inner;
    if (v.heads == 1) return v.stride >= v.inner;
    return (v.head_stride >= v.inner && v.stride >= (v.heads - 1) * v.head_stride + v.inner) ||
           (v.stride >= v.inner && v.head_stride >= (v.n - 1) * v.stride + v.inner);
}

int64_t cache_bytes(const i4d_kv8& c) { return static_cast<int64_t>(c.blocks) * c.heads * c.block_tokens * c.dim; }
int64_t cache_scales(const i4d_kv8& c) { return static_cast<int64_t>(c.blocks) * c.heads; }
#define CACHE_SPANS(c)                                                                              \
    span_of("cache k", (c).k, cache_bytes(c), 1), span_of("cache v", (c).v, cache_bytes(c), 1),     \
        span_of("k_scale", (c).k_scale, cache_scales(c), 4), span_of("v_scale", (c).v_scale, cache_scales(c), 4)
#define BATCH_SPANS(a)                                                                              \
    span_of("q_start", (a)->q_start, (a)->batch + 1, 4), span_of("lengths", (a)->lengths, (a)->batch, 4), \
        span_of("block_table", (a)->block_table, (a)->batch, (a)->table_stride, 1, 0, (a)->table_blocks, 4)

i4d_status check_cache(i4d_ctx* ctx, const i4d_kv8& c) {
    OP_ARG(c.k && c.v && c.k_scale && c.v_scale, "null cache buffer");
    OP_ARG(c.blocks > 0 && c.heads > 0, "cache of %d blocks and %d heads", c.blocks, c.heads);
    OP_ARG(c.block_tokens == 16 || c.block_tokens == 32 || c.block_tokens == 64 || c.block_tokens == 128,
           "block_tokens %d (16, 32, 64 or 128)", c.block_tokens);
    OP_ARG(c.dim > 0 && c.dim <= 256 && c.dim % 16 == 0, "dim %d (a multiple of 16 up to 256)", c.dim);
    OP_ARG(c.code == I4D_CODE_INT8 || c.code == I4D_CODE_E4M3, "unknown code %d", c.code);
    OP_ARG(aligned(c.k, 16) && aligned(c.v, 16), "cache codes need 16-byte alignment");
    OP_ARG(aligned(c.k_scale, 4) && aligned(c.v_scale, 4), "cache scales need 4-byte alignment");
    return I4D_OK;
}

Kv8Dev cache_dev(const i4d_kv8& c) {
    Kv8Dev d = {};
    d.codes[0] = static_cast<uint8_t*>(c.k);
    d.codes[1] = static_cast<uint8_t*>(c.v);
    d.scale[0] = c.k_scale;
    d.scale[1] = c.v_scale;
    d.heads = c.heads;
    d.dim = c.dim;
    d.block_tokens = c.block_tokens;
    return d;
}

i4d_status check_batch(i4d_ctx* ctx, const int32_t* q_start, const int32_t* lengths, const int32_t* table,
                       int64_t table_stride, int table_blocks, int batch, int tokens, int max_q) {
    OP_ARG(batch >= 0 && tokens >= 0 && max_q >= 0, "negative batch, tokens or max_q");
    OP_ARG(batch == 0 || (q_start && lengths && table), "null q_start, lengths or block_table");
    OP_ARG(aligned(q_start, 4) && aligned(lengths, 4) && aligned(table, 4), "index arrays need 4-byte alignment");
    OP_ARG(table_blocks >= 0 && table_stride >= 0, "negative table_stride or table_blocks");
    return I4D_OK;
}

SeqArrays seq_arrays(const OpContext& o, const i4d_kv8& c, const int32_t* q_start, const int32_t* lengths,
                     const int32_t* table, int64_t table_stride, int table_blocks, int tokens, int max_q) {
    SeqArrays s = {};
    s.q_start = q_start;
    s.lengths = lengths;
    s.table = table;
    s.table_stride = table_stride;
    s.table_blocks = table_blocks;
    s.tokens = tokens;
    s.max_q = max_q;
    s.block_tokens = c.block_tokens;
    s.blocks = c.blocks;
    s.err = o.err;
    return s;
}

constexpr int64_t kMaxGrid = 0x7fffffff;

// A kernel of the operators, in clusters of `ctas` CTAs.  Each begins with
// op_begin(), which waits for what the stream holds before it, so its launch
// may overlap that one's end.
template <typename... Params, typename... Args>
cudaError_t launch(void (*kernel)(Params...), int64_t grid, unsigned block, size_t smem, int ctas, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(ctas);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctas > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// A kernel with more shared memory than every kernel has.  `allowed`, of that
// kernel alone: the devices where it has been said how much; that is said at
// its first launch, which loads it, and not for the contexts that never call it
// (27 ms of i4d_create).  Saying it is no work for a stream and may happen
// while one is captured.
template <typename... Params, typename... Args>
cudaError_t launch_large(std::atomic<uint64_t>& allowed, int most, void (*kernel)(Params...), int64_t grid, unsigned block, size_t smem, int ctas,
                         cudaStream_t st, Args... args) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (!(allowed.load(std::memory_order_acquire) & bit)) {
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        e = cudaThreadExchangeStreamCaptureMode(&mode);
        if (e != cudaSuccess) return e;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        const cudaError_t back = cudaThreadExchangeStreamCaptureMode(&mode);
        if (e == cudaSuccess) e = back;
        if (e != cudaSuccess) return e;
        allowed.fetch_or(bit, std::memory_order_release);
    }
    return launch(kernel, grid, block, smem, ctas, st, args...);
}

// ------------------------------------------------------------------ rope

template <typename T, int V, bool IL>
cudaError_t launch_rope(const RopeDev& d, int num_sms, cudaStream_t st) {
    const int rot_items = (IL ? d.rot : d.rot / 2) / V;
    const int items = (d.heads[0] + d.heads[1]) * (rot_items + (d.copy_tail ? (d.dim - d.rot) / V : 0));
    // Few tokens: their heads are spread over CTAs, up to two waves of them
    // (40 heads, half rotated: 1200 tokens 12.4 us, 14.2 as many; 2368 16.4 both).
    if (d.tokens >= 16 * num_sms) {
        return launch(k_rope_many<T, V, IL>, (d.tokens + kRopeWarps - 1) / kRopeWarps, 32 * kRopeWarps, 0, 1, st, d);
    }
    const int most = (items + kRopeThreads - 1) / kRopeThreads;
    const int groups = std::max(1, std::min(most, 2 * num_sms / d.tokens));
    return launch(k_rope<T, V, IL>, d.tokens * groups, kRopeThreads, 0, 1, st, d, groups);
}

template <typename T>
cudaError_t launch_rope_t(const RopeDev& d, bool interleaved, bool wide, int num_sms, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    if (interleaved) return wide ? launch_rope<T, V, true>(d, num_sms, st) : launch_rope<T, 2, true>(d, num_sms, st);
    return wide ? launch_rope<T, V, false>(d, num_sms, st) : launch_rope<T, 1, false>(d, num_sms, st);
}

// ---------------------------------------------------------------- append

template <typename T, int V, int CODE>
cudaError_t launch_append(const AppendDev& d, int64_t units, int64_t unit_items, cudaStream_t st) {
    // A warp for the few values of a decode step, a CTA for a block of a prompt.
    if (unit_items <= 64) return launch(k_kv8_append<T, V, CODE, 32>, (units + 3) / 4, 128, 0, 1, st, d, static_cast<int>(units));
    return launch(k_kv8_append<T, V, CODE, 256>, units, 256, 0, 1, st, d, static_cast<int>(units));
}

template <typename T>
cudaError_t launch_append_t(const AppendDev& d, int code, bool wide, int64_t units, int64_t items, cudaStream_t st) {
    if (code == I4D_CODE_INT8)
        return wide ? launch_append<T, 8, I4D_CODE_INT8>(d, units, items, st) : launch_append<T, 1, I4D_CODE_INT8>(d, units, items, st);
    return wide ? launch_append<T, 8, I4D_CODE_E4M3>(d, units, items, st) : launch_append<T, 1, I4D_CODE_E4M3>(d, units, items, st);
}

// ------------------------------------------------------------- attention

// cuTensorMapEncodeTiled of the driver, looked up once (it comes with no
// library that this one links).
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
    static const EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found);
        return e == cudaSuccess && found == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeFn>(p) : nullptr;
    }();
    return fn;
}

// The cache's codes as a matrix of bytes, a row for each (block, head, slot),
// copied in boxes of `rows` rows of 128 bytes (64 for dims up to 64).
i4d_status encode_codes(i4d_ctx* ctx, const i4d_kv8& c, const void* codes, int rows, CUtensorMap* map) {
    const EncodeFn fn = encode_fn();
    if (!fn) return op_fail(ctx, I4D_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    const bool narrow = c.dim <= 64;
    const cuuint64_t size[2] = {static_cast<cuuint64_t>(c.dim), static_cast<cuuint64_t>(c.blocks) * c.heads * c.block_tokens};
    const cuuint64_t stride[1] = {static_cast<cuuint64_t>(c.dim)};
    const cuuint32_t box[2] = {narrow ? 64u : 128u, static_cast<cuuint32_t>(rows)}, step[2] = {1, 1};
    const auto encode = [&] {
        return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  narrow ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = encode();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {  // a thread's first CUDA call: the runtime has bound no context to it yet
        OP_CK(cudaSetDevice(op_context(ctx).device));
        r = encode();
    }
    if (r != CUDA_SUCCESS) return op_fail(ctx, I4D_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    return I4D_OK;
}

struct AttnPlan {
    int dt, nt;  // padded dim, row tiles of eight a CTA
    int row_tiles;
    int64_t segments;  // (sequence, cache head, row tile)
    int even;          // CTAs that share the tokens, or 0
    int cluster;       // else the CTAs of a segment, 1 to 8
    bool prompt;       // k_kv8_prompt: row tiles of kPrRows
    size_t part_bytes, stat_bytes, segment_bytes, lse2_bytes, score_bytes;  // multiples of 16
    size_t bytes() const { return part_bytes + stat_bytes + segment_bytes + lse2_bytes + score_bytes; }
};

int64_t score_stride(int max_length) { return (static_cast<int64_t>(max_length) + 3) / 4 * 4; }

AttnPlan attn_plan(const OpContext& o, const i4d_kv8_attention_args& a) {
    AttnPlan p = {};
    const i4d_kv8& c = a.cache;
    const int64_t rows = static_cast<int64_t>(a.max_q) * (a.heads / c.heads);
    p.dt = c.dim <= 64 ? 64 : c.dim <= 128 ? 128 : 256;
    p.nt = rows > 8 && a.dtype != I4D_F32 && p.dt <= 128 ? 2 : 1;
    // Up to 64 rows eight or sixteen a CTA on mma.sync, above 256 on tcgen05: one
    // sequence of 8192 tokens, 8 heads, 64 rows 34.8 us against 46.1, 128 rows 52
    // against 137; eight sequences cross at 45 rows (48: 112 against 105, 16: 69
    // against 101).  FP32 rows and dims above 128 have no tcgen05 form.
    p.prompt = rows > 64 && a.dtype != I4D_F32 && p.dt <= 128;
    const int tile = p.prompt ? kPrRows : 8 * p.nt;
    p.row_tiles = static_cast<int>((rows + tile - 1) / tile);
    p.segments = static_cast<int64_t>(a.batch) * c.heads * p.row_tiles;
    // Few segments of moderate length: as many CTAs of a cluster for each as
    // fit the GPU at once, which need no second kernel (one stream of 2047
    // tokens, 32 heads: 20.5 us through partial sums in memory, 13.3 to 13.8 so).  Long
    // ones: the CTAs that fit the GPU share all tokens evenly, whatever the
    // lengths are (which the device alone knows), but no more of them than have
    // two tiles a warp.  Above four row tiles a CTA takes a segment alone,
    // measured only where segments fill the GPU: 40 FP32 rows over one head of
    // 32000 tokens are five CTAs (481 us).
    const int64_t places = attn_places(p.dt, p.nt, a.dtype == I4D_F32) * static_cast<int64_t>(o.num_sms);
    p.cluster = 1;
    if (!p.prompt && p.row_tiles <= 4) {
        while (p.cluster < 8 && p.segments * p.cluster * 2 <= places && a.max_length > 128 * p.cluster) p.cluster *= 2;
        if (p.segments > places || a.max_length > 1024 * p.cluster) {
            const int64_t units = p.segments * ((a.max_length + 15) / 16);
            p.even = static_cast<int>(std::max<int64_t>(1, std::min(places, (units + 7) / 8)));
            p.cluster = 1;
        }
    }
    if (p.prompt) p.even = static_cast<int>(std::min<int64_t>(o.num_sms, p.segments * ((a.max_length + kPrTokens - 1) / kPrTokens + 1)));
    if (p.even) {
        p.part_bytes = static_cast<size_t>(p.even) * 2 * tile * c.dim * sizeof(float);
        p.stat_bytes = static_cast<size_t>(p.even) * 2 * tile * sizeof(float4);
        if (!p.prompt) p.segment_bytes = static_cast<size_t>(p.segments) * sizeof(int4);
    }
    if (a.weights) {
        p.lse2_bytes = (static_cast<size_t>(a.tokens) * a.heads * sizeof(float) + 15) / 16 * 16;
        // Few rows: their scores are kept (4 bytes a row against a token's codes
        // read again; 4 contexts of 9001 to 24571 tokens, 4 rows 73 us against 116,
        // 32 rows 161 against 232).
        if (rows <= 32) p.score_bytes = static_cast<size_t>(p.segments) * 8 * p.nt * score_stride(a.max_length) * sizeof(float);
    }
    return p;
}

i4d_status check_attention(i4d_ctx* ctx, const i4d_kv8_attention_args* a) {
    OP_ARG(a, "null arguments");
    i4d_status st = check_cache(ctx, a->cache);
    if (st == I4D_OK) st = check_batch(ctx, a->q_start, a->lengths, a->block_table, a->table_stride, a->table_blocks, a->batch, a->tokens, a->max_q);
    if (st != I4D_OK) return st;
    OP_ARG(is_dtype(a->dtype), "unknown dtype %d", a->dtype);
    OP_ARG(a->heads > 0 && a->heads % a->cache.heads == 0, "%d query heads over %d cache heads", a->heads, a->cache.heads);
    OP_ARG(a->max_length >= 0 && a->max_length <= kMaxTokens, "max_length %d", a->max_length);
    OP_ARG(a->window >= 0 && a->window <= kMaxTokens, "window %d", a->window);
    OP_ARG(static_cast<int64_t>(a->table_blocks) * a->cache.block_tokens >= a->max_length,
           "block_table rows of %d blocks hold fewer than max_length %d tokens", a->table_blocks, a->max_length);
    OP_ARG(static_cast<int64_t>(a->cache.blocks) * a->cache.heads * a->cache.block_tokens <= 0x7fffffff,
           "a cache of 2^31 or more (token, head) rows");
    OP_ARG(std::isfinite(a->scale), "scale is not finite");
    OP_ARG(static_cast<int64_t>(a->max_q) * (a->heads / a->cache.heads) <= kMaxTokens, "too many rows");
    return I4D_OK;
}

template <int DT, int CODE, int NT, bool HLQ, bool HLP>
cudaError_t launch_attn(const AttnDev& d, int64_t grid, cudaStream_t st) {
    static_assert(attn_smem<DT, NT>() <= 114688, "two CTAs an SM");
    static std::atomic<uint64_t> allowed{0};
    return launch_large(allowed, attn_smem<DT, NT>(), k_kv8_attn<DT, CODE, NT, HLQ, HLP>, grid, kAttnThreads, attn_smem<DT, NT>(), d.cluster, st, d);
}

template <int DT, int CODE>
cudaError_t launch_attn_d(const AttnDev& d, const AttnPlan& p, int64_t grid, cudaStream_t st) {
    if (d.dtype == I4D_F32) return launch_attn<DT, CODE, 1, true, true>(d, grid, st);
    if constexpr (DT <= 128) {
        if (p.nt == 2) return d.dtype == I4D_F16 ? launch_attn<DT, CODE, 2, false, true>(d, grid, st) : launch_attn<DT, CODE, 2, false, false>(d, grid, st);
    }
    return d.dtype == I4D_F16 ? launch_attn<DT, CODE, 1, false, true>(d, grid, st) : launch_attn<DT, CODE, 1, false, false>(d, grid, st);
}

template <int DT>
constexpr int kPromptSmem = PromptSmem<DT>::total + 1024;

template <int DT, int CODE, bool HLP>
cudaError_t launch_prompt(const AttnDev& d, int64_t grid, cudaStream_t st) {
    static std::atomic<uint64_t> allowed{0};
    return launch_large(allowed, kPromptSmem<DT>, k_kv8_prompt<DT, CODE, HLP>, grid, kPrThreads, kPromptSmem<DT>, 1, st, d);
}

template <int DT, int CODE>
cudaError_t launch_prompt_t(const AttnDev& d, int64_t grid, cudaStream_t st) {
    return d.dtype == I4D_F16 ? launch_prompt<DT, CODE, true>(d, grid, st) : launch_prompt<DT, CODE, false>(d, grid, st);
}

template <int CODE>
cudaError_t launch_attn_c(const AttnDev& d, const AttnPlan& p, int64_t grid, cudaStream_t st) {
    if (p.prompt) return p.dt == 64 ? launch_prompt_t<64, CODE>(d, grid, st) : launch_prompt_t<128, CODE>(d, grid, st);
    return p.dt == 64 ? launch_attn_d<64, CODE>(d, p, grid, st) : p.dt == 128 ? launch_attn_d<128, CODE>(d, p, grid, st) : launch_attn_d<256, CODE>(d, p, grid, st);
}

template <int DT, int CODE>
cudaError_t launch_weights(const AttnDev& d, int tiles, int64_t grid, cudaStream_t st) {
    if (d.dtype == I4D_F32) return launch(k_kv8_weights<DT, CODE, true>, grid, kAttnThreads, 0, 1, st, d, tiles);
    return launch(k_kv8_weights<DT, CODE, false>, grid, kAttnThreads, 0, 1, st, d, tiles);
}

template <int CODE>
cudaError_t launch_weights_c(const AttnDev& d, const AttnPlan& p, int tiles, int64_t grid, cudaStream_t st) {
    return p.dt == 64 ? launch_weights<64, CODE>(d, tiles, grid, st) : p.dt == 128 ? launch_weights<128, CODE>(d, tiles, grid, st) : launch_weights<256, CODE>(d, tiles, grid, st);
}

// ---------------------------------------------------------------- logits

template <typename T>
cudaError_t launch_logits(const LogitsDev& d, unsigned grid, int ctas, cudaStream_t st) {
    static std::atomic<uint64_t> allowed{0};
    return launch_large(allowed, logits_smem_bytes(kLogitsTouched, kLogitsPart / 32), k_logits<T>, grid, kLogitsThreads, logits_smem_bytes(d.places, d.words),
                        ctas, st, d, ctas);
}

// ----------------------------------------------------------------- evict

size_t evict_workspace(const i4d_kv8_evict_args& a) {
    const size_t old_blocks = (static_cast<size_t>(a.max_length) + a.cache.block_tokens - 1) / a.cache.block_tokens;
    return static_cast<size_t>(a.batch) * a.cache.heads * 2 * old_blocks * sizeof(float);
}

i4d_status check_evict(i4d_ctx* ctx, const i4d_kv8_evict_args* a) {
    OP_ARG(a, "null arguments");
    i4d_status st = check_cache(ctx, a->cache);
    if (st != I4D_OK) return st;
    OP_ARG(a->batch >= 0, "negative batch");
    OP_ARG(a->max_length >= 0 && a->max_length <= kMaxTokens, "max_length %d", a->max_length);
    OP_ARG(a->budget > 0 && a->recent >= 0 && a->recent <= a->budget, "budget %d, recent %d (0 <= recent <= budget, 0 < budget)", a->budget, a->recent);
    OP_ARG(a->budget <= kMaxTokens, "budget %d (2^30 at most: no sequence is longer)", a->budget);  // (an index and a step are an int)
    OP_ARG(a->table_stride >= 0 && a->table_blocks >= 0 && static_cast<int64_t>(a->table_blocks) * a->cache.block_tokens >= a->max_length,
           "block_table rows of %d blocks hold fewer than max_length %d tokens", a->table_blocks, a->max_length);
    OP_ARG(a->weights_stride >= a->max_length && a->weights_out_stride >= a->max_length, "weights' rows are shorter than max_length");
    return I4D_OK;
}

}  // namespace

namespace i4d_ops {

i4d_status ops_report(i4d_ctx* ctx) {
    const OpContext o = op_context(ctx);
    k_take_errors<<<1, 1, 0, o.err_stream>>>(o.err, o.err_taken);
    OP_CK(cudaGetLastError());
    OP_CK(cudaStreamSynchronize(o.err_stream));
    const unsigned e = *static_cast<volatile unsigned*>(o.err_taken);
    if (!e) return I4D_OK;
    if (e & kTimeout) return op_fail(ctx, I4D_ERR_TIMEOUT, "a bounded device wait of an operator gave up (error word 0x%x)", e);
    return op_fail(ctx, I4D_ERR_ARG, "an operator skipped tokens:%s%s", e & kBadSequence ? " q_start or lengths out of range;" : "",
                   e & kBadBlock ? " block id outside the pool;" : "");
}

}  // namespace i4d_ops

extern "C" {

i4d_status i4d_rope_frequencies(int rot_dim, double base, int scaling, double factor, double original_length, double low,
                                double high, uint64_t* turns_out) {
    if (!turns_out || rot_dim < 2 || rot_dim > 256 || rot_dim % 2 || !(base > 1.0) || !std::isfinite(base)) return I4D_ERR_ARG;
    if (scaling < I4D_ROPE_PLAIN || scaling > I4D_ROPE_PARTS) return I4D_ERR_ARG;
    if (scaling != I4D_ROPE_PLAIN && !(factor >= 1.0 && std::isfinite(factor))) return I4D_ERR_ARG;
    if (scaling == I4D_ROPE_BASE && rot_dim < 4) return I4D_ERR_ARG;
    if (scaling == I4D_ROPE_PARTS && !(original_length > 0.0 && high > low && std::isfinite(high) && std::isfinite(low) && std::isfinite(original_length)))
        return I4D_ERR_ARG;
    const double two_pi = 6.283185307179586476925286766559;
    if (scaling == I4D_ROPE_BASE) base *= std::pow(factor, rot_dim / (rot_dim - 2.0));
    for (int i = 0; i < rot_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rot_dim);
        if (scaling == I4D_ROPE_LINEAR) f /= factor;
        if (scaling == I4D_ROPE_PARTS) {
            const double g = std::min(1.0, std::max(0.0, (original_length * f / two_pi - low) / (high - low)));
            f *= g + (1.0 - g) / factor;
        }
        turns_out[i] = static_cast<uint64_t>(f / two_pi * 18446744073709551616.0 + 0.5);  // f <= 1 radian: under 2^62
    }
    return I4D_OK;
}

i4d_status i4d_rope(i4d_ctx* ctx, const i4d_rope_args* a) {
    if (!ctx) return I4D_ERR_ARG;
    OP_ARG(a, "null arguments");
    OP_ARG(is_dtype(a->dtype), "unknown dtype %d", a->dtype);
    OP_ARG(a->tokens >= 0 && a->q_heads > 0 && a->k_heads >= 0, "tokens %d, q_heads %d, k_heads %d", a->tokens, a->q_heads, a->k_heads);
    OP_ARG(a->dim > 0 && a->dim <= 4096, "dim %d (1 to 4096)", a->dim);
    OP_ARG(a->rot_dim >= 2 && a->rot_dim % 2 == 0 && a->rot_dim <= a->dim && a->rot_dim <= 256, "rot_dim %d (even, up to dim %d and 256)", a->rot_dim, a->dim);
    if (a->tokens == 0) return I4D_OK;
    OP_ARG(a->q && a->q_out && a->positions && a->turns, "null buffer");
    const bool has_k = a->k != nullptr && a->k_heads > 0;
    OP_ARG(!has_k || a->k_out, "null k_out");
    const int bytes = dtype_bytes(a->dtype);
    RopeDev d = {};
    const void* in[2] = {a->q, has_k ? a->k : nullptr};
    void* out[2] = {a->q_out, has_k ? a->k_out : nullptr};
    const int64_t in_s[2] = {a->q_stride, a->k_stride}, in_h[2] = {a->q_head_stride, a->k_head_stride};
    const int64_t out_s[2] = {a->q_out_stride, a->k_out_stride}, out_h[2] = {a->q_out_head_stride, a->k_out_head_stride};
    View vi[2] = {}, vo[2] = {};
    const int vec = 16 / bytes;
    bool wide = a->dim % vec == 0 && a->rot_dim % (a->interleaved ? vec : 2 * vec) == 0;
    bool copy = false;
    for (int i = 0; i < 2; ++i) {
        const int heads = i ? (has_k ? a->k_heads : 0) : a->q_heads;
        d.in[i] = in[i];
        d.out[i] = out[i];
        d.in_tok[i] = in_s[i];
        d.in_head[i] = in_h[i];
        d.out_tok[i] = out_s[i];
        d.out_head[i] = out_h[i];
        d.heads[i] = heads;
        vi[i] = {i ? "k" : "q", in[i], a->tokens, in_s[i], heads, in_h[i], a->dim, bytes};
        vo[i] = {i ? "k_out" : "q_out", out[i], a->tokens, out_s[i], heads, out_h[i], a->dim, bytes};
        if (!heads) continue;
        OP_ARG(aligned(in[i], bytes) && aligned(out[i], bytes), "misaligned %s or %s", vi[i].name, vo[i].name);
        OP_ARG(in_s[i] >= 0 && in_h[i] >= 0, "negative stride of %s", vi[i].name);
        OP_ARG(out_s[i] >= 0 && out_h[i] >= 0 && rows_apart(vo[i]), "rows of %s overlap", vo[i].name);
        wide = wide && aligned(in[i], 16) && aligned(out[i], 16) && in_s[i] % vec == 0 && in_h[i] % vec == 0 && out_s[i] % vec == 0 && out_h[i] % vec == 0;
    }
    for (int i = 0; i < 2; ++i) {
        if (!d.heads[i]) continue;
        OP_ARG(vi[i].same(vo[i]) || !overlap(vi[i], vo[i]), "%s overlaps %s", vo[i].name, vi[i].name);
        OP_ARG(!d.heads[1 - i] || !overlap(vo[i], vi[1 - i]), "%s overlaps %s", vo[i].name, vi[1 - i].name);
        copy = copy || !vi[i].same(vo[i]);
    }
    OP_ARG(!has_k || !overlap(vo[0], vo[1]), "q_out overlaps k_out");
    for (const View& v : vo) {
        const i4d_status st = check_apart(ctx, {v.span()}, {span_of("positions", a->positions, a->tokens, 4), span_of("turns", a->turns, a->rot_dim / 2, 8)});
        if (st != I4D_OK) return st;
    }
    OP_ARG(aligned(a->positions, 4) && aligned(a->turns, 8), "misaligned positions or turns");
    d.positions = a->positions;
    d.turns = a->turns;
    d.tokens = a->tokens;
    d.dim = a->dim;
    d.rot = a->rot_dim;
    d.inverse = a->inverse != 0;
    d.copy_tail = copy && a->dim > a->rot_dim;
    d.magnitude = a->magnitude;
    if (!wide && a->interleaved) OP_ARG((a->dim - a->rot_dim) % 2 == 0 || !d.copy_tail, "dim %d must be even", a->dim);
    const OpContext o = op_context(ctx);
    DeviceScope scope(o.device);
    OP_CK(scope.error());
    const cudaStream_t st = stream_of(o, a->stream);
    switch (a->dtype) {
        case I4D_F32: OP_CK(launch_rope_t<float>(d, a->interleaved != 0, wide, o.num_sms, st)); break;
        case I4D_BF16: OP_CK(launch_rope_t<__nv_bfloat16>(d, a->interleaved != 0, wide, o.num_sms, st)); break;
        default: OP_CK(launch_rope_t<__half>(d, a->interleaved != 0, wide, o.num_sms, st)); break;
    }
    return I4D_OK;
}

i4d_status i4d_kv8_append(i4d_ctx* ctx, const i4d_kv8_append_args* a) {
    if (!ctx) return I4D_ERR_ARG;
    OP_ARG(a, "null arguments");
    i4d_status st = check_cache(ctx, a->cache);
    if (st == I4D_OK) st = check_batch(ctx, a->q_start, a->lengths, a->block_table, a->table_stride, a->table_blocks, a->batch, a->tokens, a->max_q);
    if (st != I4D_OK) return st;
    OP_ARG(is_dtype(a->dtype), "unknown dtype %d", a->dtype);
    if (a->batch == 0 || a->tokens == 0 || a->max_q == 0) return I4D_OK;
    OP_ARG(a->k && a->v, "null k or v");
    const int bytes = dtype_bytes(a->dtype);
    OP_ARG(aligned(a->k, bytes) && aligned(a->v, bytes), "misaligned k or v");
    OP_ARG(a->k_stride >= 0 && a->k_head_stride >= 0 && a->v_stride >= 0 && a->v_head_stride >= 0, "negative stride");
    st = check_apart(ctx, {CACHE_SPANS(a->cache)},
                     {span_of("k", a->k, a->tokens, a->k_stride, a->cache.heads, a->k_head_stride, a->cache.dim, bytes),
                      span_of("v", a->v, a->tokens, a->v_stride, a->cache.heads, a->v_head_stride, a->cache.dim, bytes), BATCH_SPANS(a)});
    if (st != I4D_OK) return st;
    const OpContext o = op_context(ctx);
    AppendDev d = {};
    d.cache = cache_dev(a->cache);
    d.seq = seq_arrays(o, a->cache, a->q_start, a->lengths, a->block_table, a->table_stride, a->table_blocks, a->tokens, a->max_q);
    d.in[0] = a->k;
    d.in[1] = a->v;
    d.tok[0] = a->k_stride;
    d.tok[1] = a->v_stride;
    d.head[0] = a->k_head_stride;
    d.head[1] = a->v_head_stride;
    const int bs = a->cache.block_tokens;
    d.touched = touched_blocks(a->max_q, a->tokens, bs);
    const int64_t units = static_cast<int64_t>(a->batch) * d.touched * a->cache.heads * 2;
    OP_ARG(units <= kMaxGrid, "too many blocks in one call");
    // 8 elements an access: two of 16 bytes for FP32, one for the others
    const int vec = 16 / bytes;
    const bool wide = aligned(a->k, 16) && aligned(a->v, 16) && a->k_stride % vec == 0 && a->k_head_stride % vec == 0 &&
                      a->v_stride % vec == 0 && a->v_head_stride % vec == 0;
    const int64_t items = static_cast<int64_t>(std::min(a->max_q, bs)) * a->cache.dim / 8;
    DeviceScope scope(o.device);
    OP_CK(scope.error());
    const cudaStream_t s = stream_of(o, a->stream);
    switch (a->dtype) {
        case I4D_F32: OP_CK(launch_append_t<float>(d, a->cache.code, wide, units, items, s)); break;
        case I4D_BF16: OP_CK(launch_append_t<__nv_bfloat16>(d, a->cache.code, wide, units, items, s)); break;
        default: OP_CK(launch_append_t<__half>(d, a->cache.code, wide, units, items, s)); break;
    }
    return I4D_OK;
}

i4d_status i4d_kv8_read(i4d_ctx* ctx, const i4d_kv8_read_args* a) {
    if (!ctx) return I4D_ERR_ARG;
    OP_ARG(a, "null arguments");
    i4d_status st = check_cache(ctx, a->cache);
    if (st == I4D_OK) st = check_batch(ctx, a->q_start, a->lengths, a->block_table, a->table_stride, a->table_blocks, a->batch, a->tokens, a->max_q);
    if (st != I4D_OK) return st;
    if (a->batch == 0 || a->tokens == 0 || a->max_q == 0) return I4D_OK;
    OP_ARG(a->k_out && a->v_out && aligned(a->k_out, 16) && aligned(a->v_out, 16), "k_out and v_out need 16-byte alignment");
    const int64_t rows = static_cast<int64_t>(a->tokens) * a->cache.heads * a->cache.dim;
    st = check_apart(ctx, {span_of("k_out", a->k_out, rows, 2), span_of("v_out", a->v_out, rows, 2)}, {CACHE_SPANS(a->cache), BATCH_SPANS(a)});
    if (st != I4D_OK) return st;
    const OpContext o = op_context(ctx);
    ReadDev d = {};
    d.cache = cache_dev(a->cache);
    d.seq = seq_arrays(o, a->cache, a->q_start, a->lengths, a->block_table, a->table_stride, a->table_blocks, a->tokens, a->max_q);
    d.out[0] = static_cast<__nv_bfloat16*>(a->k_out);
    d.out[1] = static_cast<__nv_bfloat16*>(a->v_out);
    const int64_t per_seq = static_cast<int64_t>(a->max_q) * a->cache.heads * (a->cache.dim / 16);
    OP_ARG(per_seq <= kMaxTokens, "too many rows in one call");
    const int chunks = static_cast<int>((per_seq + kReadItems - 1) / kReadItems);
    const int64_t grid = static_cast<int64_t>(a->batch) * chunks;
    OP_ARG(grid <= kMaxGrid, "too many rows in one call");
    DeviceScope scope(o.device);
    OP_CK(scope.error());
    const cudaStream_t s = stream_of(o, a->stream);
    OP_CK(a->cache.code == I4D_CODE_INT8 ? launch(k_kv8_read<I4D_CODE_INT8>, grid, 256, 0, 1, s, d, chunks)
                                         : launch(k_kv8_read<I4D_CODE_E4M3>, grid, 256, 0, 1, s, d, chunks));
    return I4D_OK;
}

i4d_status i4d_kv8_attention_workspace(i4d_ctx* ctx, const i4d_kv8_attention_args* a, size_t* bytes_out) {
    if (!ctx) return I4D_ERR_ARG;
    const i4d_status st = check_attention(ctx, a);
    if (st != I4D_OK) return st;
    OP_ARG(bytes_out, "null bytes_out");
    const AttnPlan p = attn_plan(op_context(ctx), *a);
    *bytes_out = p.bytes();
    return I4D_OK;
}

i4d_status i4d_kv8_attention(i4d_ctx* ctx, const i4d_kv8_attention_args* a) {
    if (!ctx) return I4D_ERR_ARG;
    i4d_status st = check_attention(ctx, a);
    if (st != I4D_OK) return st;
    if (a->batch == 0 || a->tokens == 0 || a->max_q == 0) return I4D_OK;
    OP_ARG(a->q && a->out, "null q or out");
    const int bytes = dtype_bytes(a->dtype), dim = a->cache.dim;
    OP_ARG(aligned(a->q, bytes) && aligned(a->out, bytes) && aligned(a->lse, 4) && aligned(a->weights, 4), "misaligned buffer");
    OP_ARG(a->q_stride >= 0 && a->q_head_stride >= 0, "negative q stride");
    const View vq = {"q", a->q, a->tokens, a->q_stride, a->heads, a->q_head_stride, dim, bytes};
    const View vout = {"out", a->out, a->tokens, a->out_stride, a->heads, a->out_head_stride, dim, bytes};
    OP_ARG(a->out_stride >= 0 && a->out_head_stride >= 0 && rows_apart(vout), "rows of out overlap");
    OP_ARG(!overlap(vq, vout), "out overlaps q");
    OP_ARG(!a->weights || a->weights_stride >= a->max_length, "weights' rows are shorter than max_length");
    const OpContext o = op_context(ctx);
    const AttnPlan p = attn_plan(o, *a);
    const size_t need = p.bytes();
    const Span weights = span_of("weights", a->weights, static_cast<int64_t>(a->batch) * a->cache.heads, a->weights_stride, 1, 0, a->max_length, 4);
    const Span lse = span_of("lse", a->lse, static_cast<int64_t>(a->tokens) * a->heads, 4), space = span_of("workspace", a->workspace, need, 1);
    st = check_apart(ctx, {vout.span(), lse, weights, space}, {CACHE_SPANS(a->cache), BATCH_SPANS(a)});
    if (st == I4D_OK) st = check_apart(ctx, {lse, weights, space}, {vq.span()});
    if (st != I4D_OK) return st;
    OP_ARG(need == 0 || (a->workspace && aligned(a->workspace, 16)), "null or misaligned workspace (%zu bytes needed)", need);
    if (a->workspace_bytes < need) return op_fail(ctx, I4D_ERR_SIZE, "workspace of %zu bytes; %zu needed", a->workspace_bytes, need);
    AttnDev d = {};
    d.cache = cache_dev(a->cache);
    d.seq = seq_arrays(o, a->cache, a->q_start, a->lengths, a->block_table, a->table_stride, a->table_blocks, a->tokens, a->max_q);
    d.q = a->q;
    d.out = a->out;
    d.lse = a->lse;
    d.weights = a->weights;
    d.q_tok = a->q_stride;
    d.q_head = a->q_head_stride;
    d.out_tok = a->out_stride;
    d.out_head = a->out_head_stride;
    d.weights_stride = a->weights_stride;
    d.heads = a->heads;
    d.group = a->heads / a->cache.heads;
    d.window = a->window;
    d.dtype = a->dtype;
    d.max_length = a->max_length;
    d.scale_log2 = a->scale * kLog2e;
    d.batch = a->batch;
    d.row_tiles = p.row_tiles;
    d.even = p.even;
    d.cluster = p.cluster;
    d.part = static_cast<float*>(a->workspace);
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    d.stats = reinterpret_cast<float4*>(ws + p.part_bytes);
    d.segments = reinterpret_cast<int4*>(ws + p.part_bytes + p.stat_bytes);
    d.lse2 = reinterpret_cast<float*>(ws + p.part_bytes + p.stat_bytes + p.segment_bytes);
    if (p.score_bytes) d.scores = reinterpret_cast<float*>(ws + p.part_bytes + p.stat_bytes + p.segment_bytes + p.lse2_bytes);
    d.score_stride = score_stride(a->max_length);
    d.wide_out = aligned(a->out, 16) && a->out_stride * bytes % 16 == 0 && a->out_head_stride * bytes % 16 == 0;
    d.wide_q = aligned(a->q, 16) && a->q_stride * bytes % 16 == 0 && a->q_head_stride * bytes % 16 == 0;
    const int64_t grid = p.even ? p.even : p.segments * p.cluster;
    const int wtiles = (a->max_length + 16 * kAttnWarps - 1) / (16 * kAttnWarps);
    const int64_t wgrid = static_cast<int64_t>(a->batch) * a->cache.heads * wtiles;
    OP_ARG(p.segments * 8 <= kMaxGrid && wgrid <= kMaxGrid, "too many rows in one call");
    DeviceScope scope(o.device);
    OP_CK(scope.error());
    const cudaStream_t s = stream_of(o, a->stream);
    const bool int8 = a->cache.code == I4D_CODE_INT8;
    i4d_status enc = encode_codes(ctx, a->cache, a->cache.k, 16, &d.maps[0]);
    if (enc == I4D_OK) enc = encode_codes(ctx, a->cache, a->cache.v, 16, &d.maps[1]);
    if (enc != I4D_OK) return enc;
    OP_CK(int8 ? launch_attn_c<I4D_CODE_INT8>(d, p, grid, s) : launch_attn_c<I4D_CODE_E4M3>(d, p, grid, s));
    if (p.prompt) {
        if (p.even > 1) OP_CK(launch(k_kv8_prompt_join, 8 * (p.even - 1), 256, 0, 1, s, d));
    } else if (p.even > 1) OP_CK(launch(k_kv8_join, p.segments, kJoinThreads, 0, 1, s, d, 8 * p.nt));
    if (d.scores) {
        const int chunks = (a->max_length + 511) / 512;
        if (chunks > 0) {
            OP_CK(launch(k_kv8_weights_kept, static_cast<int64_t>(a->batch) * a->cache.heads * chunks, 128, 0, 1, s, d, 8 * p.nt, chunks));
        }
    } else if (a->weights && wgrid > 0)
        OP_CK(int8 ? launch_weights_c<I4D_CODE_INT8>(d, p, wtiles, wgrid, s) : launch_weights_c<I4D_CODE_E4M3>(d, p, wtiles, wgrid, s));
    return I4D_OK;
}

i4d_status i4d_kv8_evict_workspace(i4d_ctx* ctx, const i4d_kv8_evict_args* a, size_t* bytes_out) {
    if (!ctx) return I4D_ERR_ARG;
    const i4d_status st = check_evict(ctx, a);
    if (st != I4D_OK) return st;
    OP_ARG(bytes_out, "null bytes_out");
    *bytes_out = evict_workspace(*a);
    return I4D_OK;
}

i4d_status i4d_kv8_evict(i4d_ctx* ctx, const i4d_kv8_evict_args* a) {
    if (!ctx) return I4D_ERR_ARG;
    i4d_status st = check_evict(ctx, a);
    if (st != I4D_OK) return st;
    if (a->batch == 0) return I4D_OK;
    OP_ARG(a->lengths && a->lengths_out && a->keep && a->block_table && a->weights && a->weights_out, "null buffer");
    OP_ARG(aligned(a->lengths, 4) && aligned(a->lengths_out, 4) && aligned(a->keep, 4) && aligned(a->block_table, 4) &&
               aligned(a->weights, 4) && aligned(a->weights_out, 4), "arrays need 4-byte alignment");
    const int heads = a->cache.heads;
    const size_t need = evict_workspace(*a);
    OP_ARG(need == 0 || (a->workspace && aligned(a->workspace, 16)), "null or misaligned workspace (%zu bytes needed)", need);
    if (a->workspace_bytes < need) return op_fail(ctx, I4D_ERR_SIZE, "workspace of %zu bytes; %zu needed", a->workspace_bytes, need);
    const int64_t weight_rows = static_cast<int64_t>(a->batch) * heads;
    const Span win = span_of("weights", a->weights, weight_rows, a->weights_stride, 1, 0, a->max_length, 4);
    const Span wout = span_of("weights_out", a->weights_out, weight_rows, a->weights_out_stride, 1, 0, a->max_length, 4);
    OP_ARG((a->weights == a->weights_out && a->weights_stride == a->weights_out_stride) || !overlap(win, wout), "weights_out overlaps weights");
    st = check_apart(ctx, {wout, span_of("lengths_out", a->lengths_out, a->batch, 4), span_of("keep", a->keep, weight_rows * a->budget, 4),
                           span_of("workspace", a->workspace, need, 1), CACHE_SPANS(a->cache)},
                     {span_of("lengths", a->lengths, a->batch, 4), span_of("block_table", a->block_table, a->batch, a->table_stride, 1, 0, a->table_blocks, 4)});
    if (st == I4D_OK) st = check_apart(ctx, {span_of("lengths_out", a->lengths_out, a->batch, 4), span_of("keep", a->keep, weight_rows * a->budget, 4),
                                             span_of("workspace", a->workspace, need, 1), CACHE_SPANS(a->cache)}, {win});
    if (st != I4D_OK) return st;
    const OpContext o = op_context(ctx);
    EvictDev d = {};
    d.cache = cache_dev(a->cache);
    d.seq = seq_arrays(o, a->cache, nullptr, a->lengths, a->block_table, a->table_stride, a->table_blocks, 0, 0);
    d.weights = a->weights;
    d.weights_out = a->weights_out;
    d.weights_stride = a->weights_stride;
    d.weights_out_stride = a->weights_out_stride;
    d.lengths_out = a->lengths_out;
    d.keep = a->keep;
    d.old_scale = static_cast<float*>(a->workspace);
    d.old_blocks = (a->max_length + a->cache.block_tokens - 1) / a->cache.block_tokens;
    d.budget = a->budget;
    d.recent = a->recent;
    d.max_length = a->max_length;
    const int64_t rows = static_cast<int64_t>(a->batch) * heads;
    // CTAs of a row of weights: two thousand or more each; of a moved row: a
    // round's tokens each, no more than fit the GPU at once; eight at most (the
    // portable cluster size).
    int ctas = 1, movers = 1;
    while (ctas < 8 && a->max_length / (2 * ctas) >= 2048) ctas *= 2;
    while (movers < 8 && a->budget > movers * move_tokens(a->cache.dim) && rows * 4 * movers <= 2 * o.num_sms) movers *= 2;
    OP_ARG(rows * 2 * 8 <= kMaxGrid, "too many sequences in one call");
    DeviceScope scope(o.device);
    OP_CK(scope.error());
    const cudaStream_t s = stream_of(o, a->stream);
    OP_CK(launch(k_kv8_select, static_cast<unsigned>(rows * ctas), kSelectThreads, 0, ctas, s, d, ctas));
    if (a->max_length > a->budget) {
        const unsigned grid = static_cast<unsigned>(rows * 2 * movers);
        OP_CK(a->cache.code == I4D_CODE_INT8 ? launch(k_kv8_move<I4D_CODE_INT8>, grid, kMoveThreads, 0, movers, s, d, movers)
                                             : launch(k_kv8_move<I4D_CODE_E4M3>, grid, kMoveThreads, 0, movers, s, d, movers));
    }
    return I4D_OK;
}

i4d_status i4d_logits_process(i4d_ctx* ctx, const i4d_logits_args* a) {
    if (!ctx) return I4D_ERR_ARG;
    OP_ARG(a, "null arguments");
    OP_ARG(is_dtype(a->dtype), "unknown dtype %d", a->dtype);
    OP_ARG(a->rows >= 0 && a->vocab > 0 && a->vocab <= kMaxTokens, "rows %d, vocab %d", a->rows, a->vocab);
    if (a->rows == 0) return I4D_OK;
    OP_ARG(a->logits && a->out, "null logits or out");
    const int bytes = dtype_bytes(a->dtype);
    OP_ARG(aligned(a->logits, bytes) && aligned(a->out, bytes), "misaligned logits or out");
    OP_ARG(a->stride >= 0 && (a->rows == 1 || a->out_stride >= a->vocab), "stride %lld, out_stride %lld for %d entries",
           static_cast<long long>(a->stride), static_cast<long long>(a->out_stride), a->vocab);
    OP_ARG((a->logits == a->out && a->stride == a->out_stride) ||
               !overlap(View{"logits", a->logits, a->rows, a->stride, 1, 0, a->vocab, bytes}, View{"out", a->out, a->rows, a->out_stride, 1, 0, a->vocab, bytes}),
           "out overlaps logits");
    OP_ARG(!a->history || (a->history_len && a->history_stride >= 0 && a->history_max >= 0 && a->history_max <= kMaxTokens), "history without history_len, or bad history_stride or history_max");
    OP_ARG(a->history || !(a->repetition || a->frequency || a->presence || a->prompt_len), "penalties without a history");
    OP_ARG(!a->bias_ids == !a->bias_values && !a->bias_ids == !a->bias_len, "bias_ids, bias_values and bias_len go together");
    OP_ARG(!a->bias_ids || (a->bias_stride >= 0 && a->bias_max >= 0 && a->bias_max <= kMaxTokens), "bad bias_stride or bias_max");
    OP_ARG(!a->mask || a->mask_stride >= 0, "negative mask_stride");
    const Span out = span_of("out", a->out, a->rows, a->out_stride, 1, 0, a->vocab, bytes), best = span_of("best", a->best, a->rows, 4);
    i4d_status st = check_apart(
        ctx, {out, best},
        {span_of("history", a->history, a->rows, a->history_stride, 1, 0, a->history_max, 4), span_of("history_len", a->history_len, a->rows, 4),
         span_of("prompt_len", a->prompt_len, a->rows, 4), span_of("repetition", a->repetition, a->rows, 4), span_of("frequency", a->frequency, a->rows, 4),
         span_of("presence", a->presence, a->rows, 4), span_of("bias_ids", a->bias_ids, a->rows, a->bias_stride, 1, 0, a->bias_max, 4),
         span_of("bias_values", a->bias_values, a->rows, a->bias_stride, 1, 0, a->bias_max, 4), span_of("bias_len", a->bias_len, a->rows, 4),
         span_of("mask", a->mask, a->rows, a->mask_stride, 1, 0, (a->vocab + 31) / 32, 4)});
    if (st == I4D_OK) st = check_apart(ctx, {best}, {span_of("logits", a->logits, a->rows, a->stride, 1, 0, a->vocab, bytes)});
    if (st != I4D_OK) return st;
    OP_ARG(aligned(a->best, 4) && aligned(a->history, 4) && aligned(a->history_len, 4) && aligned(a->prompt_len, 4) && aligned(a->repetition, 4) &&
               aligned(a->frequency, 4) && aligned(a->presence, 4) && aligned(a->bias_ids, 4) && aligned(a->bias_values, 4) && aligned(a->bias_len, 4) &&
               aligned(a->mask, 4), "arrays need 4-byte alignment");
    LogitsDev d = {};
    d.in = a->logits;
    d.out = a->out;
    d.best = a->best;
    d.history = a->history;
    d.history_len = a->history_len;
    d.prompt_len = a->prompt_len;
    d.repetition = a->repetition;
    d.frequency = a->frequency;
    d.presence = a->presence;
    d.bias_ids = a->bias_ids;
    d.bias_values = a->bias_values;
    d.bias_len = a->bias_len;
    d.mask = a->mask;
    d.stride = a->stride;
    d.out_stride = a->out_stride;
    d.history_stride = a->history_stride;
    d.bias_stride = a->bias_stride;
    d.mask_stride = a->mask_stride;
    d.vocab = a->vocab;
    d.history_max = a->history_max;
    d.bias_max = a->bias_max;
    // CTAs of a row: parts of at least 2048 entries, eight at most (the portable
    // cluster size), no more than fill the places of two CTAs an SM once, since
    // each reads the row's whole lists (192 rows of 128001 with histories: 60 us
    // with two a row, 64 with one, 71 with four, 101 with eight).
    const OpContext o = op_context(ctx);
    int ctas = 1;
    while (ctas < 8 && a->vocab / (2 * ctas) >= 2048 && static_cast<int64_t>(a->rows) * ctas < 2 * o.num_sms) ctas *= 2;
    OP_ARG(static_cast<int64_t>(a->rows) * ctas <= kMaxGrid, "too many rows in one call");
    DeviceScope scope(o.device);
    OP_CK(scope.error());
    const unsigned grid = static_cast<unsigned>(a->rows * ctas);
    const cudaStream_t s = stream_of(o, a->stream);
    // Shared memory for the ids that the lists can hold and a CTA's part of the row.
    const int64_t ids = static_cast<int64_t>(a->history ? a->history_max : 0) + (a->bias_ids ? a->bias_max : 0);
    d.places = static_cast<int>(std::min<int64_t>(kLogitsTouched, (ids + 255) / 256 * 256));
    d.words = std::min(kLogitsPart / 32, ((a->vocab + ctas - 1) / ctas + 32 + 127) / 128 * 4);
    switch (a->dtype) {
        case I4D_F32: OP_CK(launch_logits<float>(d, grid, ctas, s)); break;
        case I4D_BF16: OP_CK(launch_logits<__nv_bfloat16>(d, grid, ctas, s)); break;
        default: OP_CK(launch_logits<__half>(d, grid, ctas, s)); break;
    }
    return I4D_OK;
}

i4d_status i4d_ops_check(i4d_ctx* ctx, void* stream) {
    if (!ctx) return I4D_ERR_ARG;
    const OpContext o = op_context(ctx);
    DeviceScope scope(o.device);
    OP_CK(scope.error());
    OP_CK(cudaStreamSynchronize(stream ? static_cast<cudaStream_t>(stream) : o.stream));
    return ops_report(ctx);
}

}  // extern "C"
