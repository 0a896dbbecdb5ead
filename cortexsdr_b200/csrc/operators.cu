// C-ABI of the operators that stand on their own: the paged 4-bit key/value cache, products with 4-bit weights,
// and log probabilities of given tokens. Argument checks here, arithmetic in kernels/.
#include <cmath>
#include <cstring>
#include <initializer_list>
#include <limits>
#include <vector>

#include "internal.hpp"
#include "kernels/kv_cache.hpp"
#include "kernels/logprobs.hpp"
#include "kernels/q4_matmul.hpp"

using namespace csdr;

namespace {

void need_dtype(int dtype) {
    if (dtype != CSDR_DTYPE_F32 && dtype != CSDR_DTYPE_BF16 && dtype != CSDR_DTYPE_F16)
        throw Error(CSDR_ERR_INVALID_ARG, "unknown dtype");
}

// Elements of `bytes` bytes are read and written whole.
void need_whole(size_t bytes, std::initializer_list<const void*> pointers) {
    for (const void* p : pointers)
        if (reinterpret_cast<uintptr_t>(p) % bytes) throw Error(CSDR_ERR_INVALID_ARG, "a pointer is not on a whole element");
}
size_t dtype_bytes(int dtype) { return dtype == CSDR_DTYPE_F32 ? 4u : 2u; }

void need_cache(csdr_kv_cache* c, uint32_t layer) {
    if (!c) throw Error(CSDR_ERR_INVALID_ARG, "cache is null");
    require_ctx(c->ctx);
    if (layer >= c->n_layers) throw Error(CSDR_ERR_INVALID_ARG, "layer out of range");
}

KvBatchView view_of(const csdr_kv_batch* b) {
    if (!b) throw Error(CSDR_ERR_INVALID_ARG, "batch is null");
    if (b->n_tokens && b->n_seqs && (!b->first_dev || !b->length_dev || !b->pages_dev))
        throw Error(CSDR_ERR_INVALID_ARG, "batch: null array");
    if (b->n_tokens > 0x7FFFFFFFu || b->n_seqs > 0x7FFFFFFEu || b->pages_per_seq == 0)
        throw Error(CSDR_ERR_INVALID_ARG, "batch: counts out of range");
    need_whole(4, {b->first_dev, b->length_dev, b->pages_dev});
    return {b->first_dev, b->length_dev, b->pages_dev, b->n_seqs, b->n_tokens, b->pages_per_seq};
}

size_t row_stride(size_t given, size_t row, const char* what) {
    if (!given) return row;
    if (given < row) throw Error(CSDR_ERR_INVALID_ARG, std::string(what) + ": stride is less than a row");
    return given;
}

}  // namespace

extern "C" {

int csdr_kv_cache_create(csdr_context* ctx, uint32_t n_layers, uint32_t n_pages, uint32_t page_tokens, uint32_t kv_heads,
                         uint32_t head_dim, float rope_theta, csdr_kv_cache** out) {
    return guard([&] {
        require_ctx(ctx);
        if (!out) throw Error(CSDR_ERR_INVALID_ARG, "out is null");
        if (!n_layers || !n_pages || !kv_heads || n_pages > 0x7FFFFFFFu || kv_heads > 65535u)      // as q_heads
            throw Error(CSDR_ERR_INVALID_ARG, "cache: zero or out-of-range field");
        if (page_tokens < kKvBlock || page_tokens > 4096u || (page_tokens & (page_tokens - 1u)))
            throw Error(CSDR_ERR_INVALID_ARG, "cache: page_tokens must be a power of two from 16 to 4096");
        if (head_dim != 64 && head_dim != 128 && head_dim != 256)
            throw Error(CSDR_ERR_UNSUPPORTED, "cache: head_dim must be 64, 128 or 256");
        if (!std::isfinite(rope_theta)) throw Error(CSDR_ERR_INVALID_ARG, "cache: rope_theta is not finite");
        if (rope_theta > 0.0f && rope_theta < 1.0f)
            throw Error(CSDR_ERR_INVALID_ARG, "cache: rope_theta must be at least 1, or none (<= 0)");
        auto c = std::make_unique<csdr_kv_cache>();
        c->ctx = ctx;
        c->n_layers = n_layers;
        c->n_pages = n_pages;
        c->page_tokens = page_tokens;
        c->kv_heads = kv_heads;
        c->head_dim = head_dim;
        c->view.n_pages = n_pages;
        c->view.kv_heads = kv_heads;
        while ((1u << c->view.page_shift) < page_tokens) ++c->view.page_shift;
        c->view.block_bytes = 18u * head_dim;
        const double bytes = static_cast<double>(n_layers) * n_pages * kv_heads * (page_tokens / kKvBlock) * c->view.block_bytes;
        if (bytes > 1e15) throw Error(CSDR_ERR_LIMIT, "cache: larger than any device");
        c->layer_bytes = static_cast<size_t>(n_pages) * kv_heads * (page_tokens / kKvBlock) * c->view.block_bytes;
        c->data = std::make_shared<DeviceBuffer>(c->layer_bytes * n_layers, ctx->device);
        c->view.base = static_cast<uint8_t*>(c->data->ptr);
        CSDR_CUDA(cudaMemsetAsync(c->data->ptr, 0, c->data->bytes, ctx->stream));
        c->workspace = std::make_shared<DeviceBuffer>(kv_attention_workspace(ctx, head_dim), ctx->device);
        CSDR_CUDA(cudaMemsetAsync(c->workspace->ptr, 0, c->workspace->bytes, ctx->stream));
        if (rope_theta > 0.0f) {
            std::vector<double> freq(head_dim / 2);
            for (uint32_t i = 0; i < head_dim / 2; ++i) freq[i] = std::pow(static_cast<double>(rope_theta), -2.0 * i / head_dim);
            c->freq = upload(ctx, freq.data(), freq.size() * 8u);
        }
        CSDR_CUDA(cudaStreamSynchronize(ctx->stream));
        *out = c.release();
    });
}

int csdr_kv_cache_destroy(csdr_kv_cache* c) {
    return guard([&] {
        if (!c) return;
        cudaSetDevice(c->ctx->device);
        cudaStreamSynchronize(c->ctx->stream);
        delete c;
    });
}

int csdr_kv_cache_bytes(const csdr_kv_cache* c, size_t* bytes) {
    return guard([&] {
        if (!c || !bytes) throw Error(CSDR_ERR_INVALID_ARG, "null argument");
        *bytes = c->data->bytes;
    });
}

int csdr_kv_cache_append_device_async(csdr_kv_cache* c, uint32_t layer, const csdr_kv_batch* batch, const void* k_dev,
                                      const void* v_dev, size_t kv_stride, int dtype, int rotate, const void* q_dev,
                                      size_t q_stride, uint32_t q_heads, void* q_out_dev, size_t q_out_stride) {
    return guard([&] {
        need_cache(c, layer);
        const KvBatchView b = view_of(batch);
        need_dtype(dtype);
        KvAppend a{};
        a.k = k_dev;
        a.v = v_dev;
        a.q = q_dev;
        a.q_out = q_out_dev;
        a.kv_stride = row_stride(kv_stride, static_cast<size_t>(c->kv_heads) * c->head_dim, "k and v");
        need_whole(dtype_bytes(dtype), {k_dev, v_dev, q_dev, q_dev ? q_out_dev : nullptr});
        if (q_dev) {
            if (!q_heads || q_heads > 65535u) throw Error(CSDR_ERR_INVALID_ARG, "q: head count out of range");
            if (!q_out_dev) throw Error(CSDR_ERR_INVALID_ARG, "q_out is null");
            a.q_heads = q_heads;
            a.q_stride = row_stride(q_stride, static_cast<size_t>(q_heads) * c->head_dim, "q");
            a.q_out_stride = row_stride(q_out_stride, static_cast<size_t>(q_heads) * c->head_dim, "q_out");
            if (q_out_dev == q_dev && a.q_stride != a.q_out_stride && b.n_tokens > 1u)
                throw Error(CSDR_ERR_INVALID_ARG, "q_out is q, but its stride is another");
        }
        if (rotate && !c->freq) throw Error(CSDR_ERR_INVALID_ARG, "the cache was made without a rotation (rope_theta <= 0)");
        if (rotate) a.freq = static_cast<const double*>(c->freq->ptr);
        if (!b.n_tokens || !b.n_seqs) return;
        if (!k_dev || !v_dev) throw Error(CSDR_ERR_INVALID_ARG, "null argument");
        launch_kv_append(c->ctx, c->layer(layer), c->head_dim, b, dtype, a);
    });
}

int csdr_kv_cache_read_device_async(csdr_kv_cache* c, uint32_t layer, const csdr_kv_batch* batch, float* k_dev, float* v_dev) {
    return guard([&] {
        need_cache(c, layer);
        const KvBatchView b = view_of(batch);
        need_whole(4, {k_dev, v_dev});
        if (!b.n_tokens || !b.n_seqs) return;
        if (!k_dev || !v_dev) throw Error(CSDR_ERR_INVALID_ARG, "null argument");
        launch_kv_read(c->ctx, c->layer(layer), c->head_dim, b, k_dev, v_dev);
    });
}

int csdr_kv_cache_attention_device_async(csdr_kv_cache* c, uint32_t layer, const csdr_kv_batch* batch, const void* q_dev,
                                         size_t q_stride, int dtype, uint32_t q_heads, float scale, void* out_dev,
                                         size_t out_stride) {
    return guard([&] {
        need_cache(c, layer);
        const KvBatchView b = view_of(batch);
        need_dtype(dtype);
        if (!q_heads || q_heads > 65535u || q_heads % c->kv_heads)
            throw Error(CSDR_ERR_INVALID_ARG, "q_heads must be a multiple of the cache's kv_heads");
        if (!std::isfinite(scale)) throw Error(CSDR_ERR_INVALID_ARG, "scale is not finite");
        need_whole(dtype_bytes(dtype), {q_dev, out_dev});
        KvAttend a{};
        a.q = q_dev;
        a.out = out_dev;
        a.q_heads = q_heads;
        a.q_stride = row_stride(q_stride, static_cast<size_t>(q_heads) * c->head_dim, "q");
        a.out_stride = row_stride(out_stride, static_cast<size_t>(q_heads) * c->head_dim, "out");
        a.scale = scale != 0.0f ? scale : 1.0f / std::sqrt(static_cast<float>(c->head_dim));
        if (!b.n_tokens || !b.n_seqs) return;
        if (!q_dev || !out_dev) throw Error(CSDR_ERR_INVALID_ARG, "null argument");
        launch_kv_attention(c->ctx, c->layer(layer), c->head_dim, b, dtype, a, c->workspace->ptr);
    });
}

int csdr_q4_create(csdr_context* ctx, const char* format, const void* payload, size_t nbytes, uint32_t rows, uint32_t cols,
                   csdr_q4_weight** out) {
    return guard([&] {
        require_ctx(ctx);
        if (!format || !payload || !out) throw Error(CSDR_ERR_INVALID_ARG, "null argument");
        const int id = dequant_format_id(format);
        const bool q4_0 = std::strcmp(format, "q4_0") == 0, q4_k = std::strcmp(format, "q4_k") == 0;
        if (id < 0 || (!q4_0 && !q4_k)) throw Error(CSDR_ERR_UNSUPPORTED, std::string("not a 4-bit block format: ") + format);
        const uint32_t unit = q4_0 ? 32u : 256u;
        if (!rows || !cols || rows > 0x7FFFFFF0u || cols > 0x7FFFFF00u) throw Error(CSDR_ERR_INVALID_ARG, "rows or columns out of range");
        if (cols % unit) throw Error(CSDR_ERR_GEOMETRY, "columns must fall on whole blocks of the format");
        if (nbytes % (q4_0 ? 18u : 144u) || dequant_output_count(id, nbytes) != static_cast<size_t>(rows) * cols)
            throw Error(CSDR_ERR_FORMAT, "payload size does not match the shape");
        auto w = std::make_unique<csdr_q4_weight>();
        w->ctx = ctx;
        w->view.format = q4_0 ? 0 : 1;
        w->view.rows = rows;
        w->view.cols = cols;
        w->view.n_units = (cols + q4_unit_cols(w->view.format) - 1u) / q4_unit_cols(w->view.format);
        w->data = std::make_shared<DeviceBuffer>(
            static_cast<size_t>((rows + 15u) / 16u) * w->view.n_units * q4_unit_bytes(w->view.format), ctx->device);
        w->view.base = static_cast<const uint8_t*>(w->data->ptr);
        DevPtr packed = upload(ctx, payload, nbytes);
        launch_q4_relay(ctx, static_cast<const uint8_t*>(packed->ptr), w->view, static_cast<uint8_t*>(w->data->ptr));
        CSDR_CUDA(cudaStreamSynchronize(ctx->stream));
        *out = w.release();
    });
}

int csdr_q4_destroy(csdr_q4_weight* w) {
    return guard([&] {
        if (!w) return;
        cudaSetDevice(w->ctx->device);
        cudaStreamSynchronize(w->ctx->stream);
        delete w;
    });
}

int csdr_q4_matmul_device_async(csdr_context* ctx, const csdr_q4_weight* w, const void* x_dev, int x_dtype, int x_layout,
                                size_t batch, float* y_dev, int y_layout, const float* bias_dev) {
    return guard([&] {
        require_ctx(ctx);
        if (!w || !x_dev || !y_dev) throw Error(CSDR_ERR_INVALID_ARG, "null argument");
        if (w->ctx->device != ctx->device) throw Error(CSDR_ERR_INVALID_ARG, "the weight lies on another device");
        need_dtype(x_dtype);
        if ((x_layout != CSDR_LAYOUT_FEATURE_MAJOR && x_layout != CSDR_LAYOUT_TOKEN_MAJOR) ||
            (y_layout != CSDR_LAYOUT_FEATURE_MAJOR && y_layout != CSDR_LAYOUT_TOKEN_MAJOR))
            throw Error(CSDR_ERR_INVALID_ARG, "unknown dtype or layout");
        need_whole(dtype_bytes(x_dtype), {x_dev});
        need_whole(4, {y_dev, bias_dev});
        if (!batch) return;
        Q4Args a{};
        a.x = x_dev;
        a.x_dtype = x_dtype;
        a.x_token = x_layout == CSDR_LAYOUT_TOKEN_MAJOR ? w->view.cols : 1;
        a.x_col = x_layout == CSDR_LAYOUT_TOKEN_MAJOR ? 1 : batch;
        a.batch = batch;
        a.y = y_dev;
        a.y_token = y_layout == CSDR_LAYOUT_TOKEN_MAJOR ? w->view.rows : 1;
        a.y_row = y_layout == CSDR_LAYOUT_TOKEN_MAJOR ? 1 : batch;
        a.bias = bias_dev;
        launch_q4_matmul(ctx, w->view, a);
    });
}

int csdr_token_logprobs_device_async(csdr_context* ctx, const void* logits_dev, int dtype, size_t stride, size_t rows, size_t vocab,
                                     const int32_t* targets_dev, float* logprobs_dev, float* entropy_dev, uint32_t top,
                                     int32_t* top_ids_dev, float* top_logprobs_dev) {
    return guard([&] {
        require_ctx(ctx);
        need_dtype(dtype);
        if (!vocab || vocab > 0x7FFFFFFFu || rows > 0x7FFFFFFFu) throw Error(CSDR_ERR_INVALID_ARG, "rows or vocabulary out of range");
        if (top > kMaxTop) throw Error(CSDR_ERR_LIMIT, "at most 32 alternatives");
        if (top > vocab) throw Error(CSDR_ERR_INVALID_ARG, "more alternatives than the vocabulary has tokens");
        LogprobArgs a{};
        a.logits = logits_dev;
        a.stride = row_stride(stride, vocab, "logits");
        a.rows = static_cast<uint32_t>(rows);
        a.vocab = static_cast<uint32_t>(vocab);
        a.targets = targets_dev;
        a.logprob = logprobs_dev;
        a.entropy = entropy_dev;
        a.top = top;
        a.top_ids = top_ids_dev;
        a.top_logprobs = top_logprobs_dev;
        need_whole(dtype_bytes(dtype), {logits_dev});
        need_whole(4, {targets_dev, logprobs_dev, entropy_dev, top_ids_dev, top_logprobs_dev});
        if (!rows) return;
        if (!logits_dev || (logprobs_dev && !targets_dev) || (top && (!top_ids_dev || !top_logprobs_dev)))
            throw Error(CSDR_ERR_INVALID_ARG, "null argument");
        launch_logprobs(ctx, dtype, a);
    });
}

}  // extern "C"
