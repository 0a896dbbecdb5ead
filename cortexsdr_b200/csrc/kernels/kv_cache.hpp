// Launchers of the paged 4-bit key/value cache (kv_cache.cu, kv_attention.cu). All asynchronous on the
// context's stream.
#pragma once

#include <cstddef>
#include <cstdint>

#include "../internal.hpp"

namespace csdr {

constexpr uint32_t kKvGroup = 64;    // values of a head that share a step and a minimum
constexpr uint32_t kKvBlock = 16;    // tokens of a block, the unit of the layout

// Where a cache's pages lie. A page holds, for each kv head, its blocks of sixteen tokens one behind the other:
//   keys     16 x head_dim / 2 bytes, a token's row after another; word (t, w) of a row, t < 4 and
//            w < head_dim / 32, holds the values 64 (w / 2) + 16 t + 8 (w % 2) + 0 .. 3 in its low half, + 4 .. 7 in its high half
//   values   8 pairs of tokens; word (g, u, x) of a pair, g < 8, u < head_dim / 64, x < 2, holds the
//            values 64 u + 8 g + 4 x + 0 .. 3 of the even token in its low half and of the odd one in its high half
//   (fp16 minimum, fp16 step in the upper half) of the keys' groups, [group][token], then of the values'
// so that a lane of the attention kernel finds what its matrix fragments take in one piece each, and a block is one
// contiguous copy. Codes of a half: codes4.cuh.
struct KvView {
    uint8_t* base = nullptr;
    uint32_t n_pages = 0, kv_heads = 0, page_shift = 0;   // tokens of a page: 1 << page_shift
    uint32_t block_bytes = 0;                             // of one block of one head
    __host__ __device__ size_t block_at(uint32_t page, uint32_t head, uint32_t token) const {
        const uint32_t per = 1u << (page_shift - 4u);
        return ((static_cast<size_t>(page) * kv_heads + head) * per + (token >> 4)) * block_bytes;
    }
};

// A ragged batch: sequence s has rows first[s] .. first[s + 1] - 1 of the operands, its last new tokens, and
// length[s] tokens with them; token p lies in page pages[s * pages_per_seq + p / page].
struct KvBatchView {
    const int32_t* first;
    const int32_t* length;
    const int32_t* pages;
    uint32_t n_seqs, n_tokens, pages_per_seq;
};

struct KvAppend {
    const void *k, *v, *q;
    void* q_out;
    size_t kv_stride, q_stride, q_out_stride;   // elements between tokens
    uint32_t q_heads;
    const double* freq;      // rotation per position of each pair; null: stored as they come
    bool q_vec, q_out_vec, kv_vec;      // rows start on 16 bytes (set by the launcher)
};
void launch_kv_append(csdr_context* ctx, const KvView& kv, uint32_t head_dim, const KvBatchView& b, int dtype, const KvAppend& a);
// The values the batch's new tokens are held as, fp32 (token, kv head, head_dim); zeros where a token has no place.
void launch_kv_read(csdr_context* ctx, const KvView& kv, uint32_t head_dim, const KvBatchView& b, float* k, float* v);

struct KvAttend {
    const void* q;
    void* out;
    size_t q_stride, out_stride;
    uint32_t q_heads;
    float scale;
};
void launch_kv_attention(csdr_context* ctx, const KvView& kv, uint32_t head_dim, const KvBatchView& b, int dtype, const KvAttend& a,
                         void* workspace);
// Zeroed once by whoever makes it; launches leave the counters at its front at zero.
size_t kv_attention_workspace(const csdr_context* ctx, uint32_t head_dim);

}  // namespace csdr

struct csdr_kv_cache {
    csdr_context* ctx = nullptr;
    uint32_t n_layers = 0, n_pages = 0, page_tokens = 0, kv_heads = 0, head_dim = 0;
    size_t layer_bytes = 0;
    csdr::KvView view;          // of layer 0
    csdr::DevPtr data, freq, workspace;
    csdr::KvView layer(uint32_t l) const {
        csdr::KvView v = view;
        v.base += static_cast<size_t>(l) * layer_bytes;
        return v;
    }
};
