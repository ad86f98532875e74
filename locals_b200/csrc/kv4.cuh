// The paged 4-bit key/value cache, as its kernels see it.
//
// Keys and values are MLX affine 4-bit groups of 64 (code i of a word at bits 4 i, value = scale * code + bias) in a pool
// of pages: words uint32 (pages, KVH, page, D / 8), scales and biases (pages, KVH, page, D / 64) in the activation dtype.
// A page is a multiple of 8 tokens, so that 8 tokens starting at a multiple of 8 always lie in one page, one after the
// other, on 16-byte boundaries in every array. Slot s = page * P + offset names a token's place.
#pragma once

#include <stdint.h>

namespace lq {

struct Kv4Pool {
    uint32_t* kq;
    uint16_t* ks;
    uint16_t* kb;
    uint32_t* vq;
    uint16_t* vs;
    uint16_t* vb;
    int pages, KVH, page;  // page: tokens a page
};

// Row of (page id, kv head, offset) in the pool's arrays; below 2^32 (checked by the host).
__device__ __forceinline__ uint32_t kv4_row(const Kv4Pool& p, int id, int kvh, int off) {
    return (uint32_t(id) * uint32_t(p.KVH) + uint32_t(kvh)) * uint32_t(p.page) + uint32_t(off);
}

}  // namespace lq
