// The paged 8-bit key/value cache: host-side checks and the device-side addressing its kernels share.
#pragma once

#include "wl_host.h"

namespace wl {

constexpr int64_t kMaxTokens = int64_t{1} << 31;
// A launch has less than 2^32 threads along its first axis.
inline bool fits_a_launch(int64_t groups, int threads) { return groups < (int64_t{1} << 32) / threads; }

inline int check_cache(const WlKvCache* c) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return WL_EINVAL_NULL;
    if (c->type != WL_KV_INT8 && c->type != WL_KV_E4M3) return WL_EINVAL_CACHE;
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return WL_EINVAL_CACHE;
    if (c->page_tokens < 16 || c->page_tokens > 1024 || (c->page_tokens & (c->page_tokens - 1))) return WL_EINVAL_CACHE;
    if (c->pages < 1 || c->pages >= (int64_t{1} << 31) || c->layers < 1 || c->layers > 4096 || c->kv_heads < 1 ||
        c->kv_heads > 4096 || c->reserved != 0)
        return WL_EINVAL_SHAPE;
    for (const void* p : {static_cast<const void*>(c->k), static_cast<const void*>(c->v)})
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return WL_EINVAL_ALIGN;
    for (const void* p : {static_cast<const void*>(c->k_scale), static_cast<const void*>(c->v_scale)})
        if (reinterpret_cast<uintptr_t>(p) % 4 != 0) return WL_EINVAL_ALIGN;
    return WL_OK;
}

inline int check_batch(const WlKvBatch* b) {
    if (!b || !b->table || !b->cu) return WL_EINVAL_NULL;
    if (b->seqs < 1 || b->seqs > 65535 || b->table_width < 1 || b->table_width > (1 << 20) ||
        b->table_stride < b->table_width || b->tokens < 1 || b->tokens >= kMaxTokens || b->max_count < 1 ||
        b->max_count > b->tokens || b->reserved != 0)
        return WL_EINVAL_SHAPE;
    for (const void* p : {static_cast<const void*>(b->table), static_cast<const void*>(b->cu)})
        if (reinterpret_cast<uintptr_t>(p) % 4 != 0) return WL_EINVAL_ALIGN;
    return WL_OK;
}

// All bits of the bytes whose index is below n
__device__ __forceinline__ uint32_t byte_mask(int n) { return n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1u; }

// 0 that the compiler takes for a lane's own: an address with it is read by a vector load. A scalar load shares its counter
// with LDS reads and comes back out of order, so the next LDS operand would wait for it to come from memory.
__device__ __forceinline__ uint32_t lane_zero() {
    uint32_t z = 0;
    __asm__("" : "+v"(z));
    return z;
}

// Loads at a pointer that all lanes share plus a lane's 32-bit offset in bytes: the pointer is kept in scalar registers, a
// lane holds the offset alone.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
struct ScalarBase {
    const __attribute__((address_space(1))) uint8_t* p;

    __device__ __forceinline__ explicit ScalarBase(const void* at) {
        uint64_t u = reinterpret_cast<uint64_t>(at);
        __asm__("" : "+s"(u));
        p = (const __attribute__((address_space(1))) uint8_t*)u;
    }
    __device__ __forceinline__ uint4 load16(uint32_t offset) const {
        return __builtin_bit_cast(uint4, *(const __attribute__((address_space(1))) u32x4*)(p + offset));
    }
    __device__ __forceinline__ uint32_t load4(uint32_t offset) const {
        return *(const __attribute__((address_space(1))) uint32_t*)(p + offset);
    }
    __device__ __forceinline__ float load_float(uint32_t offset) const { return __builtin_bit_cast(float, load4(offset)); }
};

// One layer of the cache, as the kernels see it.
struct KvLayer {
    uint8_t* k;
    uint8_t* v;
    float* k_scale;
    float* v_scale;
    int32_t pages, kv_heads, page_tokens, page_shift;  // page_shift: log2(page_tokens)

    // Byte offset of a (page, head) block, and the index of its scale: 64 bits, a cache may be far over 4 GB.
    __device__ __forceinline__ int64_t block(int page, int head) const {
        return static_cast<int64_t>(page) * kv_heads + head;
    }
    // which page of its sequence a position is in, and where in it
    __device__ __forceinline__ int column(int pos) const { return pos >> page_shift; }
    __device__ __forceinline__ int within(int pos) const { return pos & (page_tokens - 1); }
};

inline KvLayer layer_of(const WlKvCache* c, int layer) {
    KvLayer l;
    const int64_t blocks = c->pages * c->kv_heads;
    const int64_t bytes = blocks * c->page_tokens * c->head_dim;
    l.k = static_cast<uint8_t*>(c->k) + layer * bytes;
    l.v = static_cast<uint8_t*>(c->v) + layer * bytes;
    l.k_scale = c->k_scale + layer * blocks;
    l.v_scale = c->v_scale + layer * blocks;
    l.pages = static_cast<int32_t>(c->pages);
    l.kv_heads = c->kv_heads;
    l.page_tokens = c->page_tokens;
    l.page_shift = __builtin_ctz(c->page_tokens);
    return l;
}

// The sequences of a call, as the kernels see them. Everything read from device memory is cut to its range here, so no
// content of table, cu, start or length leads an access out of the caller's arrays.
struct KvSeqs {
    const int32_t* table;
    const int32_t* cu;
    int64_t table_stride;
    int32_t tokens, seqs, table_width, max_count;

    __device__ __forceinline__ int first(int b) const { return min(max(cu[b], 0), tokens); }
    __device__ __forceinline__ int count(int b, int at) const {
        return min(max(cu[b + 1], at) - at, min(tokens - at, max_count));
    }
    // The table's entry for column `col` of sequence b, as it stands there (-1 behind the table's end); and the page that an
    // entry names, or -1. Apart, so that a kernel can ask for an entry long before it uses it.
    __device__ __forceinline__ int entry(int b, int col) const {
        return static_cast<uint32_t>(col) < static_cast<uint32_t>(table_width) ? table[b * table_stride + col] : -1;
    }
    static __device__ __forceinline__ int page_of(int entry, int pages) {
        return static_cast<uint32_t>(entry) < static_cast<uint32_t>(pages) ? entry : -1;
    }
    __device__ __forceinline__ int page(int b, int col, int pages) const { return page_of(entry(b, col), pages); }
};

inline KvSeqs seqs_of(const WlKvBatch* b) {
    return {b->table, b->cu, b->table_stride, static_cast<int32_t>(b->tokens), b->seqs, b->table_width, b->max_count};
}

}  // namespace wl
