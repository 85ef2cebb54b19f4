// Writing into the paged 8-bit cache (wl_kv_append) and moving its pages (wl_kv_copy).
#include <algorithm>
#include <vector>

#include "wl_kv.h"

namespace wl {
namespace {

constexpr int kAppendThreads = 256;

// x / s of bf16 values as a byte, rounded to nearest even, for a scale that block_scale gave.
// The quotient is taken as x times 1 / s and then cut to 18 significant bits: with 8 significant bits each, x / s is a tie
// between two bytes exactly, or at least 2^-16 (relative) away from one, and the product is off by less than 2^-22, so the
// cut brings every tie back to itself and moves nothing else across one. A scale whose reciprocal leaves fp32 is divided by.
template <int TYPE>
struct Quantizer {
    float scale, inverse;
    bool dead, tiny;  // nothing but zeros, or a NaN scale: every byte is 0

    __device__ __forceinline__ explicit Quantizer(float s)
        : scale(s), inverse(1.0f / s), dead(!(s > 0.0f)), tiny(s < 1.0e-30f) {}
    __device__ __forceinline__ uint32_t operator()(uint32_t bits) const {
        const float x = bf16_to_float(bits);
        const uint32_t y = __builtin_bit_cast(uint32_t, x * inverse);
        float q = __builtin_bit_cast(float, (y + 0x20u) & ~0x3Fu);
        if (tiny) q = x / scale;
        return dead ? 0u : to_byte<TYPE>(q);
    }
    // a pair of bf16 in one word -> two bytes
    __device__ __forceinline__ uint32_t pair(uint32_t two) const { return (*this)(two & 0xFFFFu) | (*this)(two >> 16) << 8; }
};

__device__ __forceinline__ uint32_t top_of(uint32_t two, uint32_t top) {
    return max(top, max(two & 0x7FFFu, (two >> 16) & 0x7FFFu));
}

// One workgroup writes one block: a page of a sequence, one kv head, K or V (blockIdx.y's low bit), so the block's scale
// and its older bytes have one writer. Two passes over the block's new rows: their largest magnitude, then the bytes; a
// thread keeps what it read in the first one (all of it, up to 16384 new values). K's bytes lie as the rows do, 16 values of
// a token to a thread. V's lie with the tokens innermost: a thread takes two neighbouring values of 16 tokens, its loads run
// along the rows over the lanes, and it writes 16 bytes for each value; where those 16 tokens are not all new, the bytes
// there are read with them. Bound by latency: a prompt has one such workgroup for each CU or two, a step's single tokens less.
// One token of 64 sequences, 2 heads of 256: 6.0 us; 4096 tokens: 9.4 us (12.6 MB, 1.3 TB/s); with the rows read again for
// the second pass and divisions in place of the reciprocal: 14.3. Larger pages leave CUs without a workgroup: 4096 tokens take 14,
// 26, 50 and 97 us on pages of 128, 256, 512 and 1024.
template <int TYPE, int D, bool WIDE>
__global__ __launch_bounds__(kAppendThreads) void k_kv_append(KvLayer c, KvSeqs s, const int32_t* __restrict__ start,
                                                              const uint16_t* __restrict__ kx, int64_t k_ts, int64_t k_hs,
                                                              const uint16_t* __restrict__ vx, int64_t v_ts,
                                                              int64_t v_hs) {
    __shared__ uint32_t tops[kAppendThreads / 64];
    const int b = blockIdx.z, head = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    const int at = s.first(b), n = s.count(b, at);
    const int64_t from = max(start[b], 0), end = from + n;
    const int P = c.page_tokens;
    const int64_t col = c.column(static_cast<int>(from)) + static_cast<int64_t>(blockIdx.x), page0 = col * P;
    if (page0 >= end) return;
    const int page = col < s.table_width ? s.page(b, static_cast<int>(col), c.pages) : -1;
    if (page < 0) return;
    const int held = static_cast<int>(max(from - page0, int64_t{0}));
    const int stop = static_cast<int>(min(end - page0, static_cast<int64_t>(P)));  // tokens [held, stop) are new
    const int64_t ts = is_v ? v_ts : k_ts;
    // row of token t (in the page): at + (page0 + t - from)
    const uint16_t* __restrict__ x = (is_v ? vx + head * v_hs : kx + head * k_hs) + (at + (page0 - from)) * ts;
    const int64_t block = c.block(page, head);
    uint8_t* __restrict__ out = (is_v ? c.v : c.k) + block * P * D;
    float* scale = (is_v ? c.v_scale : c.k_scale) + block;
    const float old = *scale;

    // K: unit i is 16 values of token held + i / (D / 16). V: unit i is two values of the 16 tokens from 16 (i / (D / 2)).
    const int k_units = (stop - held) * (D / 16), g_new = held / 16, g_end = (stop + 15) / 16,
              v_units = (g_end - g_new) * (D / 2);
    auto read_k = [&](int i, uint32_t (&w)[8]) {
        const uint16_t* row = x + (held + i / (D / 16)) * ts + i % (D / 16) * 16;
        if constexpr (WIDE) {
            const uint4 lo = *reinterpret_cast<const uint4*>(row), hi = *reinterpret_cast<const uint4*>(row + 8);
            w[0] = lo.x, w[1] = lo.y, w[2] = lo.z, w[3] = lo.w, w[4] = hi.x, w[5] = hi.y, w[6] = hi.z, w[7] = hi.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = row[2 * j] | static_cast<uint32_t>(row[2 * j + 1]) << 16;
        }
    };
    auto read_v = [&](int i, uint32_t (&w)[16]) {
        const int t0 = (g_new + i / (D / 2)) * 16, d = i % (D / 2) * 2;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const int t = t0 + j;
            w[j] = 0;
            if (t < held || t >= stop) continue;
            const uint16_t* e = x + t * ts + d;
            if constexpr (WIDE)
                w[j] = *reinterpret_cast<const uint32_t*>(e);
            else
                w[j] = e[0] | static_cast<uint32_t>(e[1]) << 16;
        }
    };

    // what stands in V's bytes where a unit's 16 tokens are not all new
    auto read_old = [&](int i, uint4 (&w)[2]) {
        const int t0 = (g_new + i / (D / 2)) * 16, d = i % (D / 2) * 2;
        if (t0 >= held && t0 + 16 <= stop) return;
#pragma unroll
        for (int e = 0; e < 2; e++) w[e] = *reinterpret_cast<const uint4*>(out + (d + e) * P + t0);
    };

    // the largest magnitude, as bits (bf16 magnitudes order as their bits do; infinities and NaN come out largest)
    constexpr int kKeepK = 4, kKeepV = 2;
    uint32_t top = 0, kept[32];
    uint32_t(&kk)[kKeepK][8] = reinterpret_cast<uint32_t(&)[kKeepK][8]>(kept);
    uint32_t(&vv)[kKeepV][16] = reinterpret_cast<uint32_t(&)[kKeepV][16]>(kept);
    uint4 was[kKeepV][2] = {};
    if (!is_v) {
#pragma unroll
        for (int r = 0; r < kKeepK; r++) {
            const int i = threadIdx.x + r * kAppendThreads;
            if (i < k_units) read_k(i, kk[r]);
        }
#pragma unroll
        for (int r = 0; r < kKeepK; r++)
            if (static_cast<int>(threadIdx.x) + r * kAppendThreads < k_units)
#pragma unroll
                for (int j = 0; j < 8; j++) top = top_of(kk[r][j], top);
        for (int i = threadIdx.x + kKeepK * kAppendThreads; i < k_units; i += kAppendThreads) {
            uint32_t w[8];
            read_k(i, w);
#pragma unroll
            for (int j = 0; j < 8; j++) top = top_of(w[j], top);
        }
    } else {
#pragma unroll
        for (int r = 0; r < kKeepV; r++) {
            const int i = threadIdx.x + r * kAppendThreads;
            if (i < v_units) {
                read_v(i, vv[r]);
                read_old(i, was[r]);
            }
        }
#pragma unroll
        for (int r = 0; r < kKeepV; r++)
            if (static_cast<int>(threadIdx.x) + r * kAppendThreads < v_units)
#pragma unroll
                for (int j = 0; j < 16; j++) top = top_of(vv[r][j], top);
        for (int i = threadIdx.x + kKeepV * kAppendThreads; i < v_units; i += kAppendThreads) {
            uint32_t w[16];
            read_v(i, w);
#pragma unroll
            for (int j = 0; j < 16; j++) top = top_of(w[j], top);
        }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) top = max(top, __shfl_xor(top, d));
    if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
    __syncthreads();
    top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));

    int shrink = 0;
    const float now =
        top < 0x7F80u ? block_scale<TYPE>(bf16_to_float(top), held > 0, old, shrink) : __builtin_nanf("");
    const Quantizer<TYPE> quantize(now);
    auto older = [&](uint32_t byte) { return to_byte<TYPE>(ldexpf(from_byte<TYPE>(byte), -shrink)); };
    auto older4 = [&](uint32_t w) {
        return older(w & 0xFFu) | older(w >> 8 & 0xFFu) << 8 | older(w >> 16 & 0xFFu) << 16 | older(w >> 24) << 24;
    };
    if (threadIdx.x == 0) *scale = now;

    if (!is_v) {
        auto write_k = [&](int i, const uint32_t (&w)[8]) {
            uint32_t y[4];
#pragma unroll
            for (int j = 0; j < 4; j++) y[j] = quantize.pair(w[2 * j]) | quantize.pair(w[2 * j + 1]) << 16;
            *reinterpret_cast<uint4*>(out + (held + i / (D / 16)) * D + i % (D / 16) * 16) = make_uint4(y[0], y[1], y[2], y[3]);
        };
#pragma unroll
        for (int r = 0; r < kKeepK; r++) {
            const int i = threadIdx.x + r * kAppendThreads;
            if (i < k_units) write_k(i, kk[r]);
        }
        for (int i = threadIdx.x + kKeepK * kAppendThreads; i < k_units; i += kAppendThreads) {
            uint32_t w[8];
            read_k(i, w);
            write_k(i, w);
        }
        if (shrink)
            for (int i = threadIdx.x; i < held * (D / 4); i += kAppendThreads)
                reinterpret_cast<uint32_t*>(out)[i] = older4(reinterpret_cast<uint32_t*>(out)[i]);
        return;
    }
    auto write_v = [&](int i, const uint32_t (&w)[16], const uint4 (&before)[2]) {
        const int t0 = (g_new + i / (D / 2)) * 16, d = i % (D / 2) * 2;
        const bool mixed = t0 < held || t0 + 16 > stop;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            uint4* to = reinterpret_cast<uint4*>(out + (d + e) * P + t0);
            uint32_t y[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                y[j] = quantize(w[4 * j] >> (16 * e) & 0xFFFFu) | quantize(w[4 * j + 1] >> (16 * e) & 0xFFFFu) << 8 |
                       quantize(w[4 * j + 2] >> (16 * e) & 0xFFFFu) << 16 | quantize(w[4 * j + 3] >> (16 * e) & 0xFFFFu) << 24;
            if (mixed) {
                const uint32_t o[4] = {before[e].x, before[e].y, before[e].z, before[e].w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    // bytes of this word below `held` are older, those from `stop` on nobody's
                    const uint32_t low = byte_mask(held - t0 - 4 * j), high = ~byte_mask(stop - t0 - 4 * j);
                    y[j] = ((shrink ? older4(o[j]) : o[j]) & low) | (o[j] & high) | (y[j] & ~(low | high));
                }
            }
            *to = make_uint4(y[0], y[1], y[2], y[3]);
        }
    };
#pragma unroll
    for (int r = 0; r < kKeepV; r++) {
        const int i = threadIdx.x + r * kAppendThreads;
        if (i < v_units) write_v(i, vv[r], was[r]);
    }
    for (int i = threadIdx.x + kKeepV * kAppendThreads; i < v_units; i += kAppendThreads) {
        uint32_t w[16];
        uint4 before[2] = {};
        read_v(i, w);
        read_old(i, before);
        write_v(i, w, before);
    }
    if (shrink)  // the groups of 16 tokens before the first that changes
        for (int i = threadIdx.x; i < D * g_new * 4; i += kAppendThreads) {
            uint32_t* w = reinterpret_cast<uint32_t*>(out + i / (4 * g_new) * P) + i % (4 * g_new);
            *w = older4(*w);
        }
}

template <int TYPE, int D>
void launch_append(bool wide, dim3 grid, hipStream_t stream, const KvLayer& c, const KvSeqs& s, const int32_t* start,
                   const uint16_t* k, int64_t k_ts, int64_t k_hs, const uint16_t* v, int64_t v_ts, int64_t v_hs) {
    if (wide)
        k_kv_append<TYPE, D, true><<<grid, kAppendThreads, 0, stream>>>(c, s, start, k, k_ts, k_hs, v, v_ts, v_hs);
    else
        k_kv_append<TYPE, D, false><<<grid, kAppendThreads, 0, stream>>>(c, s, start, k, k_ts, k_hs, v, v_ts, v_hs);
}

// Page copies: the pairs of one launch travel in its arguments, so nothing is uploaded and a graph keeps them.
constexpr int kCopyPairs = 480;  // 3840 of the 4096 bytes that arguments may take
constexpr int kCopyThreads = 256;
constexpr int kCopyChunk = kCopyThreads * 16 * 4;  // bytes of one workgroup: four 16-byte loads a thread in flight

struct CopyPairs {
    int32_t src[kCopyPairs], dst[kCopyPairs];
};

// Bound by reading and writing: 900 pages of 4 layers, 472 MB read and written, 99 us (4.75 TB/s); 16 of 10 layers, 21 MB, 4.7 us.
// blockIdx: (chunk of the page's K then V bytes, pair, layer).
__global__ __launch_bounds__(kCopyThreads) void k_kv_copy(uint8_t* k, uint8_t* v, float* k_scale, float* v_scale,
                                                          int64_t pages, int kv_heads, int64_t page_bytes, int chunks,
                                                          CopyPairs pairs) {
    const int64_t layer = blockIdx.z, src = layer * pages + pairs.src[blockIdx.y],
                  dst = layer * pages + pairs.dst[blockIdx.y];
    const bool is_v = static_cast<int>(blockIdx.x) >= chunks;
    const int64_t at = static_cast<int64_t>(blockIdx.x - (is_v ? chunks : 0)) * kCopyChunk + threadIdx.x * 16;
    constexpr int kStep = kCopyThreads * 16;
    const uint8_t* from = (is_v ? v : k) + src * page_bytes + at;
    uint8_t* to = (is_v ? v : k) + dst * page_bytes + at;
    if (at + 3 * kStep < page_bytes) {
        u32x4 w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = *reinterpret_cast<const u32x4*>(from + i * kStep);
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<u32x4*>(to + i * kStep) = w[i];
    } else {
        for (int i = 0; at + i * kStep < page_bytes; i++)
            *reinterpret_cast<u32x4*>(to + i * kStep) = *reinterpret_cast<const u32x4*>(from + i * kStep);
    }
    if (blockIdx.x == 0)
        for (int h = threadIdx.x; h < kv_heads; h += kCopyThreads) {
            k_scale[dst * kv_heads + h] = k_scale[src * kv_heads + h];
            v_scale[dst * kv_heads + h] = v_scale[src * kv_heads + h];
        }
}

int check_copies(const WlKvCache* cache, const int32_t* src, const int32_t* dst, int64_t n) {
    for (int64_t i = 0; i < n; i++)
        if (src[i] < 0 || src[i] >= cache->pages || dst[i] < 0 || dst[i] >= cache->pages) return WL_EINVAL_PAGES;
    std::vector<int32_t> to(dst, dst + n);
    std::sort(to.begin(), to.end());
    if (std::adjacent_find(to.begin(), to.end()) != to.end()) return WL_EINVAL_PAGES;
    for (int64_t i = 0; i < n; i++)
        if (std::binary_search(to.begin(), to.end(), src[i])) return WL_EINVAL_PAGES;
    return WL_OK;
}

}  // namespace
}  // namespace wl

using namespace wl;

extern "C" {

int wl_kv_check(const WlKvCache* cache) { return check_cache(cache); }

int wl_kv_append(const WlKvCache* cache, int layer, const uint16_t* k, int64_t k_token_stride, int64_t k_head_stride,
                 const uint16_t* v, int64_t v_token_stride, int64_t v_head_stride, const WlKvBatch* batch,
                 const int32_t* start, void* stream) {
    if (const int rc = check_cache(cache)) return rc;
    if (const int rc = check_batch(batch)) return rc;
    if (!k || !v || !start) return WL_EINVAL_NULL;
    if (layer < 0 || layer >= cache->layers) return WL_EINVAL_SHAPE;
    const auto kb = reinterpret_cast<uintptr_t>(k), vb = reinterpret_cast<uintptr_t>(v);
    if (kb % 2 || vb % 2 || reinterpret_cast<uintptr_t>(start) % 4) return WL_EINVAL_ALIGN;
    // 16-byte loads of whole rows, where every row starts on 16 bytes; else one value at a time
    const bool wide = kb % 16 == 0 && vb % 16 == 0 && k_token_stride % 8 == 0 && k_head_stride % 8 == 0 &&
                      v_token_stride % 8 == 0 && v_head_stride % 8 == 0;
    const int P = cache->page_tokens;
    // a sequence's rows touch at most this many pages: one more than fill, where they begin inside one
    const int64_t touched = (int64_t{batch->max_count} + P - 2) / P + 1;
    if (!fits_a_launch(touched, kAppendThreads)) return WL_EINVAL_SHAPE;
    const dim3 grid(static_cast<uint32_t>(touched), 2 * cache->kv_heads, batch->seqs);
    const KvLayer c = layer_of(cache, layer);
    const KvSeqs s = seqs_of(batch);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    auto run = [&](auto type, auto dim) {
        launch_append<decltype(type)::value, decltype(dim)::value>(wide, grid, st, c, s, start, k, k_token_stride,
                                                                   k_head_stride, v, v_token_stride, v_head_stride);
    };
    auto with_dim = [&](auto type) {
        if (cache->head_dim == 64)
            run(type, std::integral_constant<int, 64>());
        else if (cache->head_dim == 128)
            run(type, std::integral_constant<int, 128>());
        else
            run(type, std::integral_constant<int, 256>());
    };
    if (cache->type == WL_KV_INT8)
        with_dim(std::integral_constant<int, WL_KV_INT8>());
    else
        with_dim(std::integral_constant<int, WL_KV_E4M3>());
    return launch_status();
}

int wl_kv_copy(const WlKvCache* cache, const int32_t* src_host, const int32_t* dst_host, int64_t n, void* stream) {
    if (const int rc = check_cache(cache)) return rc;
    if (n < 0 || n > cache->pages) return WL_EINVAL_SHAPE;
    if (n == 0) return WL_OK;
    if (!src_host || !dst_host) return WL_EINVAL_NULL;
    try {
        if (const int rc = check_copies(cache, src_host, dst_host, n)) return rc;
    } catch (...) {
        return static_cast<int>(hipErrorOutOfMemory);
    }
    const int64_t page_bytes = static_cast<int64_t>(cache->kv_heads) * cache->page_tokens * cache->head_dim;
    const int chunks = static_cast<int>((page_bytes + kCopyChunk - 1) / kCopyChunk);
    for (int64_t i = 0; i < n; i += kCopyPairs) {
        const int m = static_cast<int>(std::min<int64_t>(kCopyPairs, n - i));
        CopyPairs pairs;
        std::copy(src_host + i, src_host + i + m, pairs.src);
        std::copy(dst_host + i, dst_host + i + m, pairs.dst);
        k_kv_copy<<<dim3(2 * chunks, m, cache->layers), kCopyThreads, 0, static_cast<hipStream_t>(stream)>>>(
            static_cast<uint8_t*>(cache->k), static_cast<uint8_t*>(cache->v), cache->k_scale, cache->v_scale,
            cache->pages, cache->kv_heads, page_bytes, chunks, pairs);
        if (const int rc = launch_status()) return rc;
    }
    return WL_OK;
}

}  // extern "C"
