// Trees of drafted tokens (wl_kv_tree) and moving the accepted ones up in the paged 8-bit cache (wl_kv_keep).
#include <algorithm>

#include "wl_kv.h"

namespace wl {
namespace {

constexpr int kTreeThreads = 256;
constexpr int kTreeKept = 4096;  // parents of a sequence that fit in LDS

// A workgroup takes a sequence, a thread a row. Up to 64 rows are a wavefront's: each takes over the mask and the parent of the
// row that it has reached, which doubles its steps every time: 2.4 to 2.6 us in a graph, whatever the tree (walked one by one, chains of 16
// and 64 take 3.8 and 8.5, trees of 64 2.9 to 3.2); behind kernels that leave nothing of its inputs in the caches it takes up to 5.
// More rows are walked from the row to its root: parents stand before their children, so the walk ends, and meets the words
// of the row's mask from the last to the first. The workgroup behind the last sequence clears the rows before the first and
// behind the last one.
__global__ __launch_bounds__(kTreeThreads) void k_kv_tree(KvSeqs s, const int32_t* __restrict__ parents,
                                                          const int32_t* __restrict__ start, uint64_t* __restrict__ tree,
                                                          int64_t words, int64_t* __restrict__ positions) {
    __shared__ int32_t kept[kTreeKept];
    const int b = blockIdx.x;
    auto clear = [&](int from, int to) {
        for (int64_t i = from * words + threadIdx.x; i < to * words; i += kTreeThreads) tree[i] = 0;
        for (int i = from + static_cast<int>(threadIdx.x); i < to; i += kTreeThreads) positions[i] = 0;
    };
    if (b == s.seqs) {
        clear(0, s.first(0));
        clear(s.first(s.seqs), s.tokens);
        return;
    }
    const int at = s.first(b), n = s.count(b, at);
    clear(at + n, min(max(s.cu[b + 1], at), s.tokens));  // rows behind max_count
    const int32_t* mine = parents + at;
    const int64_t before = start[b];
    if (n <= 64) {  // the same for all threads
        if (threadIdx.x >= 64) return;
        const int i = threadIdx.x;
        int up = i < n ? mine[i] : -1;
        if (up >= i) up = -1;
        uint32_t lo = i < 32 ? 1u << i : 0, hi = i < 32 ? 0 : 1u << (i - 32);
        while (__any(up >= 0)) {  // up: the 2^r-th ancestor; lo, hi: the row and those before that one
            const int from = max(up, 0);
            const uint32_t more_lo = __shfl(lo, from), more_hi = __shfl(hi, from);
            const int next = __shfl(up, from);
            if (up >= 0) {
                lo |= more_lo;
                hi |= more_hi;
                up = next;
            }
        }
        if (i >= n) return;
        uint64_t* row = tree + (at + i) * words;
        row[0] = static_cast<uint64_t>(hi) << 32 | lo;
        for (int64_t w = 1; w < words; w++) row[w] = 0;
        positions[at + i] = before + __popc(lo) + __popc(hi) - 1;
        return;
    }
    for (int i = threadIdx.x; i < min(n, kTreeKept); i += kTreeThreads) kept[i] = mine[i];
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kTreeThreads) {
        uint64_t* row = tree + (at + i) * words;
        int word = static_cast<int>(words) - 1, seen = 0;
        for (; word > i >> 6; word--) row[word] = 0;
        uint64_t bits = 0;
        for (int j = i;;) {
            bits |= uint64_t{1} << (j & 63);
            seen++;
            const int p = j < kTreeKept ? kept[j] : mine[j];
            if (p < 0 || p >= j) break;
            for (; word > p >> 6; word--) {
                row[word] = bits;
                bits = 0;
            }
            j = p;
        }
        for (; word >= 0; word--) {
            row[word] = bits;
            bits = 0;
        }
        positions[at + i] = before + seen - 1;
    }
}

constexpr int kKeepThreads = 256;
constexpr int kKeepChunk = 32;  // tokens that the threads hold at a time, at most
constexpr int kKeepGroups = 4;  // of V also not more than come from so many groups of 16 tokens

// One workgroup takes one kv head's K or V of a sequence on one layer, and goes through the pages that receive tokens from the
// first to the last. A token only ever moves towards the front, so what a page receives still stands where it stood when the
// page's turn comes; within a page, a chunk of tokens is read before a barrier and written behind it. Of each page first the
// largest value, which says whether its scale holds them.
// K: a thread holds 16 values of a token. V lies with the tokens innermost: the groups of 16 tokens that the chunk's tokens come
// from are read as they lie, 16 bytes a thread, and put into LDS, where a dimension's bytes stand together; a thread picks from
// there what its dimension's next 16 tokens are, and writes them with the bytes around them (moving byte by byte, every line would
// be asked for once a token, on both sides).
// Bound by latency: a token's source (offset, row number, page, scale: a chain of four loads) is looked up once a chunk, by as many
// threads as it has tokens, and a page of one chunk is read once. 5 of 16 tokens of one sequence, 10 layers of 2 heads of 256: 5.0 us
// in a graph; up to 12 of 64 of each of 64 sequences: 21 us for 8.3 MB that move, 28 MB read and 14 written of K and V together, since of V a
// dimension's next 64 tokens are all that lies side by side (with every byte moved for itself, its source looked up for it and older
// bytes rescaled one by one: 47 us). That is on pages whose scales have grown already, and bytes that are still cached: with
// 281 blocks that grow 24 us against 22 in the same run, with a cache that was written anew before 27.
template <int TYPE, int D>
__global__ __launch_bounds__(kKeepThreads) void k_kv_keep(KvLayer c, int64_t layer_bytes, int64_t layer_blocks, KvSeqs s,
                                                          const int32_t* __restrict__ start, const int32_t* __restrict__ keep) {
    struct Entry {
        const uint8_t* from;  // the token's first byte; null: not moved
        float scale;
        int32_t place;  // of V: in its row of `rows`
    };
    __shared__ Entry entries[kKeepChunk];
    __shared__ const uint8_t* groups[kKeepGroups];
    __shared__ int32_t chunk;  // how many entries it has
    __shared__ uint32_t tops[kKeepThreads / 64];
    __shared__ uint32_t rows[D][4 * kKeepGroups + 1];  // a word more: dimensions on different banks
    const int b = blockIdx.z, head = blockIdx.x >> 1;
    const bool is_v = blockIdx.x & 1;
    const int64_t from = max(start[b], 0);
    const int at = s.first(b), n = s.count(b, at);
    const int P = c.page_tokens;
    uint8_t* data = (is_v ? c.v : c.k) + blockIdx.y * layer_bytes;
    float* scales = (is_v ? c.v_scale : c.k_scale) + blockIdx.y * layer_blocks;
    auto page_at = [&](int64_t pos) {
        const int64_t col = pos >> c.page_shift;
        return col < s.table_width ? s.page(b, static_cast<int>(col), c.pages) : -1;
    };
    auto token_at = [&](int64_t block, int t) { return data + block * P * D + (is_v ? t : t * D); };
    // a thread's share of a chunk. K: values 16 k_part .. of tokens k_token + r * kTokens; V: dimension d, every kParts-th 16 tokens
    constexpr int kTokens = kKeepThreads / (D / 16), kRuns = (kKeepChunk + kTokens - 1) / kTokens;
    constexpr int kParts = kKeepThreads / D, kTargets = (kKeepChunk / 16 + 1 + kParts - 1) / kParts;
    const int k_part = threadIdx.x % (D / 16), k_token = threadIdx.x / (D / 16), d = threadIdx.x % D, part = threadIdx.x / D;
    const int first_entry = __builtin_amdgcn_readfirstlane(part);  // the same for a wavefront
    for (int64_t col = from >> c.page_shift; n > 0 && col <= (from + n - 1) >> c.page_shift; col++) {
        const int64_t page0 = col * P;
        const int page = page_at(page0);
        if (page < 0) continue;  // the same for all threads
        const int held = static_cast<int>(max(from - page0, int64_t{0}));
        const int e0 = static_cast<int>(max(page0 - from, int64_t{0})), e1 = static_cast<int>(min(page0 + P - from, static_cast<int64_t>(n)));
        const int64_t block = c.block(page, head);
        const float old = scales[block];
        uint4 k[kRuns], before[kTargets];
        // of V, entry lane % 32: what a loop over entries reads by readlane, and which are moved
        int place = 0;
        float scale = 0.0f;
        uint32_t some = 0;
        // the tokens from row e on, as they stand -> how many
        auto read = [&](int e) {
            __syncthreads();  // the chunk before has been worked on, and written
            if (threadIdx.x < 64) {
                const int i = e + threadIdx.x;
                const bool some = threadIdx.x < kKeepChunk && i < e1;
                Entry x = {nullptr, 0.0f, 0};
                if (some) {
                    const int64_t pos = from + max(keep[at + i], i);
                    const int spage = page_at(pos), t = static_cast<int>(pos & (P - 1));
                    if (spage >= 0) {
                        const int64_t sblock = c.block(spage, head);
                        x = {token_at(sblock, t), spage == page ? old : scales[sblock], t & 15};
                    }
                }
                // V: tokens of one group of 16 as the one before follow it in its place
                const uint64_t group = reinterpret_cast<uint64_t>(x.from - x.place);
                const uint32_t lo = __shfl_up(static_cast<uint32_t>(group), 1), hi = __shfl_up(static_cast<uint32_t>(group >> 32), 1);
                const bool first = threadIdx.x == 0 || (static_cast<uint64_t>(hi) << 32 | lo) != group;
                const uint64_t firsts = __ballot(first);
                const int number = __popcll(firsts & ((uint64_t{2} << threadIdx.x) - 1)) - 1;
                const int count = __popcll(__ballot(some && (!is_v || number < kKeepGroups)));
                if (threadIdx.x == 0) {
                    chunk = count;
                    for (int g = 0; g < kKeepGroups; g++) groups[g] = nullptr;
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // a wavefront's writes to LDS are in order
                if (x.from && first && number < kKeepGroups) groups[number] = x.from - x.place;
                x.place = is_v && number < kKeepGroups ? x.place + 16 * number : 0;  // within `rows`, moved or not
                if (threadIdx.x < kKeepChunk) entries[threadIdx.x] = x;
            }
            __syncthreads();
            const int count = chunk;
            if (!is_v) {
#pragma unroll
                for (int r = 0; r < kRuns; r++) {
                    const int i = k_token + r * kTokens;
                    const uint8_t* p = i < count ? entries[i].from : nullptr;
                    k[r] = p ? *reinterpret_cast<const uint4*>(p + 16 * k_part) : make_uint4(0, 0, 0, 0);
                }
            } else {
                uint4 w[D * kKeepGroups / kKeepThreads];
#pragma unroll
                for (int r = 0; r < D * kKeepGroups / kKeepThreads; r++) {
                    const int u = threadIdx.x + r * kKeepThreads, g = u % kKeepGroups;
                    const uint8_t* p = groups[g];
                    w[r] = p ? *reinterpret_cast<const uint4*>(p + u / kKeepGroups * P) : make_uint4(0, 0, 0, 0);
                }
                const int first = static_cast<int>(from + e - page0) >> 4, last = static_cast<int>(from + e + count - 1 - page0) >> 4;
#pragma unroll
                for (int r = 0; r < kTargets; r++)
                    if (first + part + r * kParts <= last)
                        before[r] = *reinterpret_cast<const uint4*>(token_at(block, 16 * (first + part + r * kParts)) + d * P);
#pragma unroll
                for (int r = 0; r < D * kKeepGroups / kKeepThreads; r++) {
                    const int u = threadIdx.x + r * kKeepThreads;
                    uint32_t* to = &rows[u / kKeepGroups][u % kKeepGroups * 4];
                    to[0] = w[r].x, to[1] = w[r].y, to[2] = w[r].z, to[3] = w[r].w;
                }
                const Entry x = entries[threadIdx.x % kKeepChunk];
                place = x.place;
                scale = x.scale;
                some = static_cast<uint32_t>(__ballot(x.from != nullptr)) & (count < 32 ? (1u << count) - 1u : ~0u);
                __syncthreads();
            }
            return __builtin_amdgcn_readfirstlane(count);
        };
        auto byte_of = [&](int i) { return static_cast<uint32_t>(reinterpret_cast<const uint8_t*>(rows[d])[__builtin_amdgcn_readlane(place, i)]); };
        auto scale_of = [&](int i) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, scale), i)); };
        uint32_t top = 0;  // magnitudes order as their bits do; infinities and NaN come out largest
        auto measure = [&](uint32_t byte, float scale) {
            top = max(top, __builtin_bit_cast(uint32_t, from_byte<TYPE>(byte & 0xFFu) * scale) & 0x7FFFFFFFu);
        };
        int count = 0;
        for (int e = e0; e < e1; e += count) {
            count = read(e);
            if (!is_v) {
#pragma unroll
                for (int r = 0; r < kRuns; r++) {
                    const int i = k_token + r * kTokens;
                    if (i >= count || !entries[i].from) continue;
                    const uint32_t w[4] = {k[r].x, k[r].y, k[r].z, k[r].w};
#pragma unroll
                    for (int j = 0; j < 16; j++) measure(w[j / 4] >> (8 * (j % 4)), entries[i].scale);
                }
            } else {
                for (int i0 = 0; i0 < count; i0 += 8 * kParts) {
                    uint32_t bytes[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) bytes[j] = byte_of(min(i0 + first_entry + j * kParts, 31));
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int i = min(i0 + first_entry + j * kParts, 31);
                        if (some >> i & 1) measure(bytes[j], scale_of(i));
                    }
                }
            }
        }
        const bool once = count == e1 - e0;  // the page's tokens are one chunk
#pragma unroll
        for (int x = 32; x; x >>= 1) top = max(top, __shfl_xor(top, x));
        if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
        __syncthreads();  // a page of one chunk has been read, and every thread has the old scale
        top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
        int shrink = 0;
        const float now = top < 0x7F800000u ? block_scale<TYPE>(__builtin_bit_cast(float, top), true, old, shrink) : __builtin_nanf("");
        const bool dead = !(now > 0.0f);  // zeros, or a NaN scale
        // byte * scale / scale rounds to the byte
        auto stays = [&](float scale) { return scale == now && now > 1.0e-30f; };
        auto moved = [&](uint32_t byte, float scale) { return dead ? 0u : to_byte<TYPE>(from_byte<TYPE>(byte & 0xFFu) * scale / now); };
        auto older = [&](uint32_t byte) { return to_byte<TYPE>(ldexpf(from_byte<TYPE>(byte & 0xFFu), -shrink)); };
        auto older4 = [&](uint32_t w) { return older(w) | older(w >> 8) << 8 | older(w >> 16) << 16 | older(w >> 24) << 24; };
        if (shrink) {  // of K all tokens before, of V those of whole groups before the first that changes
            const int units = is_v ? D * (held / 16) : held * (D / 16), per = max(held / 16, 1);
            for (int u = threadIdx.x; u < units; u += kKeepThreads) {
                uint4* p = reinterpret_cast<uint4*>(token_at(block, 0) + (is_v ? u / per * P + u % per * 16 : 16 * u));
                const uint4 w = *p;
                *p = make_uint4(older4(w.x), older4(w.y), older4(w.z), older4(w.w));
            }
        }
        for (int e = e0; e < e1; e += count) {
            if (!once) {
                count = read(e);
                __syncthreads();
            }
            const int t = static_cast<int>(from + e - page0);  // the chunk's place in the page
            if (!is_v) {
#pragma unroll
                for (int r = 0; r < kRuns; r++) {
                    const int i = k_token + r * kTokens;
                    if (i >= count || !entries[i].from) continue;
                    const float scale = entries[i].scale;
                    uint32_t w[4] = {k[r].x, k[r].y, k[r].z, k[r].w};
                    if (!stays(scale)) {
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            w[j] = moved(w[j], scale) | moved(w[j] >> 8, scale) << 8 | moved(w[j] >> 16, scale) << 16 | moved(w[j] >> 24, scale) << 24;
                    }
                    *reinterpret_cast<uint4*>(token_at(block, t + i) + 16 * k_part) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            } else {
                const int first = t >> 4, last = (t + count - 1) >> 4;
                const bool plain = __all(stays(scale) || !(some >> (threadIdx.x % kKeepChunk) & 1));
#pragma unroll
                for (int r = 0; r < kTargets; r++) {
                    const int group = first + first_entry + r * kParts;
                    if (group > last) continue;
                    uint32_t w[4] = {before[r].x, before[r].y, before[r].z, before[r].w}, bytes[16];
                    if (e == e0 && shrink && 16 * group < t) {
                        // of the words' bytes those before the first kept token
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const uint32_t mask = byte_mask(t - 16 * group - 4 * j);
                            w[j] = (older4(w[j]) & mask) | (w[j] & ~mask);
                        }
                    }
                    const int i0 = 16 * group - t;  // the entry that the group's first byte is for
#pragma unroll
                    for (int j = 0; j < 16; j++) bytes[j] = byte_of(min(max(i0 + j, 0), 31));
                    const uint32_t which = (i0 < 0 ? some << -i0 : some >> i0) & 0xFFFFu;
                    if (!plain) {
#pragma unroll
                        for (int j = 0; j < 16; j++)
                            if (which >> j & 1) bytes[j] = moved(bytes[j], scale_of(min(max(i0 + j, 0), 31)));
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t mask = bytes_of(which >> 4 * j),
                                       y = bytes[4 * j] | bytes[4 * j + 1] << 8 | bytes[4 * j + 2] << 16 | bytes[4 * j + 3] << 24;
                        w[j] = (w[j] & ~mask) | (y & mask);
                    }
                    *reinterpret_cast<uint4*>(token_at(block, 16 * group) + d * P) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
        if (threadIdx.x == 0) scales[block] = now;
    }
}

}  // namespace
}  // namespace wl

using namespace wl;

extern "C" {

int wl_kv_tree(const WlKvBatch* batch, const int32_t* parents, const int32_t* start, uint64_t* tree, int64_t words,
               int64_t* positions, void* stream) {
    if (!batch || !batch->cu || !parents || !start || !tree || !positions) return WL_EINVAL_NULL;
    WlKvBatch b = *batch;  // without a table, of which nothing is read
    b.table = b.cu;
    b.table_width = 1;
    b.table_stride = 1;
    if (const int rc = check_batch(&b)) return rc;
    if (words < (b.max_count + 63) / 64 || words >= (int64_t{1} << 31) / 64 || words * b.tokens >= (int64_t{1} << 40)) return WL_EINVAL_SHAPE;
    if (reinterpret_cast<uintptr_t>(parents) % 4 || reinterpret_cast<uintptr_t>(start) % 4 || reinterpret_cast<uintptr_t>(tree) % 8 ||
        reinterpret_cast<uintptr_t>(positions) % 8)
        return WL_EINVAL_ALIGN;
    k_kv_tree<<<b.seqs + 1, kTreeThreads, 0, static_cast<hipStream_t>(stream)>>>(seqs_of(&b), parents, start, tree, words, positions);
    return launch_status();
}

int wl_kv_keep(const WlKvCache* cache, const WlKvBatch* batch, const int32_t* start, const int32_t* keep, void* stream) {
    if (const int rc = check_cache(cache)) return rc;
    if (const int rc = check_batch(batch)) return rc;
    if (!start || !keep) return WL_EINVAL_NULL;
    if (reinterpret_cast<uintptr_t>(start) % 4 || reinterpret_cast<uintptr_t>(keep) % 4) return WL_EINVAL_ALIGN;
    const dim3 grid(2 * cache->kv_heads, cache->layers, batch->seqs);
    const KvLayer c = layer_of(cache, 0);
    const int64_t blocks = cache->pages * cache->kv_heads, bytes = blocks * cache->page_tokens * cache->head_dim;
    auto run = [&](auto type, auto dim) {
        k_kv_keep<decltype(type)::value, decltype(dim)::value>
            <<<grid, kKeepThreads, 0, static_cast<hipStream_t>(stream)>>>(c, bytes, blocks, seqs_of(batch), start, keep);
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

}  // extern "C"
