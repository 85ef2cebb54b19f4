// Attention over the paged 8-bit cache (wl_kv_attend, wl_kv_attend_masked): the entry points, and the form for few rows.
//
// At most 16 rows of a (sequence, kv head): a wavefront takes the rows and tiles of 64 tokens, all in registers, with
// v_mfma_f32_16x16x32_bf16. Row m of the first product's t-th operand is token 16 (m / 4) + 4 t + m % 4 of the tile, so a
// lane of group g (of four) holds the scores of tokens 16 g .. 16 g + 15 of row lane % 16.
// Bound by reading the cache: 64 sequences of 250 to 16000 tokens, 2 kv heads of 256 in int8, 209 MB, in 49 us (4.3 TB/s; a
// copy of 1 GiB on the same card 5.1), 131071 tokens of one in e4m3, 134 MB, in 26 us (5.2 TB/s), and 5 us for the join. Two
// wavefronts a SIMD, each with one tile on its way and one at work: one a SIMD with two tiles in its 512 registers 40 us
// where this took 34 at that stage. 512 workgroups: 256, 768 and 1024 were 7, 11 and 6% slower. One short sequence is a
// chain of loads: 777 tokens 12.7 us in a graph, of which the join takes 4.
// With a window and sinks (MASK) the tiles between them are left out of the line, so the time goes by the window: 64 sequences of up to
// 16000 tokens in a window of 4096, 130 MB, 33 us and 5 for the join (3.9 TB/s), one token of one in a window of 128 to 4096 8.5 to
// 13.9 us in a graph, whatever lies before it. A masked call may have several blocks of 16 rows, each of which goes through the tiles
// for itself: 16 drafted tokens of 16 heads on 2 of 256 behind 776, 8 blocks a head, 12 us and 4 for the join.
#include <algorithm>

#include "wl_attend.h"

namespace wl {
namespace {

constexpr int kRows = 16;
constexpr int kFewWaves = 4;
constexpr int kFewGroups = 512;  // workgroups: two a CU
constexpr int64_t kBlockTiles = 4096;

// Where the partial results of a (sequence, kv head) lie: slot first, then two slots further for each of the other pieces,
// from `next` on. pieces is 0 where there are none.
struct Pieces {
    int32_t pieces, first, next, reserved;
};

struct FewArgs : AttendArgs {
    float* partial;      // [2 * workgroups][rows][D]
    float2* partial_ml;  // [2 * workgroups][rows]: maximum (in log2) and sum
    Pieces* pieces;      // [seqs][kv heads][blocks]
    int32_t rows;        // rows of a block, at most
    int32_t blocks;      // of 16 rows, of a (sequence, kv head), at most; 1 without MASK
    int32_t whole, groups;  // how the call is cut: not at all, or over how many workgroups
};

// One wavefront's share of a block of rows of (sequence b, kv head): its running maximum, its lanes' sums and O^T.
// PAGE: a page holds whole tiles (64 tokens or more), so a tile has one page, one address and one pair of scales.
// MASK: rows see what their window, the sinks and a tree leave them.
template <int TYPE, int D, bool PAGE, bool MASK>
struct Rows {
    static constexpr int kChunks = D / 64;  // 16-byte loads of a K row, by four lanes each
    static constexpr int kDims = D / 16;    // 16-dimension blocks of V^T

    uint4 q[2 * kChunks];  // 8 bf16 each: this lane's row, dimensions 64 i + 16 g + 8 s ..
    f32x4 o[kDims];
    float m, l;
    int limit;  // tokens that this lane's row sees; of a masked call its position plus 1
    uint64_t tree;  // this lane's row's bits of a tree of up to 64

    static __device__ __forceinline__ int token_of(const AttendArgs& a, int row0) {
        return (row0 + static_cast<int>(threadIdx.x & 15)) / a.group;
    }
    // the tree's bits of 16 tokens from `first` on
    __device__ __forceinline__ uint32_t drafted(const AttendArgs& a, Seq seq, int row0, int first) const {
        if (seq.n > 64) return tree_bits(a, seq, token_of(a, row0), first);
        const int off = first - seq.begin;
        return off >= 64 || off <= -16 ? 0 : static_cast<uint32_t>(off < 0 ? tree << -off : tree >> off);
    }

    __device__ __forceinline__ void begin(const AttendArgs& a, int head, Seq seq, int row0) {
        const int lane = threadIdx.x & 63, g = lane >> 4, row = row0 + (lane & 15), token = row / a.group;
        m = -__builtin_inff();
        l = 0.0f;
        if constexpr (MASK) {
            limit = limit_of(a, seq, token);
            tree = 0;
            if (a.mask.tree && token < seq.n && seq.n <= 64) {
                tree = *reinterpret_cast<const uint64_t*>(a.mask.tree + (seq.at + token) * a.mask.tree_stride);
                if (seq.n < 64) tree &= (uint64_t{1} << seq.n) - 1;
            }
        } else {
            limit = token >= seq.n ? 0 : seq.seen(token, a.causal);
        }
#pragma unroll
        for (int i = 0; i < kDims; i++) o[i] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
        const uint16_t* p = a.q + static_cast<int64_t>(seq.at + token) * a.q_token_stride +
                            static_cast<int64_t>(head * a.group + row % a.group) * a.q_head_stride + 16 * g;
#pragma unroll
        for (int i = 0; i < 2 * kChunks; i++) {
            const uint16_t* e = p + 64 * (i / 2) + 8 * (i % 2);
            q[i] = make_uint4(0, 0, 0, 0);
            if (token < seq.n)
                q[i] = a.wide_q ? *reinterpret_cast<const uint4*>(e)
                                : make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
        }
    }

    // A tile as it is loaded: its bytes, the scales of this lane's 16 tokens, the page they are in (below 0: not there).
    struct Tile {
        uint4 k[4][kChunks], v[kDims];
        float ks, vs;
        int page;
        const uint8_t* more;  // where v[0] came from
    };
    // V's blocks that are asked for together with K, the others are when K's registers are free: with all of them at once
    // a wavefront of 256 dimensions would not fit the 256 registers of two on a SIMD.
    static constexpr int kEarly = D == 256 ? kDims / 2 : kDims;
    int kentry, ventry;  // of the page table, for the tile that is loaded next

    // Tokens [base, base + 64) of the sequence: K's tokens of a lane's four products lie in the tile's 16-token group
    // (lane % 16) / 4, V's and the scores' in group lane / 16.
    static __device__ __forceinline__ int kgroup() { return (threadIdx.x & 15) >> 2; }
    static __device__ __forceinline__ int vgroup() { return (threadIdx.x & 63) >> 4; }

    __device__ __forceinline__ void find(const AttendArgs& a, int b, int base) {
        kentry = a.s.entry(b, a.c.column(PAGE ? base : base + 16 * kgroup()));
        ventry = PAGE ? kentry : a.s.entry(b, a.c.column(base + 16 * vgroup()));
    }
    __device__ __forceinline__ void load(const AttendArgs& a, Tile& x, int head, int base) const {
        const int P = a.c.page_tokens;
        const int kpage = KvSeqs::page_of(PAGE ? __builtin_amdgcn_readfirstlane(kentry) : kentry, a.c.pages),
                  vpage = PAGE ? kpage : KvSeqs::page_of(ventry, a.c.pages);
        const int64_t block = a.c.block(max(vpage, 0), head);
        const uint8_t *k, *v;
        if constexpr (PAGE) {  // one base for the wavefront, a lane's own offsets are the same for every tile
            k = a.c.k + (block * P + a.c.within(base)) * D;
            v = a.c.v + block * P * D + a.c.within(base);
            k += static_cast<uint32_t>((16 * kgroup() + (threadIdx.x & 3)) * D + 16 * vgroup());
            v += static_cast<uint32_t>((threadIdx.x & 15) * P + 16 * vgroup());
        } else {
            k = a.c.k + (a.c.block(max(kpage, 0), head) * P + a.c.within(base + 16 * kgroup()) + (threadIdx.x & 3)) * D +
                16 * vgroup();
            v = a.c.v + block * P * D + (threadIdx.x & 15) * P + a.c.within(base + 16 * vgroup());
        }
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < kChunks; i++) x.k[t][i] = *reinterpret_cast<const uint4*>(k + 4 * t * D + 64 * i);
        x.ks = a.c.k_scale[block] * a.scale_log2;
#pragma unroll
        for (int i = 0; i < kEarly; i++) x.v[i] = *reinterpret_cast<const uint4*>(v + 16 * i * P);
        x.vs = a.c.v_scale[block];
        x.page = vpage;
        x.more = v;
    }

    __device__ __forceinline__ void add(const AttendArgs& a, Tile& x, int base, Seq seq, int row0) {
        const int length = seq.length;
        f32x4 s[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            s[j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kChunks; i++) {
                s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight_bf16<TYPE>(x.k[j][i].x, x.k[j][i].y),
                                                               __builtin_bit_cast(bf16x8, q[2 * i]), s[j], 0, 0, 0);
                s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight_bf16<TYPE>(x.k[j][i].z, x.k[j][i].w),
                                                               __builtin_bit_cast(bf16x8, q[2 * i + 1]), s[j], 0, 0, 0);
            }
        }
        if constexpr (kEarly < kDims) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = kEarly; i < kDims; i++) x.v[i] = *reinterpret_cast<const uint4*>(x.more + 16 * i * a.c.page_tokens);
        }
        const int first = base + 16 * vgroup();
        // of this lane's 16 tokens, those that count: so many, or these
        const int mine = x.page < 0 ? 0 : min(max(limit - first, 0), 16);
        uint32_t bits = 0, own = 0;
        const bool in_tree = MASK && a.mask.tree && base + kTile > seq.begin;
        if constexpr (MASK) {
            own = in_tree ? drafted(a, seq, row0, first) : 0;
            bits = x.page < 0 ? 0 : seen_bits(a, seq, limit, first, length - first, own);
        }
        auto counts = [&](int i) { return MASK ? (bits >> i & 1) != 0 : i < mine; };
        float top = m;
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                s[j][r] = counts(4 * j + r) ? s[j][r] * x.ks : -__builtin_inff();
                top = fmaxf(top, s[j][r]);
            }
        top = max_over_groups(top);
        const float safe = top == -__builtin_inff() ? 0.0f : top;  // a row that has seen no token yet
        const float shrink = exp2_fast(m - safe);
        m = top;
        l *= shrink;
        if (__any(shrink != 1.0f)) {
#pragma unroll
            for (int i = 0; i < kDims; i++) o[i] *= shrink;
        }
        uint32_t p[8];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float e[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                e[r] = exp2_fast(s[j][r] - safe);
                l += e[r];
                // a token that does not count adds 0 whatever its block's scale is (it may be NaN)
                e[r] = counts(4 * j + r) ? e[r] * x.vs : 0.0f;
            }
            p[2 * j] = pack_bf16(e[0], e[1]);
            p[2 * j + 1] = pack_bf16(e[2], e[3]);
        }
        if constexpr (MASK) {
            // the same for tokens that no row sees, before the window and in the tree (where a byte of int8 times 0 is 0)
            const int lowest = window_begin(a, seq, 0);
            if (base + kTile > length || base < lowest || (TYPE == WL_KV_E4M3 && in_tree) || __any(x.page < 0)) {
                uint32_t kept = x.page < 0 ? 0 : low_bits(length - first) & (~low_bits(lowest - first) | low_bits(a.mask.sinks - first));
                if (TYPE == WL_KV_E4M3 && in_tree) kept &= low_bits(seq.begin - first) | any_of_16(own);
                const uint32_t m0 = bytes_of(kept), m1 = bytes_of(kept >> 4), m2 = bytes_of(kept >> 8), m3 = bytes_of(kept >> 12);
#pragma unroll
                for (int i = 0; i < kDims; i++) {
                    x.v[i].x &= m0;
                    x.v[i].y &= m1;
                    x.v[i].z &= m2;
                    x.v[i].w &= m3;
                }
            }
        } else if (base + kTile > length || __any(x.page < 0)) {
            // bytes that nobody wrote may be NaN in e4m3, which a weight of 0 does not silence
            const int there = x.page < 0 ? 0 : min(max(length - first, 0), 16);
            const uint32_t m0 = byte_mask(there), m1 = byte_mask(there - 4), m2 = byte_mask(there - 8), m3 = byte_mask(there - 12);
#pragma unroll
            for (int i = 0; i < kDims; i++) {
                x.v[i].x &= m0;
                x.v[i].y &= m1;
                x.v[i].z &= m2;
                x.v[i].w &= m3;
            }
        }
        const bf16x8 p0 = __builtin_bit_cast(bf16x8, make_uint4(p[0], p[1], p[2], p[3])),
                     p1 = __builtin_bit_cast(bf16x8, make_uint4(p[4], p[5], p[6], p[7]));
#pragma unroll
        for (int i = 0; i < kDims; i++) {
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight_bf16<TYPE>(x.v[i].x, x.v[i].y), p0, o[i], 0, 0, 0);
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight_bf16<TYPE>(x.v[i].z, x.v[i].w), p1, o[i], 0, 0, 0);
        }
    }

    // Tiles t0 (which has been found), t0 + step, .. below t1, as `span` numbers them.
    __device__ __forceinline__ void tiles(const AttendArgs& a, int b, int head, Span span, int t0, int t1, int step, Seq seq,
                                          int row0) {
        for (int t = t0; t < t1; t += step) {
            Tile x;
            const int base = span.tile(t) * kTile;
            load(a, x, head, base);
            if (t + step < t1) find(a, b, span.tile(t + step) * kTile);
            add(a, x, base, seq, row0);
        }
    }
};

template <int D>
struct JoinLds {
    float o[kFewWaves][kRows][D + 4];
    float m[kFewWaves][kRows], l[kFewWaves][kRows];
    float2 row[kRows];  // maximum and sum over the wavefronts
};

// The workgroup's wavefronts over tiles [t0, t1) of the rows; the rows are finished into out, or, with
// slot >= 0, left as a partial result.
template <int TYPE, int D, bool PAGE, bool MASK>
__device__ __forceinline__ void attend_rows(const FewArgs& a, JoinLds<D>& lds, int b, Seq seq, int head, int row0, int t0,
                                            int t1, int slot) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, m16 = lane & 15;
    const int at = seq.at, n = seq.n;
    const int rows = static_cast<int>(min(static_cast<int64_t>(n) * a.group - row0, static_cast<int64_t>(kRows)));
    Rows<TYPE, D, PAGE, MASK> r;
    const Span span = MASK ? span_of<MASK>(a, seq, 0, seq.length, kTile) : Span{0, 0, 0};
    if (t0 + wave < t1) r.find(a, b, span.tile(t0 + wave) * kTile);
    r.begin(a, head, seq, row0);
    r.tiles(a, b, head, span, t0 + wave, t1, kFewWaves, seq, row0);
    r.l = sum_over_groups(r.l);
    if (lane < kRows) {
        lds.m[wave][lane] = r.m;
        lds.l[wave][lane] = r.l;
    }
    __syncthreads();
    float top = lds.m[0][m16];
#pragma unroll
    for (int w = 1; w < kFewWaves; w++) top = fmaxf(top, lds.m[w][m16]);
    const float safe = top == -__builtin_inff() ? 0.0f : top;
    if (m16 < rows) {
        const float f = exp2_fast(r.m - safe);
#pragma unroll
        for (int i = 0; i < D / 16; i++)
            *reinterpret_cast<f32x4*>(&lds.o[wave][m16][16 * i + 4 * g]) = r.o[i] * f;
    }
    if (wave == 0 && lane < kRows) {
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < kFewWaves; w++) l += lds.l[w][lane] * exp2_fast(lds.m[w][lane] - safe);
        lds.row[lane] = make_float2(top, l);
    }
    __syncthreads();
    if (slot >= 0 && static_cast<int>(threadIdx.x) < rows) a.partial_ml[slot * a.rows + threadIdx.x] = lds.row[threadIdx.x];
    for (int i = threadIdx.x; i < rows * (D / 4); i += kFewWaves * 64) {
        const int row = i / (D / 4), d = i % (D / 4) * 4;
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kFewWaves; w++) o += *reinterpret_cast<const f32x4*>(&lds.o[w][row][d]);
        if (slot >= 0) {
            *reinterpret_cast<f32x4*>(a.partial + static_cast<int64_t>(slot * a.rows + row) * D + d) = o;
        } else {
            const float l = lds.row[row].y, inv = l == 0.0f ? 0.0f : 1.0f / l;
            const int token = (row0 + row) / a.group, h = head * a.group + (row0 + row) % a.group;
            *reinterpret_cast<uint2*>(a.out + (static_cast<int64_t>(at + token) * a.q_heads + h) * D + d) =
                make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
        }
    }
}

// Calls of few rows a sequence are bound by reading the cache, so the cache is what is shared out: the tiles of all
// sequences, kv heads and blocks of 16 rows (one, but of a masked call) stand in one line, and every workgroup takes the same number of them in a row, wherever sequences
// begin and end. A block that lies in one share is finished there; of one that is cut, each share leaves a
// partial result, which k_attend_join adds up in order. A share has at most two such ends, its first and its last.
// Where every sequence's last share may stay partly empty without more workgroups than the CUs hold at once, it does
// (`pad`): a workgroup that holds an end and a beginning runs them one after the other.
struct Line {
    uint32_t each, pad;  // tiles of a share; a block takes a multiple of pad tiles of the line

    __device__ __forceinline__ uint32_t padded(uint32_t tiles) const { return (tiles + pad - 1) / pad * pad; }
};

template <bool MASK>
__device__ __forceinline__ uint32_t tiles_of(const FewArgs& a, Seq s) {
    return s.n == 0 ? 0 : max(span_of<MASK>(a, s, 0, s.length, kTile).tiles, 1);  // without a token there are still rows to write
}
// The blocks of a sequence, of all its kv heads
template <bool MASK>
__device__ __forceinline__ uint32_t blocks_of(const FewArgs& a, Seq s) {
    return MASK ? max((s.n * a.group + kRows - 1) / kRows, 1) * a.c.kv_heads : a.c.kv_heads;
}
__device__ __forceinline__ Seq seq_or_none(const FewArgs& a, int b) { return b < a.s.seqs ? a.seq(b) : Seq{0, 0, 0, 0}; }

// Every wavefront works the division out for itself; `mine`: sequence `lane`. Shares and blocks are whole
// rounds of a workgroup (a tile for each wavefront), so that only the last round of each leaves wavefronts idle.
template <bool MASK>
__device__ __forceinline__ Line line_of(const FewArgs& a, Seq mine) {
    constexpr uint32_t W = kFewWaves;
    const uint32_t groups = a.groups;
    const int lane = threadIdx.x & 63;
    auto rounds_of = [&](Seq s) { return (tiles_of<MASK>(a, s) + W - 1) / W * blocks_of<MASK>(a, s); };
    uint32_t rounds = rounds_of(mine);
    for (int b = lane + 64; b < a.s.seqs; b += 64) rounds += rounds_of(a.seq(b));
    rounds = wave_sum(rounds);
    const uint32_t each = __builtin_amdgcn_readfirstlane(max((rounds + groups - 1) / groups, 1u) * W);
    auto shares_of = [&](Seq s) { return (tiles_of<MASK>(a, s) + each - 1) / each * blocks_of<MASK>(a, s); };
    uint32_t shares = shares_of(mine);
    for (int b = lane + 64; b < a.s.seqs; b += 64) shares += shares_of(a.seq(b));
    return {each, wave_sum(shares) <= groups ? each : W};
}

template <int TYPE, int D, bool PAGE, bool MASK>
__global__ __launch_bounds__(kFewWaves * 64, 2) void k_attend_few(FewArgs a) {
    __shared__ JoinLds<D> lds;
    const int lane = threadIdx.x & 63;
    Line line = {1, 1};
    uint32_t at, end, before = 0;  // the share, and the line before sequence b
    int b = 0;
    Seq seq;
    if (a.whole) {  // a workgroup for each block
        const uint32_t blocks = MASK ? a.blocks * a.c.kv_heads : a.c.kv_heads;
        b = blockIdx.x / blocks;
        seq = a.seq_uniform(b);
        const uint32_t tiles = tiles_of<MASK>(a, seq), block = blockIdx.x % blocks;
        if (MASK && block >= blocks_of<MASK>(a, seq)) return;
        at = block * tiles;
        end = at + tiles;
    } else {
        Seq mine = seq_or_none(a, lane);
        line = line_of<MASK>(a, mine);
        at = blockIdx.x * line.each;
        end = at + line.each;
        for (;;) {
            const uint32_t own = line.padded(tiles_of<MASK>(a, mine)) * blocks_of<MASK>(a, mine), sum = wave_scan(own);
            const uint64_t past = __ballot(before + sum > at);
            if (past) {
                const int i = __builtin_amdgcn_readfirstlane(__builtin_ctzll(past));
                before += __builtin_amdgcn_readlane(sum - own, i);
                seq.at = __builtin_amdgcn_readlane(mine.at, i);
                seq.n = __builtin_amdgcn_readlane(mine.n, i);
                seq.length = __builtin_amdgcn_readlane(mine.length, i);
                seq.begin = __builtin_amdgcn_readlane(mine.begin, i);
                b += i;
                break;
            }
            before += __builtin_amdgcn_readlane(sum, 63);
            b += 64;
            if (b >= a.s.seqs) return;
            mine = seq_or_none(a, b + lane);
        }
    }
    int slot = 2 * blockIdx.x;  // of the share's first piece, where it is cut; of another one that is, the last: slot + 1
    while (at < end) {
        const uint32_t tiles = tiles_of<MASK>(a, seq), length = __builtin_amdgcn_readfirstlane(line.padded(tiles));
        if (tiles) {
            const uint32_t blocks = blocks_of<MASK>(a, seq), block = __builtin_amdgcn_readfirstlane((at - before) / length),
                           t0 = at - before - block * length;
            // a head's blocks one after the other: they read the same keys and values
            const bool some = MASK && a.blocks > 1;
            const uint32_t each = some ? max((seq.n * a.group + kRows - 1) / kRows, 1) : 1, head = some ? block / each : block,
                           row0 = (block - head * each) * kRows;
            const uint32_t t1 = min(t0 + (end - at), length), stop = min(t1, tiles);
            const bool whole = t0 == 0 && stop == tiles;
            if (t0 < stop) {
                if (slot & 1) __syncthreads();  // the piece before still reads the LDS
                attend_rows<TYPE, D, PAGE, MASK>(a, lds, b, seq, head, row0, t0, stop, whole ? -1 : slot);
            }
            if (t0 == 0 && !a.whole && threadIdx.x == 0) {
                const int rest = whole ? 0 : (tiles - stop + line.each - 1) / line.each;
                a.pieces[(b * a.c.kv_heads + head) * (MASK ? a.blocks : 1) + row0 / kRows] = {rest ? 1 + rest : 0, slot,
                                                                                              2 * (static_cast<int>(blockIdx.x) + 1), 0};
            }
            slot |= 1;
            at += t1 - t0;
            if (t1 < length || block < blocks - 1) continue;
            before += length * blocks;
        }
        if (at >= end || ++b >= a.s.seqs) break;
        seq = a.seq_uniform(b);
    }
}

// One row of one block that was cut: its pieces' results, added up in the order of its tokens over eight
// wavefronts, then those. blockIdx: (sequence, head and block, row).
constexpr int kJoinWaves = 8;
template <int D>
__global__ __launch_bounds__(kJoinWaves * 64) void k_attend_join(FewArgs a) {
    __shared__ float weight[kFewGroups];
    __shared__ float red[2][kJoinWaves];
    __shared__ float o[kJoinWaves][D];
    const int unit = blockIdx.x / a.blocks, b = unit / a.c.kv_heads, head = unit % a.c.kv_heads, row = blockIdx.y,
              row_of_all = blockIdx.x % a.blocks * kRows + row;
    const Seq seq = a.seq(b);
    if (row_of_all >= seq.n * a.group) return;
    const Pieces cut = a.pieces[blockIdx.x];
    const int pieces = cut.pieces;
    if (pieces == 0) return;
    auto slot_of = [&](int i) { return i ? cut.next + 2 * (i - 1) : cut.first; };
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    float2 part = make_float2(-__builtin_inff(), 0.0f);  // of piece threadIdx.x
    if (static_cast<int>(threadIdx.x) < pieces) part = a.partial_ml[slot_of(threadIdx.x) * a.rows + row];
    float top = part.x;
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    if (lane == 0) red[0][wave] = top;
    __syncthreads();
    for (int w = 0; w < kJoinWaves; w++) top = fmaxf(top, red[0][w]);
    const float safe = top == -__builtin_inff() ? 0.0f : top;
    const float f = exp2_fast(part.x - safe);
    if (static_cast<int>(threadIdx.x) < pieces) weight[threadIdx.x] = f;
    float l = part.y * f;
#pragma unroll
    for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d);
    if (lane == 0) red[1][wave] = l;
    __syncthreads();
    constexpr int V = D / 64;  // values of a lane
    typedef float Lane __attribute__((ext_vector_type(V)));
    Lane acc = {};
    auto values = [&](int i) {
        return *reinterpret_cast<const Lane*>(a.partial + static_cast<int64_t>(slot_of(i) * a.rows + row) * D + lane * V);
    };
    int i = wave;
    for (; i + 7 * kJoinWaves < pieces; i += 8 * kJoinWaves) {
        Lane x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = values(i + e * kJoinWaves);
#pragma unroll
        for (int e = 0; e < 8; e++) acc += x[e] * weight[i + e * kJoinWaves];
    }
    for (; i < pieces; i += kJoinWaves) acc += values(i) * weight[i];
#pragma unroll
    for (int e = 0; e < V; e++) o[wave][lane * V + e] = acc[e];
    __syncthreads();
    if (threadIdx.x >= D) return;
    float sum = 0.0f, x = 0.0f;
    for (int w = 0; w < kJoinWaves; w++) {
        sum += red[1][w];
        x += o[w][threadIdx.x];
    }
    const int token = row_of_all / a.group, h = head * a.group + row_of_all % a.group;
    const float y = sum == 0.0f ? 0.0f : x / sum;
    a.out[(static_cast<int64_t>(seq.at + token) * a.q_heads + h) * D + threadIdx.x] =
        __builtin_bit_cast(uint16_t, static_cast<__bf16>(y));
}

// How a call of few rows is cut. whole: a workgroup for each (sequence, kv head); else the line of tiles over `groups`.
struct FewPlan {
    int64_t groups;
    bool whole;
};

// Blocks of 16 rows that a (sequence, kv head) has at most, where the call takes this form; else 0. Without a mask it takes
// one block. With one, each block converts the cache's bytes for itself, where the form for many rows does that once for 256
// rows, but starts slower: two blocks are always faster here (trees over 300 to 32000 tokens of 1 to 64 sequences: 1.1 to 2.1
// times), more of them up to about 4096 tiles over all blocks (up to 2000: 1.1 to 2.4 times, around 4000: 0.8 to 1.7, around
// 8000: 0.8 to 1.3, from 16000 on mostly below 0.9; heads of 64, 128 and 256).
int64_t few_blocks(const WlKvCache* c, int q_heads, const WlKvBatch* b, int64_t max_length, const WlKvMask* mask) {
    const int64_t blocks = (static_cast<int64_t>(b->max_count) * (q_heads / c->kv_heads) + kRows - 1) / kRows;
    if (blocks == 1 || !mask) return blocks == 1;
    const int64_t items = static_cast<int64_t>(b->seqs) * c->kv_heads * blocks;
    const int64_t tiles = (longest_span(c, b, max_length, mask, b->max_count, kTile) + kTile - 1) / kTile;
    if (blocks > 2 && items * tiles > kBlockTiles) return 0;
    const int64_t line = (int64_t{b->table_width} * c->page_tokens + kTile) / kTile * items;  // counted in 31 bits
    return line < (int64_t{1} << 31) && fits_a_launch(items, kJoinWaves * 64) ? blocks : 0;
}

FewPlan few_plan(const WlKvCache* c, const WlKvBatch* b, int64_t max_length, const WlKvMask* mask, int64_t blocks) {
    const int64_t longest = longest_span(c, b, max_length, mask, b->max_count, kTile);
    const int64_t items = static_cast<int64_t>(b->seqs) * c->kv_heads * blocks;
    // Two rounds of a workgroup cost less than one and the join: 500 tokens of 1 to 256 sequences on 8 kv heads of 128 9.2 to 45.6
    // against 10.1 to 61.5 us in a graph, on 8 of 64 5.8 to 24.1 against 8.3 to 32.8, of 32 to 256 on 2 of 256 15.3 to 28.0 against
    // 16.1 to 35.0; 300 tokens of 1 to 256 of those 12.6 to 21.5 against 13.2 to 28.5. Only where 256 dimensions, more than about
    // 400 tokens and at most 16 sequences meet do they cost more (500 tokens of one 14.2 against 13.3): the rule is not made finer
    // for that. Three rounds cost more in general (700 tokens of one sequence 18.5 against 13.4).
    if (longest <= kTile * kFewWaves * 2) return {items, true};
    // no more shares than the bound says there can be: a workgroup without one still costs its start
    const int64_t each = (longest + kTile * kFewWaves - 1) / (kTile * kFewWaves);
    return {std::min<int64_t>(kFewGroups, items * each), false};
}

int32_t block_rows(const WlKvCache* c, int q_heads, const WlKvBatch* b) {
    return static_cast<int32_t>(std::min<int64_t>(static_cast<int64_t>(b->max_count) * (q_heads / c->kv_heads), kRows));
}

// The workspace of a call of few rows: two slots of partial results a workgroup, then where they are.
struct FewSpace {
    size_t ml, pieces, bytes;  // offsets, total
};
FewSpace few_space(const WlKvCache* c, int64_t rows_of_block, const WlKvBatch* b, const FewPlan& p, int64_t blocks) {
    if (p.whole) return {0, 0, 0};
    const size_t rows = static_cast<size_t>(2 * p.groups * rows_of_block);
    const size_t ml = rows * c->head_dim * sizeof(float), pieces = ml + rows * sizeof(float2);
    return {ml, (pieces + 15) / 16 * 16, (pieces + 15) / 16 * 16 + static_cast<size_t>(b->seqs) * c->kv_heads * blocks * sizeof(Pieces)};
}

int check_attend(const WlKvCache* cache, int q_heads, const WlKvBatch* batch, int64_t max_length) {
    if (const int rc = check_cache(cache)) return rc;
    if (const int rc = check_batch(batch)) return rc;
    if (q_heads < 1 || q_heads > 65535 || q_heads % cache->kv_heads != 0 || max_length < 0) return WL_EINVAL_SHAPE;
    // positions fit 31 bits, and so do the tiles of all sequences and kv heads together
    const int64_t positions = int64_t{batch->table_width} * cache->page_tokens;
    if (positions >= (int64_t{1} << 31) || (positions + kTile) / kTile * batch->seqs * cache->kv_heads >= (int64_t{1} << 31) ||
        static_cast<int64_t>(batch->max_count) * (q_heads / cache->kv_heads) >= (int64_t{1} << 30) ||
        !fits_a_launch(int64_t{batch->seqs} * cache->kv_heads, kJoinWaves * 64))
        return WL_EINVAL_SHAPE;
    return WL_OK;
}

// Whether a row of q (element strides ts, hs) lies in out's memory (dense). For each head the first row that ends behind out's
// beginning is the one that would begin before its end.
bool out_meets_q(const uint16_t* out, const uint16_t* q, int64_t ts, int64_t hs, int64_t tokens, int64_t heads, int64_t dim) {
    using wide = __int128;  // strides are the caller's: no product of them may overflow
    const wide lo = (static_cast<wide>(reinterpret_cast<uintptr_t>(out)) - static_cast<wide>(reinterpret_cast<uintptr_t>(q))) / 2,
               hi = lo + static_cast<wide>(tokens) * heads * dim;
    const wide t_end = static_cast<wide>(ts) * (tokens - 1), h_end = static_cast<wide>(hs) * (heads - 1);
    if (std::min<wide>(t_end, 0) + std::min<wide>(h_end, 0) >= hi || std::max<wide>(t_end, 0) + std::max<wide>(h_end, 0) + dim <= lo)
        return false;  // what most calls are: apart as a whole
    for (int64_t h = 0; h < heads; h++) {
        const wide off = static_cast<wide>(hs) * h + (ts < 0 ? t_end : 0), step = ts < 0 ? -ts : ts;
        const wide gap = lo - dim - off;  // rows that begin at or before off + gap end before out
        const wide t = gap < 0 ? 0 : step == 0 ? tokens : gap / step + 1;
        if (t < tokens && off + t * step < hi) return true;
    }
    return false;
}

int check_mask(const WlKvMask* m, const WlKvBatch* b) {
    if (!m) return WL_OK;
    if (m->window < 0 || m->sinks < 0) return WL_EINVAL_SHAPE;
    if (!m->tree) return WL_OK;
    if (reinterpret_cast<uintptr_t>(m->tree) % 8) return WL_EINVAL_ALIGN;
    if (m->tree_stride < (b->max_count + 63) / 64 || m->tree_stride >= (int64_t{1} << 31)) return WL_EINVAL_SHAPE;
    // a window that begins inside the tree would have to know each drafted token's own depth
    return m->window && m->window < b->max_count ? WL_EINVAL_SHAPE : WL_OK;
}
bool hides_nothing(const WlKvMask* m) { return !m || (!m->tree && m->window == 0); }

Mask device_mask(const WlKvMask* m) {
    constexpr int64_t most = 0x7FFFFFFF;  // no position is as far
    return {reinterpret_cast<const uint32_t*>(m->tree), 2 * m->tree_stride, static_cast<int32_t>(m->window ? std::min(m->window, most) : most),
            static_cast<int32_t>(std::min(m->sinks, most))};
}

// A call of either entry point; mask: null, or what it hides (of a causal call).
int attend(const WlKvCache* cache, int layer, const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride, int q_heads,
           const WlKvBatch* batch, const int32_t* length, int64_t max_length, float scale, int causal, const WlKvMask* mask,
           uint16_t* out, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check_attend(cache, q_heads, batch, max_length)) return rc;
    if (const int rc = check_mask(mask, batch)) return rc;
    if (hides_nothing(mask)) mask = nullptr;
    if (!q || !length || !out) return WL_EINVAL_NULL;
    const float scale_log2 = scale * 1.44269504088896340736f;
    if (layer < 0 || layer >= cache->layers || !(scale >= 0.0f && scale_log2 < __builtin_inff())) return WL_EINVAL_SHAPE;
    const auto qb = reinterpret_cast<uintptr_t>(q);
    if (qb % 2 || reinterpret_cast<uintptr_t>(out) % 16 || reinterpret_cast<uintptr_t>(length) % 4) return WL_EINVAL_ALIGN;
    const size_t need = wl_kv_attend_masked_workspace_bytes(cache, q_heads, batch, max_length, mask);
    if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)) return WL_EINVAL_WORKSPACE;
    const int64_t blocks = few_blocks(cache, q_heads, batch, max_length, mask);
    if (!blocks && !attend_rows_fit(cache, q_heads, batch, max_length, mask)) return WL_EINVAL_SHAPE;
    if (out_meets_q(out, q, q_token_stride, q_head_stride, batch->tokens, q_heads, cache->head_dim)) return WL_EINVAL_OVERLAP;
    FewArgs a = {};
    a.c = layer_of(cache, layer);
    a.s = seqs_of(batch);
    a.length = length;
    a.q = q;
    a.q_token_stride = q_token_stride;
    a.q_head_stride = q_head_stride;
    a.out = out;
    a.q_heads = q_heads;
    a.group = q_heads / cache->kv_heads;
    a.scale_log2 = scale_log2;
    a.causal = causal != 0;
    if (mask) a.mask = device_mask(mask);
    a.wide_q = qb % 16 == 0 && q_token_stride % 8 == 0 && q_head_stride % 8 == 0;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (!blocks) return launch_attend_rows(cache, a, batch, max_length, mask, workspace, st);
    const FewPlan plan = few_plan(cache, batch, max_length, mask, blocks);
    a.rows = block_rows(cache, q_heads, batch);
    a.blocks = static_cast<int32_t>(blocks);
    const FewSpace space = few_space(cache, a.rows, batch, plan, blocks);
    a.partial = static_cast<float*>(workspace);
    a.partial_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + space.ml);
    a.pieces = reinterpret_cast<Pieces*>(static_cast<char*>(workspace) + space.pieces);
    a.whole = plan.whole;
    a.groups = static_cast<int32_t>(std::min<int64_t>(plan.groups, kFewGroups));
    auto run = [&](auto type, auto dim, auto page) {
        constexpr int T = decltype(type)::value, D = decltype(dim)::value;
        constexpr bool P = decltype(page)::value;
        const uint32_t groups = static_cast<uint32_t>(plan.groups);
        if (mask)
            k_attend_few<T, D, P, true><<<groups, kFewWaves * 64, 0, st>>>(a);
        else
            k_attend_few<T, D, P, false><<<groups, kFewWaves * 64, 0, st>>>(a);
        if (const int rc = launch_status()) return rc;
        if (!plan.whole)
            k_attend_join<D><<<dim3(static_cast<uint32_t>(batch->seqs * cache->kv_heads * blocks), a.rows), kJoinWaves * 64, 0, st>>>(a);
        return launch_status();
    };
    auto with_page = [&](auto type, auto dim) {
        return cache->page_tokens >= kTile ? run(type, dim, std::true_type()) : run(type, dim, std::false_type());
    };
    auto with_dim = [&](auto type) {
        if (cache->head_dim == 64) return with_page(type, std::integral_constant<int, 64>());
        if (cache->head_dim == 128) return with_page(type, std::integral_constant<int, 128>());
        return with_page(type, std::integral_constant<int, 256>());
    };
    if (cache->type == WL_KV_INT8) return with_dim(std::integral_constant<int, WL_KV_INT8>());
    return with_dim(std::integral_constant<int, WL_KV_E4M3>());
}

}  // namespace
}  // namespace wl

using namespace wl;

extern "C" {

size_t wl_kv_attend_workspace_bytes(const WlKvCache* cache, int q_heads, const WlKvBatch* batch, int64_t max_length) {
    return wl_kv_attend_masked_workspace_bytes(cache, q_heads, batch, max_length, nullptr);
}

size_t wl_kv_attend_masked_workspace_bytes(const WlKvCache* cache, int q_heads, const WlKvBatch* batch, int64_t max_length,
                                           const WlKvMask* mask) {
    if (check_attend(cache, q_heads, batch, max_length) || check_mask(mask, batch)) return 0;
    if (hides_nothing(mask)) mask = nullptr;
    const int64_t blocks = few_blocks(cache, q_heads, batch, max_length, mask);
    if (!blocks) return attend_rows_workspace(cache, q_heads, batch, max_length, mask);
    return few_space(cache, block_rows(cache, q_heads, batch), batch, few_plan(cache, batch, max_length, mask, blocks), blocks).bytes;
}

int wl_kv_attend(const WlKvCache* cache, int layer, const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride,
                 int q_heads, const WlKvBatch* batch, const int32_t* length, int64_t max_length, float scale, int causal,
                 uint16_t* out, void* workspace, size_t workspace_bytes, void* stream) {
    return attend(cache, layer, q, q_token_stride, q_head_stride, q_heads, batch, length, max_length, scale, causal, nullptr, out,
                  workspace, workspace_bytes, stream);
}

int wl_kv_attend_masked(const WlKvCache* cache, int layer, const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride,
                        int q_heads, const WlKvBatch* batch, const int32_t* length, int64_t max_length, float scale,
                        const WlKvMask* mask, uint16_t* out, void* workspace, size_t workspace_bytes, void* stream) {
    return attend(cache, layer, q, q_token_stride, q_head_stride, q_heads, batch, length, max_length, scale, 1, mask, out, workspace,
                  workspace_bytes, stream);
}

}  // extern "C"
