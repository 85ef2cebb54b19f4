// Attention over the paged 8-bit cache for more than 16 rows of a (sequence, kv head): prompts, chunks of them, drafts.
//
// A workgroup takes 256 rows, a wavefront 32 of them (v_mfma_f32_32x32x16_bf16), and goes through the cache in tiles of
// 8192 / D tokens. The workgroup turns a tile's bytes into bf16 once, into LDS, in the order in which the products take
// them (16 bytes a lane, 1 KB a k-step, so every read is a straight run over the lanes): each of K's and V's values is
// converted by one of eight wavefronts and used by all. LDS holds a ring of four tiles: while one is multiplied, the
// bytes of the tile two ahead are on their way in registers, and are converted into its place; a barrier stands behind every
// second tile (behind every one: 2% slower).
// With a window, sinks or a tree of drafts (MASK) a row tile goes through the tiles that some row of it sees, a wavefront through the
// parts that some row of its own sees, and of these just those that not all rows see whole are masked (4096 tokens behind as many in a
// window of 1024, 16 heads of 256: 87 to 91 us, 790 to 760 TFLOP/s of what the rows see).
// Token 16 h + i of a 32-token part is row 8 (i / 4) + 4 h + i % 4 of the first product, so a lane of half h holds the
// scores of tokens 16 h .. 16 h + 15 of row lane % 32, which is how the second product takes the weights.
// The running maximum is moved only when a score exceeds it by 2^8 (the weights stay below 2^8, fp32 sums hold them): the
// multiplication of a wavefront's 32 x D sums by the change is the dearest step of the softmax, and becomes rare.
// Bound by what a wavefront does between its products: 4096 tokens of 16 heads of 256 on 2 kv heads take 185 to 200 us (the
// card in hand), 740 to 690 TFLOP/s where a large product of matrices reaches 1213; 32 on 8 heads of 128 158 to 177 us, 870 to
// 780; 32 on 8 of 64 111 us, 620. The matrix core is busy half of the time, the rest is softmax and conversion, of which two
// wavefronts a SIMD hide some behind each other's products: more wavefronts, or two tiles in flight in one, have no registers with
// 256 dimensions (192 of 256 hold q and the sums; 64 rows a wavefront of 512 registers spill 500); with 128 and 64, where 188 and
// 142 are used, two in flight would fit and have not been built. 16 rows a tile straight from registers, as the form for few rows
// has it, took 435 us, every wavefront converting all bytes for itself. Bytes copied into LDS by the loads themselves and converted
// from there: 240 against 225 us at that stage, since LDS reads then wait for the copies.
#include <algorithm>

#include "wl_attend.h"

namespace wl {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWaves = 8;
constexpr int kThreads = kWaves * 64;
constexpr int kGroupRows = kWaves * 32;
constexpr int kRing = 4;  // tiles in LDS: two are multiplied between barriers, two are filled
constexpr int kMaxPieces = 16;
// Of a masked call with so few (row tile, kv head)s that 16 pieces of each leave CUs idle, as a drafted tree behind a long cache
// (64 drafted tokens of 16 heads of 256 behind 32000: 160 us with 16 pieces, 77 with 64, where each of 256 workgroups multiplies for
// 35 us and then writes its partial results, 67 MB together, that the second kernel reads again: 13 and 17 us).
constexpr int kMaxMaskedPieces = 64;
constexpr int kCus = 256;
constexpr int64_t kPartialBytes = 256 << 20;  // for partial results, at most
constexpr float kSlack = 8.0f;  // log2: how far a score may lie above the running maximum

struct RowsArgs : AttendArgs {
    float* partial;      // [pieces][tokens][q_heads][D]
    float2* partial_ml;  // [pieces][tokens][q_heads]: maximum (in log2) and sum
    int32_t* each;       // tiles that a piece has at most, as the first kernel found it for the second
    int32_t row_tiles;   // of 256 rows, in a sequence, at most
    int32_t pieces;      // a row tile's cache is cut into at most this many
    int32_t few_tiles;   // less than 2 kCus (row tile, kv head)s
};

// What a part of 16 tokens needs beside its bytes. V's scale goes into the exponent, so that a weight comes out of its exp2
// with the scale on it and the sum of the weights takes it off once for all 16: a multiplication less for each weight. Not so
// a scale that would push the weights out of fp32's range on the way (or is 0 or NaN): `rest` is that scale, and else 1.
struct Part {
    float ks;       // K's scale with the softmax's scale and log2 e
    float log2_vs;  // log2 of what V's scale puts into the exponent
    float inverse;  // 1 / that
    float rest;
};

template <int D>
struct Shape {
    static constexpr int kTokens = 8192 / D;     // of a tile
    static constexpr int kParts = kTokens / 16;  // scales apart
    static constexpr int kSubs = kTokens / 32;   // of the first product's rows
    static constexpr int kSteps = D / 16;        // k-steps of the first product
    static constexpr int kBlocks = D / 32;       // of V's dimensions
    // Swizzles of a k-step's 64 slots of 16 bytes: 16 lanes that write together fill 16 slots in a row's worth of banks,
    // whichever k-steps those belong to. Four different ones for K: a reader keeps their addresses.
    static __device__ __forceinline__ constexpr int k_swizzle(int step) { return 4 * (step & 3); }
    static __device__ __forceinline__ constexpr int v_swizzle(int part) { return part * (16 / kParts); }
};

template <int D>
struct Lds {
    uint4 k[kRing][Shape<D>::kSubs * Shape<D>::kSteps][64];
    uint4 v[kRing][Shape<D>::kBlocks * Shape<D>::kSubs * 2][64];
    Part part[kRing][Shape<D>::kParts];
    int count[kRing][Shape<D>::kParts];  // tokens that are there; with MASK as bits
};

// One thread's share of a tile on its way: 16 values of one token of K, 16 tokens of one dimension of V. PAGE: a page holds
// whole tiles, so a tile has one page and one pair of scales, all threads share its address, and the registers that other
// tiles need for theirs are scalar ones (with 256 dimensions a wavefront has none to spare).
template <int TYPE, int D, bool PAGE, bool MASK>
struct Stage {
    using S = Shape<D>;
    uint4 k, v;
    float ks, vs;
    int kentry, ventry;  // of the page table, for the tile that is loaded next
    int count;

    // 16 lanes take 4 tokens by 64 values
    static __device__ __forceinline__ int k_token() { return (threadIdx.x >> 4) / (D / 64) * 4 + ((threadIdx.x >> 2) & 3); }
    static __device__ __forceinline__ int k_chunk() { return (threadIdx.x >> 4) % (D / 64) * 4 + (threadIdx.x & 3); }
    static __device__ __forceinline__ int v_dim() { return threadIdx.x / S::kParts; }
    static __device__ __forceinline__ int v_part() { return threadIdx.x % S::kParts; }

    __device__ __forceinline__ void find(const AttendArgs& a, int b, int base) {
        if constexpr (PAGE) {
            const int col = a.c.column(base);  // uniform, but read by a vector load: see lane_zero()
            kentry = col < a.s.table_width ? static_cast<int>(ScalarBase(a.s.table + b * a.s.table_stride + col).load4(lane_zero())) : -1;
        } else {
            kentry = a.s.entry(b, a.c.column(base + k_token()));
        }
        ventry = PAGE ? kentry : a.s.entry(b, a.c.column(base + 16 * v_part()));
    }
    __device__ __forceinline__ void load(const AttendArgs& a, int head, int base, int length) {
        const int P = a.c.page_tokens;
        const int kpage = KvSeqs::page_of(PAGE ? __builtin_amdgcn_readfirstlane(kentry) : kentry, a.c.pages),
                  vpage = PAGE ? kpage : KvSeqs::page_of(ventry, a.c.pages);
        const int64_t kb = a.c.block(max(kpage, 0), head), vb = a.c.block(max(vpage, 0), head);
        if constexpr (PAGE) {
            k = ScalarBase(a.c.k + (kb * P + a.c.within(base)) * D).load16(k_token() * D + 16 * k_chunk());
            v = ScalarBase(a.c.v + vb * P * D + a.c.within(base)).load16(v_dim() * P + 16 * v_part());
            count = vpage < 0 ? 0 : length - base;  // of the tile
            ks = ScalarBase(a.c.k_scale + kb).load_float(lane_zero());
            vs = ScalarBase(a.c.v_scale + vb).load_float(lane_zero());
        } else {
            k = *reinterpret_cast<const uint4*>(a.c.k + (kb * P + a.c.within(base + k_token())) * D + 16 * k_chunk());
            v = *reinterpret_cast<const uint4*>(a.c.v + vb * P * D + v_dim() * P + a.c.within(base + 16 * v_part()));
            count = vpage < 0 ? 0 : length - base;
            if (threadIdx.x < S::kParts) {
                ks = a.c.k_scale[vb];
                vs = a.c.v_scale[vb];
            }
        }
    }
    // The tile at `base`, of the workgroup's rows from row0 on. hidden_from, hidden_to: no row sees the tokens between, counted from the
    // sequence's end
    __device__ __forceinline__ void store(const AttendArgs& a, Lds<D>& lds, int buffer, int base, Seq seq, int row0, int hidden_from,
                                          int hidden_to) const {
        const int t = k_token(), step = k_chunk(), i = t & 15;
        const int row = 8 * (i >> 2) + 4 * ((t >> 4) & 1) + (i & 3);
        uint4* to = lds.k[buffer][(t >> 5) * S::kSteps + step];
        const int sw = S::k_swizzle(step);
        to[row ^ sw] = __builtin_bit_cast(uint4, eight_bf16<TYPE>(k.x, k.y));
        to[(32 + row) ^ sw] = __builtin_bit_cast(uint4, eight_bf16<TYPE>(k.z, k.w));
        uint4 w = v;
        const int n = min(max(count - 16 * v_part(), 0), 16);  // tokens that are there, of this thread's part
        if (MASK && count > 0 && -count < hidden_to) {  // the tile begins before the window; see below
            const int behind = 16 * v_part() - count;  // where this part begins, counted as well
            const uint32_t kept = low_bits(count - 16 * v_part()) & (~low_bits(hidden_to - behind) | low_bits(hidden_from - behind));
            w.x &= bytes_of(kept);
            w.y &= bytes_of(kept >> 4);
            w.z &= bytes_of(kept >> 8);
            w.w &= bytes_of(kept >> 12);
        } else if (count < S::kTokens) {  // bytes that nobody wrote may be NaN in e4m3, which a weight of 0 does not silence
            w.x &= byte_mask(n);
            w.y &= byte_mask(n - 4);
            w.z &= byte_mask(n - 8);
            w.w &= byte_mask(n - 12);
        }
        // The same for drafted tokens that none of the rows sees; looked up just where there are such bytes, since they are what nobody wrote
        if constexpr (MASK && TYPE == WL_KV_E4M3) {
            if (a.mask.tree && base + S::kTokens > seq.begin && (has_nan(w.x) || has_nan(w.y) || has_nan(w.z) || has_nan(w.w))) {
                const int at = base + 16 * v_part(), last = min((row0 + kGroupRows - 1) / a.group, seq.n - 1);
                uint32_t kept = low_bits(seq.begin - at);
                for (int token = row0 / a.group; token <= last; token++) kept |= tree_bits(a, seq, token, at);
                w.x &= bytes_of(kept);
                w.y &= bytes_of(kept >> 4);
                w.z &= bytes_of(kept >> 8);
                w.w &= bytes_of(kept >> 12);
            }
        }
        const int d = v_dim(), x = v_part(), slot = ((x & 1) * 32 + (d & 31)) ^ S::v_swizzle(x);
        uint4(*pair)[64] = &lds.v[buffer][((d >> 5) * S::kSubs + (x >> 1)) * 2];
        pair[0][slot] = __builtin_bit_cast(uint4, eight_bf16<TYPE>(w.x, w.y));
        pair[1][slot] = __builtin_bit_cast(uint4, eight_bf16<TYPE>(w.z, w.w));
        if (threadIdx.x < S::kParts) {
            int id = threadIdx.x;
            if constexpr (MASK && D == 256) {
                // asked for again for every tile: kept, what is addressed with it would be spilled, and come back from memory between
                // the loads and the barrier
                id = __builtin_amdgcn_mbcnt_lo(~0u, 0);
                __asm__ volatile("" : "+v"(id));
            }
            // never 0: a masked score is -inf, and times the scale it has to stay that (a block of zeros scores 0 all the same)
            const float scaled = ks * a.scale_log2;
            const bool fold = vs >= 8.6736174e-19f && vs <= 1.1529215e18f;  // 2^-60 .. 2^60
            lds.part[buffer][id] = {scaled == 0.0f ? 1.17549435e-38f : scaled, fold ? __builtin_amdgcn_logf(vs) : 0.0f,
                                             fold ? 1.0f / vs : 1.0f, fold ? 1.0f : vs};
            lds.count[buffer][id] = MASK ? low_bits(n) : n;
        }
    }
};

__device__ __forceinline__ float other_half(float x, bool add) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t r0 = r[0], r1 = r[1];
    const float p = __builtin_bit_cast(float, r0), q = __builtin_bit_cast(float, r1);
    return add ? p + q : fmaxf(p, q);
}

// A wavefront's 32 rows: q, the running maximum, its lanes' sums and O^T.
template <int D>
struct Wave {
    using S = Shape<D>;
    bf16x8 q[S::kSteps];
    f32x16 o[S::kBlocks];
    float m, l;

    // The 32 tokens of part u of a tile; seen: of this lane's 16 tokens, those that its row may see, as many from the first on or,
    // with MASK, as bits.
    // Operands come from LDS four products ahead (two with 256 dimensions), V's first ones before the softmax.
    template <bool MASK>
    __device__ __forceinline__ void add(const Lds<D>& lds, int buffer, int u, int seen) {
        constexpr int kAhead = D == 256 ? 2 : 4;  // no registers for more with 256 dimensions
        int lane = threadIdx.x & 63;
        // with 256 dimensions its slots are worked out for every tile: kept, they would cost five registers
        if constexpr (D == 256) __asm__ volatile("" : "+v"(lane));
        const int half = lane >> 5;
        const uint4(*kt)[64] = &lds.k[buffer][u * S::kSteps];
        f32x16 s = (f32x16)(0.0f);
        uint4 f[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) f[i] = kt[i][lane ^ S::k_swizzle(i)];
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < S::kSteps; i++) {
            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, f[i % kAhead]), q[i], s, 0, 0, 0);
            if (i + kAhead < S::kSteps) f[i % kAhead] = kt[i + kAhead][lane ^ S::k_swizzle(i + kAhead)];
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        const Part part = lds.part[buffer][2 * u + half];
        const int there = lds.count[buffer][2 * u + half];
        const int mine = MASK ? seen & there : min(there, seen);
        // a lane that sees no token of its block is not to meet the block's scales: they may be NaN
        const float ks = mine > 0 ? part.ks : 1.0f, rest = mine > 0 ? part.rest : 1.0f;
        const int slot = lane ^ S::v_swizzle(2 * u + half);
        auto v = [&](int i) { return lds.v[buffer][(i / 2 * S::kSubs + u) * 2 + i % 2][slot]; };
#pragma unroll
        for (int i = 0; i < kAhead; i++) f[i] = v(i);
        __builtin_amdgcn_sched_barrier(0);
        if (__any(MASK ? mine != 0xFFFF : mine < 16)) {
#pragma unroll
            for (int i = 0; i < 16; i++) s[i] = (MASK ? mine >> i & 1 : i < mine) ? s[i] : -__builtin_inff();
        }
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 16; i++) top = fmaxf(top, s[i]);
        top = other_half(top * ks, false);
        if (__any(top > m + kSlack || (m == -__builtin_inff() && top > m))) {
            const float now = fmaxf(m, top), shrink = now == -__builtin_inff() ? 1.0f : exp2_fast(m - now);
            m = now;
            l *= shrink;
#pragma unroll
            for (int i = 0; i < S::kBlocks; i++) o[i] *= shrink;
        }
        const float shift = part.log2_vs - (m == -__builtin_inff() ? 0.0f : m);
        float sum = 0.0f;
        uint32_t p[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float e0 = exp2_fast(__builtin_fmaf(s[2 * i], ks, shift)), e1 = exp2_fast(__builtin_fmaf(s[2 * i + 1], ks, shift));
            sum += e0 + e1;
            p[i] = pack_bf16(e0, e1);
        }
        l = __builtin_fmaf(sum, part.inverse, l);
        if (__any(rest != 1.0f)) {  // rounded once more, where a scale is as far out as that
#pragma unroll
            for (int i = 0; i < 8; i++)
                p[i] = pack_bf16(__builtin_bit_cast(float, p[i] << 16) * rest, __builtin_bit_cast(float, p[i] & 0xFFFF0000u) * rest);
        }
        __builtin_amdgcn_s_setprio(1);
        const bf16x8 p0 = __builtin_bit_cast(bf16x8, make_uint4(p[0], p[1], p[2], p[3])),
                     p1 = __builtin_bit_cast(bf16x8, make_uint4(p[4], p[5], p[6], p[7]));
#pragma unroll
        for (int i = 0; i < 2 * S::kBlocks; i++) {
            o[i / 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, f[i % kAhead]), i % 2 ? p1 : p0,
                                                               o[i / 2], 0, 0, 0);
            if (i + kAhead < 2 * S::kBlocks) f[i % kAhead] = v(i + kAhead);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
    }
};

// Tiles of the cache that rows [row0, row0 + 256) of a sequence see; at least one where there are rows, which have to be
// written even if they see nothing.
template <bool MASK>
__device__ __forceinline__ Span span_at(const AttendArgs& a, Seq seq, int row0, int tile_tokens) {
    const int last = min((row0 + kGroupRows - 1) / a.group, seq.n - 1);
    return span_of<MASK>(a, seq, row0 / a.group, MASK && a.mask.tree ? seq.length : seq.seen(last, a.causal), tile_tokens);
}
template <bool MASK>
__device__ __forceinline__ int tiles_of(const AttendArgs& a, Seq seq, int row0, int tile_tokens) {
    return row0 >= seq.n * a.group ? 0 : max(span_at<MASK>(a, seq, row0, tile_tokens).tiles, 1);
}

// A row tile's tiles in pieces of at most `each`, as equal as can be, unless that were too many pieces.
struct Cut {
    int pieces, size;
};
__device__ __forceinline__ Cut cut_of(int tiles, int each, int most) {
    const int pieces = min((tiles + each - 1) / each, most);
    return {pieces, pieces ? (tiles + pieces - 1) / pieces : 0};
}

// What a workgroup takes: the pieces of all row tiles in order of their size, the largest first, one for each kv head. A
// causal prompt's row tiles see from one to all of its tokens, and a call's sequences may differ as much: were they taken as
// they come, the last large one would run on alone. Every workgroup ranks the pieces for itself, by 64 classes of size.
struct Work {
    int b, row0, piece, pieces, t0, t1;
};
constexpr int kClasses = 64;
constexpr int kLeast = 4;  // tiles that are worth a piece
struct PlanLds {
    uint32_t classes[kClasses];
    uint32_t sums[kWaves];
    uint32_t candidates[kWaves][2];
    Work work;
};

template <int D, bool MASK>
__device__ __forceinline__ bool find_work(const RowsArgs& a, PlanLds& lds, Work& work) {
    constexpr int T = Shape<D>::kTokens;
    const uint32_t wanted = blockIdx.x / a.c.kv_heads;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    // max_count may say nothing (all rows of the call): where that makes for many empty row tiles, the longest sequence
    // says how many there are (1000 sequences of 8 rows: 8.9 ms without, 0.45 ms with, 0.43 ms where max_count says it)
    uint32_t row_tiles = a.row_tiles;
    if (row_tiles > 1 && a.s.seqs * row_tiles > 2 * kThreads) {
        int most = 1;
        for (int b = threadIdx.x; b < a.s.seqs; b += kThreads) most = max(most, a.seq(b).n);
#pragma unroll
        for (int d = 32; d; d >>= 1) most = max(most, __shfl_xor(most, d));
        if (lane == 0) lds.sums[wave] = most;
        __syncthreads();
        for (int i = 0; i < kWaves; i++) most = max(most, static_cast<int>(lds.sums[i]));
        row_tiles = __builtin_amdgcn_readfirstlane((most * a.group + kGroupRows - 1) / kGroupRows);
        __syncthreads();  // the maxima have been read
    }
    const uint32_t items = a.s.seqs * row_tiles;
    auto tiles_read = [&](uint32_t i) {
        return i < items ? tiles_of<MASK>(a, a.seq(i / row_tiles), static_cast<int>(i % row_tiles) * kGroupRows, T) : 0;
    };
    const int own_tiles = tiles_read(threadIdx.x);  // for most calls all there is
    auto tiles_at = [&](uint32_t i) { return i == threadIdx.x ? own_tiles : tiles_read(i); };
    uint32_t total = 0;
    for (uint32_t i = threadIdx.x; i < items; i += kThreads) total += tiles_at(i);
    total = wave_sum(total);
    if (lane == 0) lds.sums[wave] = total;
    if (threadIdx.x < kClasses) lds.classes[threadIdx.x] = 0;
    __syncthreads();
    total = 0;
    for (int i = 0; i < kWaves; i++) total += lds.sums[i];
    int each = max(static_cast<int>((static_cast<uint64_t>(total) * a.c.kv_heads + kCus - 1) / kCus), kLeast);
    if (a.pieces > 1 && !a.few_tiles) {
        each += each / 2;  // more than a CU's share alone, see rows_plan
    } else if (a.pieces > 1) {
        // A CU's share of the whole, or up to three quarters more of it where that brings the pieces down to one a CU: every
        // row tile's last piece makes them more than the shares are, and the few that are left over run on alone
        // (512 tokens of 16 on 2 heads of 256 behind 16000: 243 us without, 170 with; five ragged prompts of up to 301 of 32
        // on 8 heads of 128 40.6 and 33.6; calls that no candidate suits stay as they are).
        // (item, kv head)s are less than 2 kCus here, so the pieces of one candidate fit 16 bits.
        auto candidate = [&](int i) { return each + (each * i + 3) / 4; };
        uint32_t n01 = 0, n23 = 0;
        for (uint32_t i = threadIdx.x; i < items; i += kThreads) {
            const int tiles = tiles_at(i);
            n01 += cut_of(tiles, candidate(0), a.pieces).pieces | cut_of(tiles, candidate(1), a.pieces).pieces << 16;
            n23 += cut_of(tiles, candidate(2), a.pieces).pieces | cut_of(tiles, candidate(3), a.pieces).pieces << 16;
        }
        n01 = wave_sum(n01);
        n23 = wave_sum(n23);
        if (lane == 0) {
            lds.candidates[wave][0] = n01;
            lds.candidates[wave][1] = n23;
        }
        __syncthreads();
        n01 = n23 = 0;
        for (int i = 0; i < kWaves; i++) {
            n01 += lds.candidates[i][0];
            n23 += lds.candidates[i][1];
        }
        const uint32_t most = kCus / a.c.kv_heads;
        const int best = (n01 & 0xFFFF) <= most ? 0 : n01 >> 16 <= most ? 1 : (n23 & 0xFFFF) <= most ? 2 : n23 >> 16 <= most ? 3 : 0;
        each = __builtin_amdgcn_readfirstlane(candidate(best));
    }
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.pieces > 1) *a.each = each;
    auto class_of = [&](Cut c) { return kClasses - 1 - min(static_cast<int>(c.size * (kClasses - 1ll) / each), kClasses - 1); };
    for (uint32_t i = threadIdx.x; i < items; i += kThreads) {
        const Cut c = cut_of(tiles_at(i), each, a.pieces);
        if (c.pieces) atomicAdd(&lds.classes[class_of(c)], static_cast<uint32_t>(c.pieces));
    }
    __syncthreads();
    const uint32_t own = lds.classes[lane], sum = wave_scan(own);
    const uint64_t past = __ballot(sum > wanted);
    if (!past) return false;
    const int mine = __builtin_ctzll(past);
    const uint32_t rank = wanted - __builtin_amdgcn_readlane(sum - own, mine);  // in its class, in the order of the row tiles
    uint32_t before = 0;
    for (uint32_t i0 = 0; i0 < items; i0 += kThreads) {
        const uint32_t i = i0 + threadIdx.x;
        const int tiles = tiles_at(i);
        const Cut c = cut_of(tiles, each, a.pieces);
        const uint32_t n = c.pieces && class_of(c) == mine ? c.pieces : 0, upto = wave_scan(n);
        __syncthreads();  // the sums before have been read
        if (lane == 63) lds.sums[wave] = upto;
        __syncthreads();
        uint32_t at = before + upto - n;
        for (int j = 0; j < kWaves; j++) {
            if (j < wave) at += lds.sums[j];
            before += lds.sums[j];
        }
        if (at <= rank && rank < at + n) {
            const int piece = rank - at;
            lds.work = {static_cast<int>(i / row_tiles), static_cast<int>(i % row_tiles) * kGroupRows, piece, c.pieces,
                        min(piece * c.size, tiles), min((piece + 1) * c.size, tiles)};
        }
        if (before > rank) break;
    }
    __syncthreads();
    work = lds.work;
    work.b = __builtin_amdgcn_readfirstlane(work.b);
    work.row0 = __builtin_amdgcn_readfirstlane(work.row0);
    work.piece = __builtin_amdgcn_readfirstlane(work.piece);
    work.pieces = __builtin_amdgcn_readfirstlane(work.pieces);
    work.t0 = __builtin_amdgcn_readfirstlane(work.t0);
    work.t1 = __builtin_amdgcn_readfirstlane(work.t1);
    return true;
}

// blockIdx: (rank of the piece, kv head).
template <int TYPE, int D, bool PAGE, bool MASK>
__global__ __launch_bounds__(kThreads, 2) void k_attend_rows(RowsArgs a) {
    using S = Shape<D>;
    __shared__ union {
        Lds<D> lds;
        PlanLds plan;
    } shared;
    Lds<D>& lds = shared.lds;
    Work cut;
    if (!find_work<D, MASK>(a, shared.plan, cut)) return;
    __syncthreads();  // the plan has been read
    const int b = cut.b, row0 = cut.row0, piece = cut.piece, head = blockIdx.x % a.c.kv_heads;
    const Seq seq = a.seq_uniform(b);

    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, half = lane >> 5;
    const int row = row0 + 32 * wave + (lane & 31), token = row / a.group;
    const bool there = token < seq.n;
    const int limit = MASK ? limit_of(a, seq, token) : there ? seq.seen(token, a.causal) : 0;
    const uint16_t* qp = a.q + static_cast<int64_t>(seq.at + token) * a.q_token_stride +
                         static_cast<int64_t>(head * a.group + row % a.group) * a.q_head_stride + 8 * half;
    const int most = MASK && a.mask.tree                            ? seq.length
                     : __builtin_amdgcn_readlane(limit, 31) > 0 ? __builtin_amdgcn_readlane(limit, 31)
                                                                : seq.length;
    const Span span = MASK ? span_at<MASK>(a, seq, row0, S::kTokens) : Span{0, 0, 0};
    auto base_of = [&](int t) { return span.tile(t) * S::kTokens; };
    // the tokens between the sinks and the first row's window, of the workgroup's rows (counted from the sequence's end) and of the wavefront's
    const int hidden_from = MASK ? a.mask.sinks - seq.length : 0, hidden_to = MASK ? window_begin(a, seq, row0 / a.group) - seq.length : 0;
    // tokens that some row of the wavefront sees begin there; that every row sees (in front of a tree), from whole_from to whole_to
    const int window_at = MASK ? window_begin(a, seq, __builtin_amdgcn_readfirstlane(token)) : 0;
    int whole_from = 0, whole_to = 0;
    if constexpr (MASK) {
        const int last = min((row0 + 32 * __builtin_amdgcn_readfirstlane(wave) + 31) / a.group, seq.n - 1);
        whole_from = max(max(seq.begin + (a.mask.tree ? seq.n : last + 1), 0) - a.mask.window, 0);
        whole_to = a.mask.tree ? seq.begin : __builtin_amdgcn_readfirstlane(limit);
    }

    Stage<TYPE, D, PAGE, MASK> st;
    st.find(a, b, base_of(cut.t0));
    st.load(a, head, base_of(cut.t0), seq.length);
    Wave<D> w;
#pragma unroll
    for (int i = 0; i < S::kSteps; i++) {
        const uint16_t* e = qp + 16 * i;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (there)
            x = a.wide_q ? *reinterpret_cast<const uint4*>(e)
                         : make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
        w.q[i] = __builtin_bit_cast(bf16x8, x);
    }
#pragma unroll
    for (int i = 0; i < S::kBlocks; i++) w.o[i] = (f32x16)(0.0f);
    w.m = -__builtin_inff();
    w.l = 0.0f;
    const bool idle = !__any(there);

    st.store(a, lds, 0, base_of(cut.t0), seq, row0, hidden_from, hidden_to);
    if (cut.t0 + 1 < cut.t1) {
        st.find(a, b, base_of(cut.t0 + 1));
        st.load(a, head, base_of(cut.t0 + 1), seq.length);
        st.store(a, lds, 1, base_of(cut.t0 + 1), seq, row0, hidden_from, hidden_to);
    }
    // q is here before the loop: were it still on its way, the first product of every round would wait for that round's loads
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    st.find(a, b, base_of(cut.t0 + 2));
    __syncthreads();
    for (int t = cut.t0; t < cut.t1; t++) {
        const int buffer = (t - cut.t0) & (kRing - 1), base = base_of(t);
        if (t + 2 < cut.t1) {
            st.load(a, head, base_of(t + 2), seq.length);
            st.find(a, b, base_of(t + 3));
        }
#pragma unroll
        for (int u = 0; u < S::kSubs; u++) {
            if (idle || base + 32 * u >= most) break;
            const int at = base + 32 * u + 16 * half;
            if constexpr (MASK) {
                if (base + 32 * u + 32 <= window_at && base + 32 * u >= a.mask.sinks) continue;
                int seen = 0xFFFF;
                if (base + 32 * u < whole_from || base + 32 * u + 32 > whole_to) {  // a few tiles: the row is worked out again, as below
                    const int r = (row0 + static_cast<int>((threadIdx.x >> 6) * 32 + (threadIdx.x & 31) + lane_zero())) / a.group;
                    const uint32_t drafted = a.mask.tree && base + 32 * u + 32 > seq.begin ? tree_bits(a, seq, r, at) : 0;
                    seen = seen_bits(a, seq, limit_of(a, seq, r), at, 16, drafted);
                }
                w.template add<MASK>(lds, buffer, u, seen);
            } else {
                w.template add<MASK>(lds, buffer, u, limit - at);
            }
        }
        if (t + 2 < cut.t1) st.store(a, lds, (buffer + 2) & (kRing - 1), base_of(t + 2), seq, row0, hidden_from, hidden_to);
        if (buffer & 1) __syncthreads();
    }
    const float m = w.m, l = other_half(w.l, true);
    f32x16(&o)[S::kBlocks] = w.o;
    // worked out again: the loop has no register to keep them in
    const int out_row = row0 + static_cast<int>((threadIdx.x >> 6) * 32 + (threadIdx.x & 31) + lane_zero());
    const int out_token = out_row / a.group;
    if (out_token >= seq.n) return;
    const int64_t place = static_cast<int64_t>(seq.at + out_token) * a.q_heads + head * a.group + out_row % a.group;
    if (cut.pieces == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t* out = a.out + place * D + 4 * half;
#pragma unroll
        for (int i = 0; i < S::kBlocks; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                *reinterpret_cast<uint2*>(out + 32 * i + 8 * j) =
                    make_uint2(pack_bf16(o[i][4 * j] * inv, o[i][4 * j + 1] * inv),
                               pack_bf16(o[i][4 * j + 2] * inv, o[i][4 * j + 3] * inv));
        return;
    }
    const int64_t slot = static_cast<int64_t>(piece) * a.s.tokens * a.q_heads + place;
    float* out = a.partial + slot * D + 4 * half;
#pragma unroll
    for (int i = 0; i < S::kBlocks; i++)
#pragma unroll
        for (int j = 0; j < 4; j++)
            *reinterpret_cast<f32x4*>(out + 32 * i + 8 * j) =
                (f32x4){o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]};
    if (half == 0) a.partial_ml[slot] = make_float2(m, l);
}

// Adds up the pieces of the row tiles that were cut, up to kMaxPieces of them: a wavefront takes four rows, so that a row's chain of loads is shared
// (one row each: 21 us for a prompt of 4096 tokens, of which it adds up half, 12 us for the five ragged ones of up to 300;
// four: 15 and 7). blockIdx: (16 rows, kv head), sequence.
constexpr int kMergeWaves = 4, kWaveRows = 4, kMergeRows = kMergeWaves * kWaveRows;
static_assert(64 / kWaveRows == kMaxPieces && kGroupRows % kMergeRows == 0, "a lane for each piece of each row");
template <int D, bool MASK>
__global__ __launch_bounds__(kMergeWaves * 64) void k_attend_merge(RowsArgs a) {
    const int b = blockIdx.y, head = blockIdx.x % a.c.kv_heads, lane = threadIdx.x & 63;
    const int first = __builtin_amdgcn_readfirstlane(blockIdx.x / a.c.kv_heads * kMergeRows + (threadIdx.x >> 6) * kWaveRows);
    const Seq seq = a.seq_uniform(b);
    const int rows = seq.n * a.group;
    if (first >= rows) return;
    const int pieces = cut_of(tiles_of<MASK>(a, seq, first / kGroupRows * kGroupRows, Shape<D>::kTokens), *a.each, a.pieces).pieces;
    if (pieces < 2) return;
    constexpr int V = D / 64;
    typedef float Lane __attribute__((ext_vector_type(V)));
    const int64_t stride = static_cast<int64_t>(a.s.tokens) * a.q_heads;
    const int row = min(first + lane / kMaxPieces, rows - 1), piece = lane % kMaxPieces;
    const int place = (seq.at + row / a.group) * a.q_heads + head * a.group + row % a.group;
    const float2 ml = piece < pieces ? a.partial_ml[piece * stride + place] : make_float2(-__builtin_inff(), 0.0f);
    float top = ml.x;
#pragma unroll
    for (int d = kMaxPieces / 2; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float own = exp2_fast(ml.x - (top == -__builtin_inff() ? 0.0f : top));
    float l = ml.y * own;
#pragma unroll
    for (int d = kMaxPieces / 2; d; d >>= 1) l += __shfl_xor(l, d);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    int at[kWaveRows];
    Lane sum[kWaveRows];
#pragma unroll
    for (int r = 0; r < kWaveRows; r++) {
        at[r] = __builtin_amdgcn_readlane(place, r * kMaxPieces);
        sum[r] = (Lane)(0.0f);
    }
    auto of_lane = [](float x, int i) {
        return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), i));
    };
    for (int i = 0; i < pieces; i++) {
        Lane x[kWaveRows];
#pragma unroll
        for (int r = 0; r < kWaveRows; r++) x[r] = *reinterpret_cast<const Lane*>(a.partial + (i * stride + at[r]) * D + lane * V);
#pragma unroll
        for (int r = 0; r < kWaveRows; r++) sum[r] += x[r] * of_lane(own, r * kMaxPieces + i);
    }
#pragma unroll
    for (int r = 0; r < kWaveRows; r++) {
        if (first + r >= rows) break;
        const float f = of_lane(inv, r * kMaxPieces);
        uint16_t* out = a.out + static_cast<int64_t>(at[r]) * D + lane * V;
        if constexpr (V == 4) {
            *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(sum[r][0] * f, sum[r][1] * f), pack_bf16(sum[r][2] * f, sum[r][3] * f));
        } else if constexpr (V == 2) {
            *reinterpret_cast<uint32_t*>(out) = pack_bf16(sum[r][0] * f, sum[r][1] * f);
        } else {
            *out = __builtin_bit_cast(uint16_t, static_cast<__bf16>(sum[r][0] * f));
        }
    }
}

// The same for more than kMaxPieces of them, which few rows have: a workgroup a row, its pieces in turn over the wavefronts.
// blockIdx: (row, kv head), sequence.
template <int D>
__global__ __launch_bounds__(kMergeWaves * 64) void k_attend_merge_row(RowsArgs a) {
    __shared__ float part[kMergeWaves][D];
    const int b = blockIdx.y, head = blockIdx.x % a.c.kv_heads, row = blockIdx.x / a.c.kv_heads, wave = threadIdx.x >> 6,
              lane = threadIdx.x & 63;
    const Seq seq = a.seq_uniform(b);
    if (row >= seq.n * a.group) return;
    const int pieces = cut_of(tiles_of<true>(a, seq, row / kGroupRows * kGroupRows, Shape<D>::kTokens), *a.each, a.pieces).pieces;
    if (pieces < 2) return;
    constexpr int V = D / 64;
    typedef float Lane __attribute__((ext_vector_type(V)));
    const int64_t stride = static_cast<int64_t>(a.s.tokens) * a.q_heads;
    const int64_t place = static_cast<int64_t>(seq.at + row / a.group) * a.q_heads + head * a.group + row % a.group;
    auto values = [&](int i) { return *reinterpret_cast<const Lane*>(a.partial + (i * stride + place) * D + lane * V); };
    constexpr int kMost = kMaxMaskedPieces / kMergeWaves;
    Lane x[kMost];
#pragma unroll
    for (int i = 0; i < kMost; i++) x[i] = values(min(wave + kMergeWaves * i, pieces - 1));
    const float2 ml = lane < pieces ? a.partial_ml[lane * stride + place] : make_float2(-__builtin_inff(), 0.0f);
    float top = ml.x;
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float own = exp2_fast(ml.x - (top == -__builtin_inff() ? 0.0f : top));  // 0 behind the last piece
    float l = ml.y * own;
#pragma unroll
    for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d);
    Lane sum = {};
#pragma unroll
    for (int i = 0; i < kMost; i++) {
        const int piece = wave + kMergeWaves * i;
        if (piece < pieces) sum += x[i] * __shfl(own, piece);
    }
#pragma unroll
    for (int e = 0; e < V; e++) part[wave][lane * V + e] = sum[e];
    __syncthreads();
    if (threadIdx.x >= D) return;
    float y = 0.0f;
#pragma unroll
    for (int w = 0; w < kMergeWaves; w++) y += part[w][threadIdx.x];
    a.out[place * D + threadIdx.x] = __builtin_bit_cast(uint16_t, static_cast<__bf16>(l == 0.0f ? 0.0f : y / l));
}

// How the row tiles' caches are cut. Calls of few row tiles would leave CUs idle, and a causal prompt's last row tiles would
// run on alone: a cache is cut into pieces of a CU's share of the whole where that is less. From twice as many row tiles as
// CUs on, taking the large ones first is enough while none is more than a CU's share: so for the rows of one sequence, which see
// the same cache or up to it. Of several sequences one may be far longer than the others, which the device alone sees: where its
// tiles would take longer than the second kernel costs, a row tile of more than one and a half shares is cut (64 sequences of 8 kv
// heads of 128, 5 tokens each, of which one has 100000 in the cache, the others 100: 2616 us without, 183 with; all of them 5000:
// 280 and 286; all 100 with a bound that says 8192: 17.3 and 20.9). Where there is no room for at least four pieces, the rows are so many that none stands out.
struct RowsPlan {
    int64_t row_tiles, pieces, groups;
    bool few_tiles;
};
constexpr int kLong = 64;  // tiles: about 80 us for one workgroup
RowsPlan rows_plan(const WlKvCache* c, int q_heads, const WlKvBatch* b, int64_t max_length, const WlKvMask* mask) {
    const int64_t tokens = 8192 / c->head_dim, group = q_heads / c->kv_heads;
    const int64_t rows = mask && mask->tree ? b->max_count : std::min<int64_t>(b->max_count, (kGroupRows + group - 2) / group + 1);
    const int64_t longest = longest_span(c, b, max_length, mask, rows, tokens);  // that a row tile goes through
    const int64_t row_tiles = (b->max_count * group + kGroupRows - 1) / kGroupRows;
    // (row tile, kv head)s: as many as the sequences' most rows have room for, and no more than all rows together fill
    const int64_t items = std::min(row_tiles * b->seqs, b->tokens * group / kGroupRows + b->seqs) * c->kv_heads;
    const int64_t most = (longest + tokens - 1) / tokens;  // tiles of the last row tile
    // how many pieces come of it is known on the device alone: room for as many as the partial results may take
    const int64_t room = kPartialBytes / (b->tokens * q_heads * c->head_dim * static_cast<int64_t>(sizeof(float)));
    const bool few_tiles = items < 2 * kCus;
    // With a window the row tiles of one sequence go through as many tiles each, from the window's length on: where they fill the CUs
    // to nine tenths nothing is cut, and the second kernel (5 us of 102 for 4096 tokens in a window of 1024) is left out. With fewer
    // tokens than a window before them the first rows see less. Where there is one round of row tiles, and the longest is more than a
    // CU's share and the three quarters of it by which the device lets a piece grow, they are cut (4096 tokens of 16 on 2 heads of 256
    // with nothing before, in a window of 3840: 225 us uncut, 195 cut; of 3584, where the two are nearly equal, 212 and 196, and 8192
    // of 8 on one of 64 in 7168 188 and 194; of 3000 183 and 189; two rounds, of 7680 tokens, in a window of 7200: 479 and 491).
    const int64_t all = std::min<int64_t>(max_length, int64_t{b->table_width} * c->page_tokens);
    if (mask && longest < all && b->seqs == 1 && few_tiles && 10 * items >= 9 * ((items + kCus - 1) / kCus * kCus)) {
        const int64_t window = mask->window, rows_all = b->max_count,  // products below 2^60: one round has at most 2^16 rows
            missing = mask->tree ? 0 : std::max<int64_t>(window - (all - rows_all), 0);  // of the first row's window
        if (items > kCus || 7 * items * (2 * window * rows_all - missing * missing) >= 8 * kCus * window * rows_all)
            return {row_tiles, 1, items, true};
    }
    if (!few_tiles && (b->seqs == 1 || most < kLong || room < 4)) return {row_tiles, 1, items, false};
    const int64_t limit = mask && items < kCus / kMaxPieces ? kMaxMaskedPieces : kMaxPieces;
    const int64_t pieces = std::max<int64_t>(1, std::min({limit, (most + kLeast - 1) / kLeast, room}));
    // the pieces of n tiles are less than n / each + 1, those of all (row tile, kv head)s less than kCus + items
    return {row_tiles, pieces, pieces == 1 ? items : std::min(items * pieces, items + kCus), few_tiles};
}

}  // namespace

size_t attend_rows_workspace(const WlKvCache* c, int q_heads, const WlKvBatch* b, int64_t max_length, const WlKvMask* mask) {
    const RowsPlan p = rows_plan(c, q_heads, b, max_length, mask);
    if (p.pieces == 1) return 0;
    return 16 + static_cast<size_t>(p.pieces * b->tokens * q_heads) * (c->head_dim * sizeof(float) + sizeof(float2));
}

static int64_t merge_groups(const WlKvCache* c, int64_t group, const WlKvBatch* b) {
    return (b->max_count * group + kMergeRows - 1) / kMergeRows * c->kv_heads;
}

bool attend_rows_fit(const WlKvCache* c, int q_heads, const WlKvBatch* b, int64_t max_length, const WlKvMask* mask) {
    const RowsPlan p = rows_plan(c, q_heads, b, max_length, mask);
    return p.row_tiles * b->seqs < (int64_t{1} << 31) && fits_a_launch(p.groups, kThreads) &&
           fits_a_launch(p.pieces > kMaxPieces ? int64_t{b->max_count} * q_heads : merge_groups(c, q_heads / c->kv_heads, b),
                         kMergeWaves * 64);
}

int launch_attend_rows(const WlKvCache* c, const AttendArgs& call, const WlKvBatch* b, int64_t max_length, const WlKvMask* mask,
                       void* workspace, hipStream_t stream) {
    const RowsPlan p = rows_plan(c, call.q_heads, b, max_length, mask);
    RowsArgs a;
    static_cast<AttendArgs&>(a) = call;
    a.each = static_cast<int32_t*>(workspace);
    a.partial = static_cast<float*>(workspace) + 4;
    a.partial_ml = reinterpret_cast<float2*>(a.partial + p.pieces * b->tokens * call.q_heads * c->head_dim);
    a.row_tiles = static_cast<int32_t>(p.row_tiles);
    a.pieces = static_cast<int32_t>(p.pieces);
    a.few_tiles = p.few_tiles;
    const dim3 grid(static_cast<uint32_t>(p.groups));
    const dim3 merge(static_cast<uint32_t>(merge_groups(c, call.group, b)), b->seqs);
    auto with_mask = [&](auto type, auto dim, auto masked) {
        constexpr int T = decltype(type)::value, D = decltype(dim)::value;
        constexpr bool MASK = decltype(masked)::value;
        if (c->page_tokens >= Shape<D>::kTokens)
            k_attend_rows<T, D, true, MASK><<<grid, kThreads, 0, stream>>>(a);
        else
            k_attend_rows<T, D, false, MASK><<<grid, kThreads, 0, stream>>>(a);
        if (const int rc = launch_status()) return rc;
        if constexpr (MASK) {
            if (p.pieces > kMaxPieces) {
                k_attend_merge_row<D><<<dim3(static_cast<uint32_t>(b->max_count * call.group * c->kv_heads), b->seqs), kMergeWaves * 64, 0,
                                        stream>>>(a);
                return launch_status();
            }
        }
        if (p.pieces > 1) k_attend_merge<D, MASK><<<merge, kMergeWaves * 64, 0, stream>>>(a);
        return launch_status();
    };
    auto run = [&](auto type, auto dim) {
        return mask ? with_mask(type, dim, std::true_type()) : with_mask(type, dim, std::false_type());
    };
    auto with_dim = [&](auto type) {
        if (c->head_dim == 64) return run(type, std::integral_constant<int, 64>());
        if (c->head_dim == 128) return run(type, std::integral_constant<int, 128>());
        return run(type, std::integral_constant<int, 256>());
    };
    if (c->type == WL_KV_INT8) return with_dim(std::integral_constant<int, WL_KV_INT8>());
    return with_dim(std::integral_constant<int, WL_KV_E4M3>());
}

}  // namespace wl
