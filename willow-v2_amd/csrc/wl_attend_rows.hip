// Attention over the paged 8-bit cache for more than 16 rows of a (sequence, kv head): prompts, chunks of them, drafts.
//
// A workgroup takes 256 rows, a wavefront 32 of them (v_mfma_f32_32x32x16_bf16), and goes through the cache in tiles of
// 8192 / D tokens. The workgroup turns a tile's bytes into bf16 once, into LDS, in the order in which the products take
// them (16 bytes a lane, 1 KB a k-step, so every read is a straight run over the lanes): each of K's and V's values is
// converted by one of eight wavefronts and used by all. Two tiles are in LDS: while one is multiplied, the next one's
// bytes are on their way in registers, and are converted into the other.
// Token 16 h + i of a 32-token part is row 8 (i / 4) + 4 h + i % 4 of the first product, so a lane of half h holds the
// scores of tokens 16 h .. 16 h + 15 of row lane % 32, which is how the second product takes the weights.
// The running maximum is moved only when a score exceeds it by 2^8 (the weights stay below 2^8, fp32 sums hold them): the
// multiplication of a wavefront's 32 x D sums by the change is the dearest step of the softmax, and becomes rare.
#include <algorithm>

#include "wl_attend.h"

namespace wl {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWaves = 8;
constexpr int kThreads = kWaves * 64;
constexpr int kGroupRows = kWaves * 32;
constexpr int kMaxPieces = 16;
constexpr int kCus = 256;
constexpr float kSlack = 8.0f;  // log2: how far a score may lie above the running maximum

struct RowsArgs : AttendArgs {
    float* partial;      // [pieces][tokens][q_heads][D]
    float2* partial_ml;  // [pieces][tokens][q_heads]: maximum (in log2) and sum
    int32_t row_tiles;   // of 256 rows, at most
    int32_t pieces;      // a row tile's cache is cut into at most this many
    int32_t tiles_each;  // .. of about this many tiles
};

// What a part of 16 tokens needs beside its bytes.
struct Part {
    float ks, vs;  // scales (K's with the softmax's scale and log2 e)
    int count;     // tokens that are there
    int unused;
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
    uint4 k[2][Shape<D>::kSubs * Shape<D>::kSteps][64];
    uint4 v[2][Shape<D>::kBlocks * Shape<D>::kSubs * 2][64];
    Part part[2][Shape<D>::kParts];
};

// One thread's share of a tile on its way: 16 values of one token of K, 16 tokens of one dimension of V. PAGE: a page holds
// whole tiles, so a tile has one page and one pair of scales, all threads share its address, and the registers that other
// tiles need for theirs are scalar ones (with 256 dimensions a wavefront has none to spare).
template <int TYPE, int D, bool PAGE>
struct Stage {
    using S = Shape<D>;
    uint4 k, v;
    float ks, vs;
    int kpage, vpage, count;

    // 16 lanes take 4 tokens by 64 values
    static __device__ __forceinline__ int k_token() { return (threadIdx.x >> 4) / (D / 64) * 4 + ((threadIdx.x >> 2) & 3); }
    static __device__ __forceinline__ int k_chunk() { return (threadIdx.x >> 4) % (D / 64) * 4 + (threadIdx.x & 3); }
    static __device__ __forceinline__ int v_dim() { return threadIdx.x / S::kParts; }
    static __device__ __forceinline__ int v_part() { return threadIdx.x % S::kParts; }

    __device__ __forceinline__ void find(const AttendArgs& a, int b, int base) {
        if constexpr (PAGE) {
            kpage = vpage = __builtin_amdgcn_readfirstlane(a.s.page(b, a.c.column(base), a.c.pages));
        } else {
            kpage = a.s.page(b, a.c.column(base + k_token()), a.c.pages);
            vpage = a.s.page(b, a.c.column(base + 16 * v_part()), a.c.pages);
        }
    }
    __device__ __forceinline__ void load(const AttendArgs& a, int head, int base, int length) {
        const int P = a.c.page_tokens;
        const int64_t kb = a.c.block(max(kpage, 0), head), vb = a.c.block(max(vpage, 0), head);
        if constexpr (PAGE) {
            const uint8_t* kp = a.c.k + (kb * P + a.c.within(base)) * D;
            const uint8_t* vp = a.c.v + vb * P * D + a.c.within(base);
            k = *reinterpret_cast<const uint4*>(kp + static_cast<uint32_t>(k_token() * D + 16 * k_chunk()));
            v = *reinterpret_cast<const uint4*>(vp + static_cast<uint32_t>(v_dim() * P + 16 * v_part()));
            count = vpage < 0 ? 0 : length - base;  // of the tile
            ks = a.c.k_scale[kb];
            vs = a.c.v_scale[vb];
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
    __device__ __forceinline__ void store(const AttendArgs& a, Lds<D>& lds, int buffer) const {
        const int t = k_token(), step = k_chunk(), i = t & 15;
        const int row = 8 * (i >> 2) + 4 * ((t >> 4) & 1) + (i & 3);
        uint4* to = lds.k[buffer][(t >> 5) * S::kSteps + step];
        const int sw = S::k_swizzle(step);
        to[row ^ sw] = __builtin_bit_cast(uint4, eight_bf16<TYPE>(k.x, k.y));
        to[(32 + row) ^ sw] = __builtin_bit_cast(uint4, eight_bf16<TYPE>(k.z, k.w));
        uint4 w = v;
        const int n = min(max(count - 16 * v_part(), 0), 16);  // tokens that are there, of this thread's part
        if (count < S::kTokens) {  // bytes that nobody wrote may be NaN in e4m3, which a weight of 0 does not silence
            w.x &= byte_mask(n);
            w.y &= byte_mask(n - 4);
            w.z &= byte_mask(n - 8);
            w.w &= byte_mask(n - 12);
        }
        const int d = v_dim(), x = v_part(), slot = ((x & 1) * 32 + (d & 31)) ^ S::v_swizzle(x);
        uint4(*pair)[64] = &lds.v[buffer][((d >> 5) * S::kSubs + (x >> 1)) * 2];
        pair[0][slot] = __builtin_bit_cast(uint4, eight_bf16<TYPE>(w.x, w.y));
        pair[1][slot] = __builtin_bit_cast(uint4, eight_bf16<TYPE>(w.z, w.w));
        if (threadIdx.x < S::kParts) {
            // never 0: a masked score is -inf, and times the scale it has to stay that (a block of zeros scores 0 all the same)
            const float scaled = ks * a.scale_log2;
            lds.part[buffer][threadIdx.x] = {scaled == 0.0f ? 1.17549435e-38f : scaled, vs, n, 0};
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

    // The 32 tokens of part u of a tile; seen: of this lane's 16 tokens, those that its row may see.
    // Operands come from LDS four products ahead, V's first ones before the softmax.
    __device__ __forceinline__ void add(const Lds<D>& lds, int buffer, int u, int seen) {
        constexpr int kAhead = D == 256 ? 2 : 4;  // no registers for more with 256 dimensions
        const int lane = threadIdx.x & 63, half = lane >> 5;
        const uint4(*kt)[64] = &lds.k[buffer][u * S::kSteps];
        f32x16 s = (f32x16)(0.0f);
        uint4 f[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) f[i] = kt[i][lane ^ S::k_swizzle(i)];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < S::kSteps; i++) {
            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, f[i % kAhead]), q[i], s, 0, 0, 0);
            if (i + kAhead < S::kSteps) f[i % kAhead] = kt[i + kAhead][lane ^ S::k_swizzle(i + kAhead)];
            __builtin_amdgcn_sched_barrier(0);
        }
        const Part part = lds.part[buffer][2 * u + half];
        const int mine = min(part.count, seen);
        // a lane that sees no token of its block is not to meet the block's scales: they may be NaN
        const float ks = mine > 0 ? part.ks : 1.0f, vs = mine > 0 ? part.vs : 0.0f;
        const int slot = lane ^ S::v_swizzle(2 * u + half);
        auto v = [&](int i) { return lds.v[buffer][(i / 2 * S::kSubs + u) * 2 + i % 2][slot]; };
#pragma unroll
        for (int i = 0; i < kAhead; i++) f[i] = v(i);
        __builtin_amdgcn_sched_barrier(0);
        if (__any(mine < 16)) {
#pragma unroll
            for (int i = 0; i < 16; i++) s[i] = i < mine ? s[i] : -__builtin_inff();
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
        const float safe = m == -__builtin_inff() ? 0.0f : m;
        uint32_t p[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float e0 = exp2_fast(__builtin_fmaf(s[2 * i], ks, -safe)), e1 = exp2_fast(__builtin_fmaf(s[2 * i + 1], ks, -safe));
            l += e0 + e1;
            p[i] = pack_bf16(e0 * vs, e1 * vs);
        }
        const bf16x8 p0 = __builtin_bit_cast(bf16x8, make_uint4(p[0], p[1], p[2], p[3])),
                     p1 = __builtin_bit_cast(bf16x8, make_uint4(p[4], p[5], p[6], p[7]));
#pragma unroll
        for (int i = 0; i < 2 * S::kBlocks; i++) {
            o[i / 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, f[i % kAhead]), i % 2 ? p1 : p0,
                                                               o[i / 2], 0, 0, 0);
            if (i + kAhead < 2 * S::kBlocks) f[i % kAhead] = v(i + kAhead);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// Which tiles of the cache a workgroup takes of its row tile; pieces == 0: none.
struct Cut {
    int t0, t1, pieces;
};
__device__ __forceinline__ Cut cut_of(const RowsArgs& a, Seq seq, int row0, int piece, int tile_tokens) {
    if (row0 >= seq.n * a.group) return {0, 0, 0};
    const int last = min((row0 + kGroupRows - 1) / a.group, seq.n - 1);
    const int seen = a.causal ? min(seq.length, max(seq.length - seq.n + last + 1, 0)) : seq.length;
    const int tiles = (seen + tile_tokens - 1) / tile_tokens;
    const int pieces = max(min(a.pieces, (tiles + a.tiles_each - 1) / a.tiles_each), 1);
    const int size = (tiles + pieces - 1) / pieces;
    return {min(piece * size, tiles), min((piece + 1) * size, tiles), pieces};
}

// blockIdx.x: (row tile, latest tokens first as they see most of the cache; piece; kv head), blockIdx.y: sequence.
template <int TYPE, int D, bool PAGE>
__global__ __launch_bounds__(kThreads, 2) void k_attend_rows(RowsArgs a) {
    using S = Shape<D>;
    __shared__ Lds<D> lds;
    const int b = blockIdx.y, head = blockIdx.x % a.c.kv_heads, rest = blockIdx.x / a.c.kv_heads;
    const int piece = rest % a.pieces, row0 = (a.row_tiles - 1 - rest / a.pieces) * kGroupRows;
    const Seq seq = a.seq_uniform(b);
    const Cut cut = cut_of(a, seq, row0, piece, S::kTokens);
    if (piece >= cut.pieces) return;

    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, half = lane >> 5;
    const int row = row0 + 32 * wave + (lane & 31), token = row / a.group;
    const bool there = token < seq.n;
    const int limit = !there ? 0 : a.causal ? min(seq.length, max(seq.length - seq.n + token + 1, 0)) : seq.length;
    const uint16_t* qp = a.q + static_cast<int64_t>(seq.at + token) * a.q_token_stride +
                         static_cast<int64_t>(head * a.group + row % a.group) * a.q_head_stride + 8 * half;
    const int most = __builtin_amdgcn_readlane(limit, 31) > 0 ? __builtin_amdgcn_readlane(limit, 31) : seq.length;

    Stage<TYPE, D, PAGE> st;
    st.find(a, b, cut.t0 * S::kTokens);
    st.load(a, head, cut.t0 * S::kTokens, seq.length);
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

    st.store(a, lds, 0);
    st.find(a, b, (cut.t0 + 1) * S::kTokens);
    __syncthreads();
    for (int t = cut.t0; t < cut.t1; t++) {
        const int buffer = (t - cut.t0) & 1, base = t * S::kTokens;
        if (t + 1 < cut.t1) {
            st.load(a, head, base + S::kTokens, seq.length);
            st.find(a, b, base + 2 * S::kTokens);
        }
#pragma unroll
        for (int u = 0; u < S::kSubs; u++) {
            if (idle || base + 32 * u >= most) break;
            w.add(lds, buffer, u, limit - base - 32 * u - 16 * half);
        }
        if (t + 1 < cut.t1) st.store(a, lds, buffer ^ 1);
        __syncthreads();
    }
    const float m = w.m, l = other_half(w.l, true);
    f32x16(&o)[S::kBlocks] = w.o;
    if (!there) return;
    const int64_t place = static_cast<int64_t>(seq.at + token) * a.q_heads + head * a.group + row % a.group;
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

// Adds up the pieces of the row tiles that were cut: a wavefront a row, 32 rows a workgroup. blockIdx as above, with 32 rows
// for a row tile's 256 and no pieces.
constexpr int kMergeWaves = 4, kMergeRows = 32;
template <int D>
__global__ __launch_bounds__(kMergeWaves * 64) void k_attend_merge(RowsArgs a) {
    const int b = blockIdx.y, head = blockIdx.x % a.c.kv_heads, first = blockIdx.x / a.c.kv_heads * kMergeRows;
    const Seq seq = a.seq_uniform(b);
    const Cut cut = cut_of(a, seq, first / kGroupRows * kGroupRows, 0, Shape<D>::kTokens);
    if (cut.pieces < 2) return;
    constexpr int V = D / 64;
    typedef float Lane __attribute__((ext_vector_type(V)));
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t piece = static_cast<int64_t>(a.s.tokens) * a.q_heads;
    for (int row = first + wave; row < first + kMergeRows && row < seq.n * a.group; row += kMergeWaves) {
        const int64_t place = static_cast<int64_t>(seq.at + row / a.group) * a.q_heads + head * a.group + row % a.group;
        float2 ml[kMaxPieces];
        float top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < kMaxPieces; i++)
            if (i < cut.pieces) {
                ml[i] = a.partial_ml[i * piece + place];
                top = fmaxf(top, ml[i].x);
            }
        const float safe = top == -__builtin_inff() ? 0.0f : top;
        Lane sum = {};
        float l = 0.0f;
#pragma unroll
        for (int i = 0; i < kMaxPieces; i++)
            if (i < cut.pieces) {
                const float f = exp2_fast(ml[i].x - safe);
                l += ml[i].y * f;
                sum += *reinterpret_cast<const Lane*>(a.partial + (i * piece + place) * D + lane * V) * f;
            }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t* out = a.out + place * D + lane * V;
#pragma unroll
        for (int e = 0; e < V; e++) out[e] = __builtin_bit_cast(uint16_t, static_cast<__bf16>(sum[e] * inv));
    }
}

// How the row tiles' caches are cut. Calls of few row tiles would leave CUs idle, and in a causal one the last row tiles
// would run on alone: every row tile's cache is cut into pieces of a CU's share of the whole, where that is less.
struct RowsPlan {
    int64_t row_tiles, pieces, tiles_each;
};
RowsPlan rows_plan(const WlKvCache* c, int q_heads, const WlKvBatch* b, int64_t max_length) {
    const int64_t tokens = 8192 / c->head_dim, group = q_heads / c->kv_heads;
    const int64_t longest = std::max<int64_t>(1, std::min<int64_t>(max_length, int64_t{b->table_width} * c->page_tokens));
    const int64_t row_tiles = (b->max_count * group + kGroupRows - 1) / kGroupRows;
    const int64_t items = row_tiles * c->kv_heads * b->seqs;
    const int64_t most = (longest + tokens - 1) / tokens;  // tiles of the last row tile
    const int64_t mean = std::max<int64_t>(1, (longest - std::min<int64_t>(b->max_count, longest) / 2 + tokens - 1) / tokens);
    const int64_t each = std::max<int64_t>(4, (items * mean + kCus - 1) / kCus);
    return {row_tiles, std::min<int64_t>(kMaxPieces, (most + each - 1) / each), each};
}

}  // namespace

size_t attend_rows_workspace(const WlKvCache* c, int q_heads, const WlKvBatch* b, int64_t max_length) {
    const RowsPlan p = rows_plan(c, q_heads, b, max_length);
    if (p.pieces == 1) return 0;
    return static_cast<size_t>(p.pieces * b->tokens * q_heads) * (c->head_dim * sizeof(float) + sizeof(float2));
}

int launch_attend_rows(const WlKvCache* c, const AttendArgs& call, const WlKvBatch* b, int64_t max_length, void* workspace,
                       hipStream_t stream) {
    const RowsPlan p = rows_plan(c, call.q_heads, b, max_length);
    RowsArgs a;
    static_cast<AttendArgs&>(a) = call;
    a.partial = static_cast<float*>(workspace);
    a.partial_ml = reinterpret_cast<float2*>(a.partial + p.pieces * b->tokens * call.q_heads * c->head_dim);
    a.row_tiles = static_cast<int32_t>(p.row_tiles);
    a.pieces = static_cast<int32_t>(p.pieces);
    a.tiles_each = static_cast<int32_t>(p.tiles_each);
    const int64_t blocks = p.row_tiles * p.pieces * c->kv_heads;
    if (blocks >= (int64_t{1} << 31) || p.row_tiles * (kGroupRows / kMergeRows) * c->kv_heads >= (int64_t{1} << 31))
        return WL_EINVAL_SHAPE;
    const dim3 grid(static_cast<uint32_t>(blocks), b->seqs);
    const dim3 merge(static_cast<uint32_t>(p.row_tiles * (kGroupRows / kMergeRows) * c->kv_heads), b->seqs);
    auto run = [&](auto type, auto dim) {
        constexpr int T = decltype(type)::value, D = decltype(dim)::value;
        if (c->page_tokens >= Shape<D>::kTokens)
            k_attend_rows<T, D, true><<<grid, kThreads, 0, stream>>>(a);
        else
            k_attend_rows<T, D, false><<<grid, kThreads, 0, stream>>>(a);
        if (const int rc = launch_status()) return rc;
        if (p.pieces > 1) k_attend_merge<D><<<merge, kMergeWaves * 64, 0, stream>>>(a);
        return launch_status();
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
