// Attention over the paged 8-bit cache (wl_kv_attend).
//
// Every query row of a kv head's group (row = token * group + head in the group) meets the same keys and values, so the
// rows are the matrix core's second axis. A wavefront takes 16 rows and tiles of 64 tokens, all in registers:
//   S^T = K Q^T    v_mfma_f32_16x16x32_bf16, A = 16 tokens of K, B = 16 rows of q; the result's lane holds one row
//                  (lane % 16) and four of the 16 tokens, so a row's statistics are a lane's own values and two exchanges
//                  over the four groups of lanes;
//   O^T = V^T P^T  A = 16 of V's dimensions over 32 tokens, B = the weights, which the lanes hold in just the order in
//                  which this product takes them: no exchange and no LDS between the two products.
// That works because an operand's inner index may be any permutation as long as both operands share it, and the first
// product's token rows may be any tokens: row m of its t-th product is token 16 (m / 4) + 4 t + m % 4 of the tile. A lane
// of group g then holds the scores of tokens 16 g .. 16 g + 15, and reads 16 consecutive bytes of V^T for each dimension.
// Bytes become bf16 exactly (|int8| <= 127 and e4m3 have at most 8 significant bits); a block's scale multiplies its
// scores in fp32, and V's scale multiplies the weights in fp32 before they are rounded to bf16.
#include <algorithm>
#include <type_traits>

#include "wl_kv.h"

namespace wl {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 64;       // tokens of a tile
constexpr int kRows = 16;       // query rows of a workgroup
constexpr int kFewWaves = 4;
constexpr int kFewGroups = 512; // workgroups of a split call: two a CU

struct AttendArgs {
    KvLayer c;
    KvSeqs s;
    const int32_t* length;
    const uint16_t* q;
    int64_t q_token_stride, q_head_stride;
    uint16_t* out;
    float* partial;   // [2 * workgroups][kRows][D]
    float2* partial_ml;  // [2 * workgroups][kRows]: maximum (in log2) and sum
    int32_t q_heads, group;
    float scale_log2;  // scale * log2(e)
    int32_t causal, wide_q;

    __device__ __forceinline__ int len(int b) const {
        const int64_t most = static_cast<int64_t>(s.table_width) * c.page_tokens;
        return static_cast<int>(min(static_cast<int64_t>(max(length[b], 0)), most));
    }
};

template <int TYPE>
__device__ __forceinline__ uint32_t two_bf16(uint32_t w, bool high) {
    if constexpr (TYPE == WL_KV_INT8) {
        const int i0 = static_cast<int8_t>(high ? w >> 16 : w), i1 = static_cast<int8_t>(high ? w >> 24 : w >> 8);
        const uint32_t f0 = __builtin_bit_cast(uint32_t, static_cast<float>(i0)),
                       f1 = __builtin_bit_cast(uint32_t, static_cast<float>(i1));
        return __builtin_amdgcn_perm(f1, f0, 0x07060302u);  // the upper halves: exact, 8 significant bits
    } else {
        return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)
                                                 : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
    }
}

// 8 bytes of the cache as bf16
template <int TYPE>
__device__ __forceinline__ bf16x8 eight_bf16(uint32_t lo, uint32_t hi) {
    uint4 r;
    r.x = two_bf16<TYPE>(lo, false);
    r.y = two_bf16<TYPE>(lo, true);
    r.z = two_bf16<TYPE>(hi, false);
    r.w = two_bf16<TYPE>(hi, true);
    return __builtin_bit_cast(bf16x8, r);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The bytes of w whose index is below n (0 .. 4)
__device__ __forceinline__ uint32_t keep_bytes(uint32_t w, int n) {
    return n >= 4 ? w : n <= 0 ? 0u : w & ((1u << (8 * n)) - 1u);
}

// One wavefront's share of rows [row0, row0 + 16) of (sequence b, kv head): its running maximum, its lanes' sums and O^T.
template <int TYPE, int D>
struct Rows {
    static constexpr int kChunks = D / 64;  // 16-byte loads of a K row, by four lanes each
    static constexpr int kDims = D / 16;    // 16-dimension blocks of V^T

    uint4 q[2 * kChunks];  // 8 bf16 each: this lane's row, dimensions 64 i + 16 g + 8 s ..
    f32x4 o[kDims];
    float m, l;
    int limit;  // tokens that this lane's row sees

    __device__ __forceinline__ void begin(const AttendArgs& a, int b, int head, int row0, int at, int n, int length) {
        const int lane = threadIdx.x & 63, g = lane >> 4, row = row0 + (lane & 15);
        const int token = row / a.group;
        m = -__builtin_inff();
        l = 0.0f;
        limit = 0;
#pragma unroll
        for (int i = 0; i < kDims; i++) o[i] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
        if (token < n) {
            limit = a.causal ? min(length, max(length - n + token + 1, 0)) : length;
            const uint16_t* p = a.q + static_cast<int64_t>(at + token) * a.q_token_stride +
                                static_cast<int64_t>(head * a.group + row % a.group) * a.q_head_stride + 16 * g;
            if (a.wide_q) {
#pragma unroll
                for (int i = 0; i < 2 * kChunks; i++)
                    q[i] = *reinterpret_cast<const uint4*>(p + 64 * (i / 2) + 8 * (i % 2));
            } else {
#pragma unroll
                for (int i = 0; i < 2 * kChunks; i++) {
                    const uint16_t* e = p + 64 * (i / 2) + 8 * (i % 2);
                    q[i] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2 * kChunks; i++) q[i] = make_uint4(0, 0, 0, 0);
        }
    }

    // tokens [base, base + 64) of the sequence
    __device__ __forceinline__ void tile(const AttendArgs& a, int b, int head, int base, int length) {
        const int lane = threadIdx.x & 63, g = lane >> 4, m16 = lane & 15;
        const int P = a.c.page_tokens;
        // K: this lane's tokens of the four products lie in the tile's 16-token group m16 / 4; V and the scores: group g
        const int kpos = base + 16 * (m16 >> 2), vpos = base + 16 * g;
        const int kpage = a.s.page(b, a.c.column(kpos), a.c.pages), vpage = a.s.page(b, a.c.column(vpos), a.c.pages);
        const uint8_t* kp = a.c.k + (a.c.block(max(kpage, 0), head) * P + a.c.within(kpos) + (m16 & 3)) * D + 16 * g;
        const uint8_t* vp = a.c.v + a.c.block(max(vpage, 0), head) * P * D + m16 * P + a.c.within(vpos);
        uint4 kr[4][kChunks], vr[kDims];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < kChunks; i++) kr[t][i] = *reinterpret_cast<const uint4*>(kp + 4 * t * D + 64 * i);
#pragma unroll
        for (int i = 0; i < kDims; i++) vr[i] = *reinterpret_cast<const uint4*>(vp + 16 * i * P);
        const float ks = a.c.k_scale[a.c.block(max(vpage, 0), head)] * a.scale_log2;
        const float vs = a.c.v_scale[a.c.block(max(vpage, 0), head)];
        const int mine = vpage < 0 ? 0 : min(max(limit - vpos, 0), 16);  // of this lane's 16 tokens, those that count

        f32x4 s[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            s[t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < kChunks; i++) {
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight_bf16<TYPE>(kr[t][i].x, kr[t][i].y),
                                                               __builtin_bit_cast(bf16x8, q[2 * i]), s[t], 0, 0, 0);
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight_bf16<TYPE>(kr[t][i].z, kr[t][i].w),
                                                               __builtin_bit_cast(bf16x8, q[2 * i + 1]), s[t], 0, 0, 0);
            }
        }
        float top = m;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                s[t][r] = 4 * t + r < mine ? s[t][r] * ks : -__builtin_inff();
                top = fmaxf(top, s[t][r]);
            }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
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
        for (int t = 0; t < 4; t++) {
            float e[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                e[r] = exp2_fast(s[t][r] - safe);
                l += e[r];
                // a token that does not count adds 0 whatever its block's scale is (it may be NaN)
                e[r] = 4 * t + r < mine ? e[r] * vs : 0.0f;
            }
            p[2 * t] = pack_bf16(e[0], e[1]);
            p[2 * t + 1] = pack_bf16(e[2], e[3]);
        }
        if (base + kTile > length || __any(vpage < 0)) {
            // bytes that nobody wrote may be NaN in e4m3, which a weight of 0 does not silence
            const int there = vpage < 0 ? 0 : min(max(length - vpos, 0), 16);
#pragma unroll
            for (int i = 0; i < kDims; i++) {
                vr[i].x = keep_bytes(vr[i].x, there);
                vr[i].y = keep_bytes(vr[i].y, there - 4);
                vr[i].z = keep_bytes(vr[i].z, there - 8);
                vr[i].w = keep_bytes(vr[i].w, there - 12);
            }
        }
        const bf16x8 p0 = __builtin_bit_cast(bf16x8, make_uint4(p[0], p[1], p[2], p[3])),
                     p1 = __builtin_bit_cast(bf16x8, make_uint4(p[4], p[5], p[6], p[7]));
#pragma unroll
        for (int i = 0; i < kDims; i++) {
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight_bf16<TYPE>(vr[i].x, vr[i].y), p0, o[i], 0, 0, 0);
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(eight_bf16<TYPE>(vr[i].z, vr[i].w), p1, o[i], 0, 0, 0);
        }
    }
};

template <int D>
struct JoinLds {
    float o[kFewWaves][kRows][D + 4];
    float m[kFewWaves][kRows], l[kFewWaves][kRows];
};

// The workgroup's four wavefronts over tiles [t0, t1) of rows [row0, row0 + 16); the rows are finished into out, or, with
// slot >= 0, left as a partial result.
template <int TYPE, int D>
__device__ __forceinline__ void attend_rows(const AttendArgs& a, JoinLds<D>& lds, int b, int head, int row0, int t0, int t1,
                                            int64_t slot) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, m16 = lane & 15;
    const int at = a.s.first(b), n = a.s.count(b, at), length = a.len(b);
    const int rows = static_cast<int>(min(static_cast<int64_t>(n) * a.group - row0, static_cast<int64_t>(kRows)));
    Rows<TYPE, D> r;
    r.begin(a, b, head, row0, at, n, length);
    for (int t = t0 + wave; t < t1; t += kFewWaves) r.tile(a, b, head, t * kTile, length);
    r.l += __shfl_xor(r.l, 16);
    r.l += __shfl_xor(r.l, 32);
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
        for (int i = 0; i < Rows<TYPE, D>::kDims; i++)
            *reinterpret_cast<f32x4*>(&lds.o[wave][m16][16 * i + 4 * g]) = r.o[i] * f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * (D / 4); i += kFewWaves * 64) {
        const int row = i / (D / 4), d = i % (D / 4) * 4;
        float m = lds.m[0][row];
#pragma unroll
        for (int w = 1; w < kFewWaves; w++) m = fmaxf(m, lds.m[w][row]);
        const float ms = m == -__builtin_inff() ? 0.0f : m;
        float l = 0.0f;
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kFewWaves; w++) {
            l += lds.l[w][row] * exp2_fast(lds.m[w][row] - ms);
            o += *reinterpret_cast<const f32x4*>(&lds.o[w][row][d]);
        }
        if (slot >= 0) {
            *reinterpret_cast<f32x4*>(a.partial + (slot * kRows + row) * D + d) = o;
            if (d == 0) a.partial_ml[slot * kRows + row] = make_float2(m, l);
        } else {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const int token = (row0 + row) / a.group, h = head * a.group + (row0 + row) % a.group;
            *reinterpret_cast<uint2*>(a.out + (static_cast<int64_t>(at + token) * a.q_heads + h) * D + d) =
                make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
        }
    }
    __syncthreads();
}

// Calls of more than 16 rows a sequence: a workgroup for each 16 rows, sequence and kv head.
template <int TYPE, int D>
__global__ __launch_bounds__(kFewWaves * 64, 2) void k_attend_tiles(AttendArgs a) {
    __shared__ JoinLds<D> lds;
    const int b = blockIdx.z, head = blockIdx.y, row0 = blockIdx.x * kRows;
    const int at = a.s.first(b), n = a.s.count(b, at), length = a.len(b);
    if (static_cast<int64_t>(row0) >= static_cast<int64_t>(n) * a.group) return;
    const int last = min((row0 + kRows - 1) / a.group, n - 1);
    const int seen = a.causal ? min(length, max(length - n + last + 1, 0)) : length;
    attend_rows<TYPE, D>(a, lds, b, head, row0, 0, (seen + kTile - 1) / kTile, -1);
}

// Calls of at most 16 rows a sequence are bound by reading the cache, so the cache is what is shared out: the tiles of all
// sequences and kv heads stand in one line, and every workgroup takes the same number of them in a row, wherever sequences
// begin and end. A (sequence, head) that lies in one share is finished there; of one that is cut, each share leaves a
// partial result, which k_attend_join adds up in order. A share has at most two such pieces, its first and its last.
struct Share {
    int64_t total, each;
};

__device__ __forceinline__ int seq_tiles(const AttendArgs& a, int b) {
    if (b >= a.s.seqs || a.s.count(b, a.s.first(b)) == 0) return 0;
    return max((a.len(b) + kTile - 1) / kTile, 1);  // a sequence without a token still has its rows to write
}

__device__ __forceinline__ Share share_of(const AttendArgs& a, int groups) {
    int64_t total = 0;
    for (int b = threadIdx.x & 63; b < a.s.seqs; b += 64) total += seq_tiles(a, b);
#pragma unroll
    for (int d = 32; d; d >>= 1) total += __shfl_xor(total, d);
    total *= a.c.kv_heads;
    return {total, max((total + groups - 1) / groups, static_cast<int64_t>(kFewWaves))};
}

// The sequence that tile `at` of the line belongs to, and the tiles before it (every lane gets both); at < total.
__device__ __forceinline__ int seq_at(const AttendArgs& a, int64_t at, int64_t& before) {
    const int lane = threadIdx.x & 63;
    before = 0;
    for (int b0 = 0;; b0 += 64) {
        int64_t sum = static_cast<int64_t>(seq_tiles(a, b0 + lane)) * a.c.kv_heads;
        const int64_t own = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t other = __shfl_up(sum, d);
            if (lane >= d) sum += other;
        }
        const uint64_t past = __ballot(before + sum > at);
        if (past) {
            const int i = __ffsll(static_cast<unsigned long long>(past)) - 1;
            before += __shfl(sum - own, i);
            return b0 + i;
        }
        if (b0 + 64 >= a.s.seqs) return a.s.seqs;
        before += __shfl(sum, 63);
    }
}

template <int TYPE, int D>
__global__ __launch_bounds__(kFewWaves * 64, 2) void k_attend_few(AttendArgs a) {
    __shared__ JoinLds<D> lds;
    const Share share = share_of(a, gridDim.x);
    int64_t at = blockIdx.x * share.each;
    const int64_t end = min(at + share.each, share.total);
    if (at >= end) return;
    int64_t before;
    int b = seq_at(a, at, before);
    bool first = true;
    while (at < end && b < a.s.seqs) {
        const int tiles = seq_tiles(a, b);
        if (tiles == 0) {
            b++;
            continue;
        }
        const int head = static_cast<int>((at - before) / tiles), t0 = static_cast<int>((at - before) % tiles);
        const int t1 = static_cast<int>(min(static_cast<int64_t>(tiles), t0 + (end - at)));
        const bool whole = t0 == 0 && t1 == tiles;
        attend_rows<TYPE, D>(a, lds, b, head, 0, t0, t1, whole ? -1 : 2 * static_cast<int64_t>(blockIdx.x) + !first);
        first = false;
        at += t1 - t0;
        if (t1 == tiles && head == a.c.kv_heads - 1) {
            before += static_cast<int64_t>(tiles) * a.c.kv_heads;
            b++;
        }
    }
}

// One row of one (sequence, kv head) that was cut: its partial results, in the order of its tokens. blockIdx: (sequence and
// head, row). A wavefront adds up every eighth part, then the eight sums are added in order.
constexpr int kJoinWaves = 8;
template <int D>
__global__ __launch_bounds__(kJoinWaves * 64) void k_attend_join(AttendArgs a, int groups) {
    __shared__ float2 ml[kJoinWaves];
    __shared__ float o[kJoinWaves][D];
    const int b = blockIdx.x / a.c.kv_heads, head = blockIdx.x % a.c.kv_heads, row = blockIdx.y;
    const int at = a.s.first(b), n = a.s.count(b, at);
    if (row >= n * a.group) return;
    const Share share = share_of(a, groups);
    int64_t before = 0;
    for (int i = threadIdx.x & 63; i < b; i += 64) before += seq_tiles(a, i);
#pragma unroll
    for (int d = 32; d; d >>= 1) before += __shfl_xor(before, d);
    const int tiles = seq_tiles(a, b);
    before = before * a.c.kv_heads + static_cast<int64_t>(head) * tiles;
    const int64_t w0 = before / share.each, w1 = (before + tiles - 1) / share.each;
    if (w0 == w1) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    constexpr int V = D / 64;  // values of a lane
    float m = -__builtin_inff(), l = 0.0f, acc[V] = {};
    for (int64_t w = w0 + wave; w <= w1; w += kJoinWaves) {
        // the first share holds this head's beginning behind whatever it began with; the others begin with this head
        const int64_t slot = 2 * w + (w == w0 && before != w0 * share.each);
        const float2 part = a.partial_ml[slot * kRows + row];
        const float top = fmaxf(m, part.x), safe = top == -__builtin_inff() ? 0.0f : top;
        const float f = exp2_fast(m - safe), fp = exp2_fast(part.x - safe);
        const float* p = a.partial + (slot * kRows + row) * D + lane * V;
#pragma unroll
        for (int i = 0; i < V; i++) acc[i] = acc[i] * f + p[i] * fp;
        l = l * f + part.y * fp;
        m = top;
    }
#pragma unroll
    for (int i = 0; i < V; i++) o[wave][lane * V + i] = acc[i];
    if (lane == 0) ml[wave] = make_float2(m, l);
    __syncthreads();
    if (threadIdx.x >= D) return;
    float top = ml[0].x;
    for (int w = 1; w < kJoinWaves; w++) top = fmaxf(top, ml[w].x);
    const float safe = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f, x = 0.0f;
    for (int w = 0; w < kJoinWaves; w++) {
        const float f = exp2_fast(ml[w].x - safe);
        sum += ml[w].y * f;
        x += o[w][threadIdx.x] * f;
    }
    const int token = row / a.group, h = head * a.group + row % a.group;
    const float y = sum == 0.0f ? 0.0f : x / sum;
    a.out[(static_cast<int64_t>(at + token) * a.q_heads + h) * D + threadIdx.x] =
        __builtin_bit_cast(uint16_t, static_cast<__bf16>(y));
}

// How a call is split: workgroups of the one-line form, 0 for the form by rows.
int few_groups(const WlKvCache* c, int q_heads, const WlKvBatch* b, int64_t max_length) {
    const int64_t rows = static_cast<int64_t>(b->max_count) * (q_heads / c->kv_heads);
    if (rows > kRows) return 0;
    const int64_t longest = std::max<int64_t>(1, std::min<int64_t>(max_length, int64_t{b->table_width} * c->page_tokens));
    const int64_t tiles = (longest + kTile - 1) / kTile * b->seqs * c->kv_heads;
    return static_cast<int>(std::min<int64_t>(kFewGroups, (tiles + kFewWaves - 1) / kFewWaves));
}

size_t partial_bytes(int groups, int D) {
    return groups > 1 ? static_cast<size_t>(2 * groups) * kRows * (D * sizeof(float) + sizeof(float2)) : 0;
}

int check_attend(const WlKvCache* cache, int q_heads, const WlKvBatch* batch, int64_t max_length) {
    if (const int rc = check_cache(cache)) return rc;
    if (const int rc = check_batch(batch)) return rc;
    if (q_heads < 1 || q_heads > 65535 || q_heads % cache->kv_heads != 0 || max_length < 0) return WL_EINVAL_SHAPE;
    if (static_cast<int64_t>(batch->max_count) * (q_heads / cache->kv_heads) >= (int64_t{1} << 31)) return WL_EINVAL_SHAPE;
    return WL_OK;
}

}  // namespace
}  // namespace wl

using namespace wl;

extern "C" {

size_t wl_kv_attend_workspace_bytes(const WlKvCache* cache, int q_heads, const WlKvBatch* batch, int64_t max_length) {
    if (check_attend(cache, q_heads, batch, max_length)) return 0;
    return partial_bytes(few_groups(cache, q_heads, batch, max_length), cache->head_dim);
}

int wl_kv_attend(const WlKvCache* cache, int layer, const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride,
                 int q_heads, const WlKvBatch* batch, const int32_t* length, int64_t max_length, float scale, int causal,
                 uint16_t* out, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check_attend(cache, q_heads, batch, max_length)) return rc;
    if (!q || !length || !out) return WL_EINVAL_NULL;
    if (layer < 0 || layer >= cache->layers || !(scale > -__builtin_inff() && scale < __builtin_inff())) return WL_EINVAL_SHAPE;
    const auto qb = reinterpret_cast<uintptr_t>(q);
    if (qb % 2 || reinterpret_cast<uintptr_t>(out) % 16 || reinterpret_cast<uintptr_t>(length) % 4) return WL_EINVAL_ALIGN;
    const int groups = few_groups(cache, q_heads, batch, max_length);
    const size_t need = partial_bytes(groups, cache->head_dim);
    if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)) return WL_EINVAL_WORKSPACE;
    AttendArgs a = {};
    a.c = layer_of(cache, layer);
    a.s = seqs_of(batch);
    a.length = length;
    a.q = q;
    a.q_token_stride = q_token_stride;
    a.q_head_stride = q_head_stride;
    a.out = out;
    a.partial = static_cast<float*>(workspace);
    a.partial_ml = reinterpret_cast<float2*>(a.partial + static_cast<size_t>(2 * groups) * kRows * cache->head_dim);
    a.q_heads = q_heads;
    a.group = q_heads / cache->kv_heads;
    a.scale_log2 = scale * 1.44269504088896340736f;
    a.causal = causal != 0;
    a.wide_q = qb % 16 == 0 && q_token_stride % 8 == 0 && q_head_stride % 8 == 0;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t rows = static_cast<int64_t>(batch->max_count) * a.group;
    auto run = [&](auto type, auto dim) {
        constexpr int T = decltype(type)::value, D = decltype(dim)::value;
        if (groups == 0) {
            const dim3 grid(static_cast<uint32_t>((rows + kRows - 1) / kRows), cache->kv_heads, batch->seqs);
            k_attend_tiles<T, D><<<grid, kFewWaves * 64, 0, st>>>(a);
            return launch_status();
        }
        k_attend_few<T, D><<<groups, kFewWaves * 64, 0, st>>>(a);
        if (const int rc = launch_status()) return rc;
        if (groups > 1) {
            k_attend_join<D><<<dim3(batch->seqs * cache->kv_heads, static_cast<uint32_t>(rows)), kJoinWaves * 64, 0, st>>>(
                a, groups);
            return launch_status();
        }
        return 0;
    };
    auto with_dim = [&](auto type) {
        if (cache->head_dim == 64) return run(type, std::integral_constant<int, 64>());
        if (cache->head_dim == 128) return run(type, std::integral_constant<int, 128>());
        return run(type, std::integral_constant<int, 256>());
    };
    if (cache->type == WL_KV_INT8) return with_dim(std::integral_constant<int, WL_KV_INT8>());
    return with_dim(std::integral_constant<int, WL_KV_E4M3>());
}

}  // extern "C"
