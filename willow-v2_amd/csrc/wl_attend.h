// What the attention kernels share: the call as they see it, bytes of the cache as bf16, sums over a wavefront.
//
// Every query row of a kv head's group (row = token * group + head in the group) meets the same keys and values, so the
// rows are the matrix core's second axis, and both products are taken transposed:
//   S^T = K Q^T    A = tokens of K, B = rows of q; the result's lane holds one row and several of the tokens, so a row's
//                  statistics are a lane's own values and one or two exchanges;
//   O^T = V^T P^T  A = dimensions of V over tokens, B = the weights, which the lanes hold in just the order in which this
//                  product takes them: no exchange and no LDS between the two products.
// That works because an operand's inner index may be any permutation as long as both operands share it, and the first
// product's token rows may be any tokens: they are dealt out so that a lane holds the scores of 16 consecutive tokens of a
// page, whose values are 16 consecutive bytes of V^T for each dimension.
// Bytes become bf16 exactly (|int8| <= 127 and e4m3 have at most 8 significant bits); a block's scale multiplies its
// scores in fp32, and V's scale multiplies the weights in fp32 before they are rounded to bf16 (the weights' one rounding: the
// matrix core takes them in no more bits at this rate).
#pragma once

#include <type_traits>

#include "wl_kv.h"

namespace wl {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTile = 64;       // tokens of a tile

// A sequence of the call: its first row, its rows, its tokens (as many as the table has pages for), and the position of its
// first row, which its whole length says.
struct Seq {
    int at, n, length, begin;

    // tokens that its row `i` may see
    __device__ __forceinline__ int seen(int i, bool causal) const {
        return causal ? min(length, max(begin + i + 1, 0)) : length;
    }
};

struct AttendArgs {
    KvLayer c;
    KvSeqs s;
    const int32_t* length;
    const uint16_t* q;
    int64_t q_token_stride, q_head_stride;
    uint16_t* out;
    int32_t q_heads, group;
    float scale_log2;  // scale * log2(e)
    int32_t causal, wide_q;

    __device__ __forceinline__ Seq seq(int b) const {
        Seq q;
        q.at = s.first(b);
        q.n = s.count(b, q.at);
        const int all = max(length[b], 0);
        q.length = min(all, s.table_width << c.page_shift);
        q.begin = all - q.n;
        return q;
    }
    // the same for a b that all lanes share, in scalar registers
    __device__ __forceinline__ Seq seq_uniform(int b) const {
        const Seq q = seq(b);
        return {__builtin_amdgcn_readfirstlane(q.at), __builtin_amdgcn_readfirstlane(q.n),
                __builtin_amdgcn_readfirstlane(q.length), __builtin_amdgcn_readfirstlane(q.begin)};
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

// Over the four lanes that hold one row's values: lanes 16, 32 and 48 apart.
template <typename F>
__device__ __forceinline__ float over_groups(float x, F f) {
    // a bit_cast straight from a vector's element reads element 0: each goes through a value
    uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t a0 = a[0], a1 = a[1];
    u = __builtin_bit_cast(uint32_t, f(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1)));
    const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t b0 = b[0], b1 = b[1];
    return f(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}
__device__ __forceinline__ float max_over_groups(float x) {
    return over_groups(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float sum_over_groups(float x) {
    return over_groups(x, [](float a, float b) { return a + b; });
}

// Inclusive sum over the wavefront's lanes, by row shifts and broadcasts.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
    int v = static_cast<int>(x);
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15, 31
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return static_cast<uint32_t>(v);
}
__device__ __forceinline__ uint32_t wave_sum(uint32_t x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Calls of more rows than the few-row form takes (wl_attend_rows.hip).
size_t attend_rows_workspace(const WlKvCache* c, int q_heads, const WlKvBatch* b, int64_t max_length);
bool attend_rows_fit(const WlKvCache* c, int q_heads, const WlKvBatch* b, int64_t max_length);  // launches hold the call
int launch_attend_rows(const WlKvCache* c, const AttendArgs& a, const WlKvBatch* b, int64_t max_length, void* workspace,
                       hipStream_t stream);

}  // namespace wl
