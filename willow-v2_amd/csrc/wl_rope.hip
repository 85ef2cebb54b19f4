// Rotary positions with several axes (wl_rope), behind a norm of each head (wl_norm_rope).
#include <type_traits>

#include "wl_host.h"

namespace wl {
namespace {

constexpr int kRopeThreads = 256;

struct RopeArgs {
    WlRopeTensor q, k;
    const int64_t* positions;
    int64_t positions_stride;
    const double* inv_freq;
    int32_t sections[WL_MAX_ROPE_AXES];
    int32_t tokens, head_dim, half, axes, interleaved;
    float scale;
};

// The axis that frequency j belongs to.
__device__ __forceinline__ int axis_of(const RopeArgs& a, int j) {
    if (a.interleaved) {
        const int r = j % a.axes;
        return r > 0 && j < a.axes * a.sections[r] ? r : 0;
    }
    int axis = 0;
    for (int i = 0, end = 0; i + 1 < a.axes; i++) {
        end += a.sections[i];
        if (j >= end) axis = i + 1;
    }
    return axis;
}

// Cosine and sine of frequency j at a token's position, times the scale.
__device__ __forceinline__ float2 turn_of(const RopeArgs& a, int j, int token) {
    const double pos = static_cast<double>(a.positions[axis_of(a, j) * a.positions_stride + token]);
    const double turns = pos * a.inv_freq[j] * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(static_cast<float>(2.0 * (turns - __builtin_rint(turns))), &s, &c);
    return make_float2(a.scale * c, a.scale * s);
}

template <typename T>
__device__ __forceinline__ float load_value(const T* p);
template <>
__device__ __forceinline__ float load_value(const float* p) {
    return *p;
}
template <>
__device__ __forceinline__ float load_value(const uint16_t* p) {
    return __builtin_bit_cast(float, static_cast<uint32_t>(*p) << 16);
}
__device__ __forceinline__ void store_value(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_value(uint16_t* p, float x) {
    *p = __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
}

// One workgroup takes a token: the cosines and sines of its angles once into LDS, then every head's values by them, 32 lanes
// a head. The first eight heads' values are asked for before the angles are worked out (more of them help few tokens by less
// than 0.4 us and cost many 2 to 3). The angle is taken in turns in 64 bits (a
// position of a million at the first frequency is 1.6e5 turns, of which fp32 would keep 6 bits of the fraction) and only its
// fraction goes on in 32.
// VEC: values a thread moves at once (16 bytes where every row and the half split are that aligned, else one).
// Bound by reading and writing q and k once (4096 tokens of 16 + 2 heads of 256 in bf16, 75 MB: 20.9 us, 3.6 TB/s); a token
// a workgroup, since one with more runs through their heads one pass after the other (1024 tokens: 9.0 us, with two tokens a
// workgroup 10.8, with four 13.9; 4096 tokens: all within 0.6 us).
template <typename T, int VEC>
__global__ __launch_bounds__(kRopeThreads) void k_rope(RopeArgs a) {
    extern __shared__ float2 turn[];  // [half]: cos, sin
    struct alignas(sizeof(T) * VEC) Run {
        T v[VEC];
    };
    constexpr int kRows = kRopeThreads / 32, kEarly = 1;
    const int token = blockIdx.x, lane = threadIdx.x % 32;
    // a head: half / VEC pairs of runs, then what is not rotated
    const int pairs = a.half / VEC, units = pairs + (a.head_dim - 2 * a.half) / VEC, heads = a.q.heads + a.k.heads;
    struct Head {
        const T* in;
        T* out;
    };
    auto head_at = [&](int i) -> Head {
        const WlRopeTensor& x = i >= a.q.heads ? a.k : a.q;
        const int h = i >= a.q.heads ? i - a.q.heads : i;
        return {static_cast<const T*>(x.in) + token * x.in_token_stride + h * x.in_head_stride,
                static_cast<T*>(x.out) + token * x.out_token_stride + h * x.out_head_stride};
    };
    auto load = [&](const Head& x, int u, Run& lo, Run& hi) {
        lo = *reinterpret_cast<const Run*>(x.in + (u < pairs ? u : u + pairs) * VEC);
        if (u < pairs) hi = *reinterpret_cast<const Run*>(x.in + a.half + u * VEC);
    };
    auto finish = [&](const Head& x, int u, Run lo, Run hi) {
        if (u >= pairs) {
            if (x.in != x.out) *reinterpret_cast<Run*>(x.out + (u + pairs) * VEC) = lo;
            return;
        }
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const float2 cs = turn[u * VEC + e];
            const float p = load_value(lo.v + e), q = load_value(hi.v + e);
            store_value(lo.v + e, p * cs.x - q * cs.y);
            store_value(hi.v + e, q * cs.x + p * cs.y);
        }
        *reinterpret_cast<Run*>(x.out + u * VEC) = lo;
        *reinterpret_cast<Run*>(x.out + a.half + u * VEC) = hi;
    };
    Run lo[kEarly], hi[kEarly];
#pragma unroll
    for (int r = 0; r < kEarly; r++) {
        const int i = threadIdx.x / 32 + r * kRows;
        if (i < heads && lane < units) load(head_at(i), lane, lo[r], hi[r]);
    }
    for (int j = threadIdx.x; j < a.half; j += kRopeThreads) turn[j] = turn_of(a, j, token);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kEarly; r++) {
        const int i = threadIdx.x / 32 + r * kRows;
        if (i < heads && lane < units) finish(head_at(i), lane, lo[r], hi[r]);
    }
    for (int i = threadIdx.x / 32; i < heads; i += kRows)
        for (int u = i < kEarly * kRows ? lane + 32 : lane; u < units; u += 32) {
            Run x, y;
            load(head_at(i), u, x, y);
            finish(head_at(i), u, x, y);
        }
}

// The norm of each head before it turns. Weights: fp32 or bf16, null: all 1.
struct NormArgs {
    const void *q_weight, *k_weight;
    float eps, offset;  // offset: 1 where weights are zero-centred
    int32_t bf16;
};

// Heads of any size and alignment: as k_rope, a workgroup a token and 32 lanes a head, with a head's sum of squares over its lanes between reading and turning; the
// first run of values stays in registers meanwhile (all of a head up to 32 runs: 256 values of bf16, 128 of fp32), the others
// are read again. Both weights go into LDS beside the cosines. Bound by its instructions: every value takes its weight, cosine and sine
// from LDS, and rows that are not 16-byte aligned move value by value (4096 tokens of 16 + 2 heads of 256 in bf16 at odd strides 42 us;
// aligned heads of 320, 94 MB, 35; further runs of values asked for ahead of their turn: none the faster), which is why aligned heads of the
// usual sizes have k_norm_rope_lanes.
template <typename T, int VEC>
__global__ __launch_bounds__(kRopeThreads) void k_norm_rope(RopeArgs a, NormArgs n) {
    extern __shared__ float2 turn[];  // [half]: cos, sin; then the weights of q and of k [head_dim]
    float* weight = reinterpret_cast<float*>(turn + a.half);
    struct alignas(sizeof(T) * VEC) Run {
        T v[VEC];
    };
    constexpr int kRows = kRopeThreads / 32, kEarly = 1;
    const int token = blockIdx.x, lane = threadIdx.x % 32;
    const int pairs = a.half / VEC, units = pairs + (a.head_dim - 2 * a.half) / VEC, heads = a.q.heads + a.k.heads;
    struct Head {
        const T* in;
        T* out;
        const float* w;
    };
    auto head_at = [&](int i) -> Head {
        const bool is_k = i >= a.q.heads;
        const WlRopeTensor& x = is_k ? a.k : a.q;
        const int h = is_k ? i - a.q.heads : i;
        return {static_cast<const T*>(x.in) + token * x.in_token_stride + h * x.in_head_stride,
                static_cast<T*>(x.out) + token * x.out_token_stride + h * x.out_head_stride, weight + (is_k ? a.head_dim : 0)};
    };
    // unit u: run u of each half of what turns, then the rest
    auto load = [&](const Head& x, int u, Run& lo, Run& hi) {
        lo = *reinterpret_cast<const Run*>(x.in + (u < pairs ? u : u + pairs) * VEC);
        if (u < pairs) hi = *reinterpret_cast<const Run*>(x.in + a.half + u * VEC);
    };
    auto squares = [&](int u, const Run& lo, const Run& hi) {
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const float p = load_value(lo.v + e);
            s = __builtin_fmaf(p, p, s);
        }
        if (u < pairs)
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const float p = load_value(hi.v + e);
                s = __builtin_fmaf(p, p, s);
            }
        return s;
    };
    auto finish = [&](const Head& x, int u, Run lo, Run hi, float inv) {
        const int at = (u < pairs ? u : u + pairs) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; e++) {
            const float p = load_value(lo.v + e) * inv * x.w[at + e];
            if (u < pairs) {
                const float2 cs = turn[u * VEC + e];
                const float q = load_value(hi.v + e) * inv * x.w[a.half + at + e];
                store_value(lo.v + e, p * cs.x - q * cs.y);
                store_value(hi.v + e, q * cs.x + p * cs.y);
            } else {
                store_value(lo.v + e, p);
            }
        }
        *reinterpret_cast<Run*>(x.out + at) = lo;
        if (u < pairs) *reinterpret_cast<Run*>(x.out + a.half + at) = hi;
    };
    Run lo[kEarly], hi[kEarly];
#pragma unroll
    for (int r = 0; r < kEarly; r++) {
        const int i = threadIdx.x / 32 + r * kRows;
        lo[r] = hi[r] = {};
        if (i < heads && lane < units) load(head_at(i), lane, lo[r], hi[r]);
    }
    for (int j = threadIdx.x; j < 2 * a.head_dim; j += kRopeThreads) {
        const bool is_k = j >= a.head_dim;
        const void* w = is_k ? n.k_weight : n.q_weight;
        const int d = is_k ? j - a.head_dim : j;
        weight[j] = !w ? 1.0f : n.offset + (n.bf16 ? load_value(static_cast<const uint16_t*>(w) + d) : static_cast<const float*>(w)[d]);
    }
    for (int j = threadIdx.x; j < a.half; j += kRopeThreads) turn[j] = turn_of(a, j, token);
    __syncthreads();
    auto whole = [&](int i, const Run& first, const Run& second) {  // the head, of which the lanes hold 32 units
        const Head x = head_at(i);
        float sum = lane < units ? squares(lane, first, second) : 0.0f;
        for (int u = lane + 32; u < units; u += 32) {
            Run y, z = {};
            load(x, u, y, z);
            sum += squares(u, y, z);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor(sum, d);
        const float inv = 1.0f / sqrtf(sum / a.head_dim + n.eps);
        if (lane < units) finish(x, lane, first, second, inv);
        for (int u = lane + 32; u < units; u += 32) {
            Run y, z = {};
            load(x, u, y, z);
            finish(x, u, y, z, inv);
        }
    };
#pragma unroll
    for (int r = 0; r < kEarly; r++) {
        const int i = threadIdx.x / 32 + r * kRows;
        if (i < heads) whole(i, lo[r], hi[r]);
    }
    for (int i = threadIdx.x / 32 + kEarly * kRows; i < heads; i += kRows) {
        Run y = {}, z = {};
        if (lane < units) load(head_at(i), lane, y, z);
        whole(i, y, z);
    }
}

// 16 bytes of a head as fp32, and back.
template <typename T>
constexpr int kVec = 16 / sizeof(T);
template <typename T>
__device__ __forceinline__ void unpack(uint4 w, float (&x)[kVec<T>]) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            x[i] = __builtin_bit_cast(float, v[i]);
        } else {
            x[2 * i] = __builtin_bit_cast(float, v[i] << 16);
            x[2 * i + 1] = __builtin_bit_cast(float, v[i] & 0xFFFF0000u);
        }
    }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&x)[kVec<T>]) {
    typedef __bf16 Pair __attribute__((ext_vector_type(2)));
    typedef float Floats __attribute__((ext_vector_type(2)));
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4)
            v[i] = __builtin_bit_cast(uint32_t, x[i]);
        else
            v[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((Floats){x[2 * i], x[2 * i + 1]}, Pair));
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// The sum over a head's lanes, 8 to 64 of them side by side.
template <int LANES>
__device__ __forceinline__ float sum_over(float x) {
    auto dpp = [](float v, auto control) {
        return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(control)::value, 0xf, 0xf, true));
    };
    x = dpp(x, std::integral_constant<int, 0xB1>());   // neighbours
    x = dpp(x, std::integral_constant<int, 0x4E>());   // pairs
    x = dpp(x, std::integral_constant<int, 0x141>());  // four and four, mirrored
    if constexpr (LANES >= 16) x = dpp(x, std::integral_constant<int, 0x140>());  // eight and eight
    if constexpr (LANES >= 32) {
        const uint32_t u = __builtin_bit_cast(uint32_t, x);
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        const uint32_t r0 = r[0], r1 = r[1];
        x = __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1);
    }
    if constexpr (LANES >= 64) {
        const uint32_t u = __builtin_bit_cast(uint32_t, x);
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        const uint32_t r0 = r[0], r1 = r[1];
        x = __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1);
    }
    return x;
}

// Heads of 16 bytes for each of 8 to 64 lanes, everything aligned: a lane has the same dimensions of every head, and its
// partner's, in another lane, the ones that they turn with: out = (x a + partner's x b) / rms with a = weight cos and b = -+ the
// partner's weight sin (weight and 0 where nothing turns). These factors are worked out once for a token, into LDS, and a head
// costs a load, a sum over its lanes, its partner's 16 bytes, three operations a value and a store.
// Bound by reading and writing: 4096 tokens of 16 + 2 heads of 256 in bf16, 75 MB, 16 to 17 us (4.4 to 4.7 TB/s); 64 tokens 5.1 us in a
// graph, a chain of loads and the cosines.
// per: tokens of a workgroup, two of them in bf16 from 2049 tokens on, where one each would be more workgroups than the CUs hold at
// once (in a graph of ten calls on the same tensors, with one, two, four: 1024 tokens 7.4, 8.3, 10.1 us; 2048 10.6, 11.3, 12.6; 2300 13.1,
// 12.4, 14.2; 4096 18.3, 15.8, 17.1; 16384 81.6, 71.0, 69.2). fp32 keeps one: with one and two 2048 tokens take 15.9 and 16.4, 4096 27.2 and
// 26.5, 16384 127 and 124, from memory 4096 took 36.9 and 37.8.
template <typename T, int LANES>
__global__ __launch_bounds__(kRopeThreads) void k_norm_rope_lanes(RopeArgs a, NormArgs n, int per) {
    constexpr int V = kVec<T>, D = V * LANES, kGroups = kRopeThreads / LANES;
    extern __shared__ float4 tables[];  // factors a of q [per][D], of k, factors b of q, of k; then cosines and sines [per][half]
    float* fa = reinterpret_cast<float*>(tables);
    float* fb = fa + 2 * per * D;
    float2* turn = reinterpret_cast<float2*>(fb + 2 * per * D);
    const int first = blockIdx.x * per, tokens = min(per, a.tokens - first);
    const int unit = threadIdx.x % LANES, heads = a.q.heads + a.k.heads, pairs = a.half / V;
    const int other = unit < pairs ? unit + pairs : unit < 2 * pairs ? unit - pairs : unit;
    int token = 0, head = threadIdx.x / LANES;  // of this group
    auto forward = [&] {
        for (; head >= heads && token < tokens; head -= heads) token++;
    };
    auto load = [&] {
        const bool is_k = head >= a.q.heads;
        const T* p = static_cast<const T*>(is_k ? a.k.in : a.q.in) + (first + token) * (is_k ? a.k.in_token_stride : a.q.in_token_stride) +
                     (is_k ? head - a.q.heads : head) * (is_k ? a.k.in_head_stride : a.q.in_head_stride);
        return *reinterpret_cast<const uint4*>(p + unit * V);
    };
    forward();
    uint4 next = make_uint4(0, 0, 0, 0);
    if (token < tokens) next = load();
    for (int j = threadIdx.x; j < tokens * a.half; j += kRopeThreads) turn[j] = turn_of(a, j % a.half, first + j / a.half);
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += kRopeThreads) {
        const void* w = i < D ? n.q_weight : n.k_weight;
        const int d = i % D, j = d < a.half ? d : d - a.half, e = d < a.half ? d + a.half : j;
        const bool turns = d < 2 * a.half;
        auto weight = [&](int at) {
            return !w ? 1.0f : n.offset + (n.bf16 ? load_value(static_cast<const uint16_t*>(w) + at) : static_cast<const float*>(w)[at]);
        };
        const float own = weight(d), others = turns ? weight(e) : 0.0f;
        for (int t = 0; t < tokens; t++) {
            const float2 cs = turns ? turn[t * a.half + j] : make_float2(1.0f, 0.0f);
            const int to = (i < D ? t : per + t) * D + d;
            fa[to] = own * cs.x;
            fb[to] = d < a.half ? -others * cs.y : others * cs.y;
        }
    }
    __syncthreads();
    while (token < tokens) {
        const bool is_k = head >= a.q.heads;
        const uint4 w = next;
        const int at = (is_k ? per + token : token) * D + unit * V;
        T* out = static_cast<T*>(is_k ? a.k.out : a.q.out) + (first + token) * (is_k ? a.k.out_token_stride : a.q.out_token_stride) +
                 (is_k ? head - a.q.heads : head) * (is_k ? a.k.out_head_stride : a.q.out_head_stride);
        head += kGroups;
        forward();
        if (token < tokens) next = load();
        const uint4 p = make_uint4(__shfl(w.x, other, LANES), __shfl(w.y, other, LANES), __shfl(w.z, other, LANES), __shfl(w.w, other, LANES));
        float x[V], y[V], z[V];
        unpack<T>(w, x);
        unpack<T>(p, y);
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < V; e++) sum = __builtin_fmaf(x[e], x[e], sum);
        const float mean = sum_over<LANES>(sum) * (1.0f / D) + n.eps;
        float inv = __builtin_amdgcn_rsqf(mean);
        if (__any(!(mean > 1.0e-30f))) inv = mean > 1.0e-30f ? inv : 1.0f / sqrtf(mean);  // each head by its own mean alone
#pragma unroll
        for (int e = 0; e < V; e++) z[e] = inv * __builtin_fmaf(x[e], fa[at + e], y[e] * fb[at + e]);
        *reinterpret_cast<uint4*>(out + unit * V) = pack<T>(z);
    }
}

template <typename T, int VEC>
void launch_norm_rope(const RopeArgs& a, const NormArgs& n, hipStream_t stream) {
    auto lanes = [&](auto count) {
        const int per = sizeof(T) == 2 && a.tokens > 2048 ? 2 : 1;
        const size_t lds = (4 * sizeof(float) * a.head_dim + sizeof(float2) * a.half) * per;
        k_norm_rope_lanes<T, decltype(count)::value><<<(a.tokens + per - 1) / per, kRopeThreads, lds, stream>>>(a, n, per);
    };
    if constexpr (VEC > 1) {
        if (a.head_dim == 8 * VEC) return lanes(std::integral_constant<int, 8>());
        if (a.head_dim == 16 * VEC) return lanes(std::integral_constant<int, 16>());
        if (a.head_dim == 32 * VEC) return lanes(std::integral_constant<int, 32>());
        if (a.head_dim == 64 * VEC) return lanes(std::integral_constant<int, 64>());
    }
    k_norm_rope<T, VEC><<<a.tokens, kRopeThreads, sizeof(float2) * a.half + 2 * sizeof(float) * a.head_dim, stream>>>(a, n);
}

template <typename T, int VEC>
void launch_rope(const RopeArgs& a, hipStream_t stream) {
    k_rope<T, VEC><<<a.tokens, kRopeThreads, sizeof(float2) * a.half, stream>>>(a);
}

int check_rope_tensor(const WlRopeTensor* x, int size) {
    if (!x->in || !x->out) return WL_EINVAL_NULL;
    if (x->heads < 1 || x->heads > 65535 || x->reserved != 0) return WL_EINVAL_SHAPE;
    if (reinterpret_cast<uintptr_t>(x->in) % size || reinterpret_cast<uintptr_t>(x->out) % size) return WL_EINVAL_ALIGN;
    return WL_OK;
}

// Whether no two of the rows [t * token, + dim) + h * head (t < tokens, h < heads) share an element. Rows dt tokens and dh heads
// apart lie |dt token + dh head| apart; of each dh the nearest two dt are looked at.
bool rows_apart(int64_t token, int64_t head, int64_t tokens, int64_t heads, int64_t dim) {
    using wide = __int128;  // strides are the caller's: no product of them may overflow
    auto size = [](wide x) { return x < 0 ? -x : x; };
    const wide ts = size(token), hs = size(head);
    if ((heads == 1 || hs >= dim) && (tokens == 1 || ts >= hs * (heads - 1) + dim)) return true;  // all of a token, then the next
    if (tokens > 1 && ts < dim) return false;
    if (tokens == 1) return false;
    for (int64_t dh = 1; dh < heads; dh++) {
        const wide off = wide{head} * dh, near = -off / token;
        for (wide dt = near - 1; dt <= near + 1; dt++)
            if (size(dt) < tokens && size(off + dt * token) < dim) return false;
    }
    return true;
}

bool aligned16(const WlRopeTensor* x, int size) {
    const int64_t n = 16 / size;
    return reinterpret_cast<uintptr_t>(x->in) % 16 == 0 && reinterpret_cast<uintptr_t>(x->out) % 16 == 0 &&
           x->in_token_stride % n == 0 && x->in_head_stride % n == 0 && x->out_token_stride % n == 0 &&
           x->out_head_stride % n == 0;
}

// Checks a call's arguments and fills in the kernels' (a: all zeros); wide: 16 bytes may be moved at once.
int rope_args(RopeArgs& a, bool& wide, const WlRopeTensor* q, const WlRopeTensor* k, int dtype, int64_t tokens, int head_dim,
              int rotary_dim, const int64_t* positions, int64_t positions_stride, const double* inv_freq, int axes,
              const int32_t* sections_host, int interleaved, float scale) {
    if (!q || !positions || !inv_freq || !sections_host) return WL_EINVAL_NULL;
    if (dtype != WL_DTYPE_F32 && dtype != WL_DTYPE_BF16) return WL_EINVAL_DTYPE;
    const int size = dtype == WL_DTYPE_F32 ? 4 : 2;
    if (const int rc = check_rope_tensor(q, size)) return rc;
    if (k)
        if (const int rc = check_rope_tensor(k, size)) return rc;
    if (tokens < 1 || tokens >= (int64_t{1} << 32) / kRopeThreads || head_dim < 2 || head_dim > 1024 || rotary_dim < 2 ||
        rotary_dim > head_dim || rotary_dim % 2 || axes < 1 || axes > WL_MAX_ROPE_AXES)
        return WL_EINVAL_SHAPE;
    for (const WlRopeTensor* x : {q, k})
        if (x && !rows_apart(x->out_token_stride, x->out_head_stride, tokens, x->heads, head_dim)) return WL_EINVAL_SHAPE;
    // one tensor's result where the other is read or written
    if (k && (q->out == k->out || q->out == k->in || k->out == q->in)) return WL_EINVAL_OVERLAP;
    if (reinterpret_cast<uintptr_t>(positions) % 8 || reinterpret_cast<uintptr_t>(inv_freq) % 8) return WL_EINVAL_ALIGN;
    a.half = rotary_dim / 2;
    int64_t sum = 0;
    for (int i = 0; i < axes; i++) {
        const int n = sections_host[i];
        if (n < 0 || n > a.half) return WL_EINVAL_SHAPE;
        if (interleaved && i > 0 && n > 0 && i + axes * (n - 1) >= a.half) return WL_EINVAL_SHAPE;
        a.sections[i] = n;
        sum += n;
    }
    if (sum != a.half) return WL_EINVAL_SHAPE;
    a.q = *q;
    if (k) a.k = *k;
    a.positions = positions;
    a.positions_stride = positions_stride;
    a.inv_freq = inv_freq;
    a.tokens = static_cast<int32_t>(tokens);
    a.head_dim = head_dim;
    a.axes = axes;
    a.interleaved = interleaved != 0;
    a.scale = scale;
    const int vec = 16 / size;
    wide = a.half % vec == 0 && head_dim % vec == 0 && aligned16(q, size) && (!k || aligned16(k, size));
    return WL_OK;
}

}  // namespace
}  // namespace wl

using namespace wl;

extern "C" {

int wl_rope(const WlRopeTensor* q, const WlRopeTensor* k, int dtype, int64_t tokens, int head_dim, int rotary_dim,
            const int64_t* positions, int64_t positions_stride, const double* inv_freq, int axes, const int32_t* sections_host,
            int interleaved, float scale, void* stream) {
    RopeArgs a = {};
    bool wide;
    if (const int rc = rope_args(a, wide, q, k, dtype, tokens, head_dim, rotary_dim, positions, positions_stride, inv_freq, axes,
                                 sections_host, interleaved, scale))
        return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == WL_DTYPE_F32)
        wide ? launch_rope<float, 4>(a, st) : launch_rope<float, 1>(a, st);
    else
        wide ? launch_rope<uint16_t, 8>(a, st) : launch_rope<uint16_t, 1>(a, st);
    return launch_status();
}

int wl_norm_rope(const WlRopeTensor* q, const WlRopeTensor* k, int dtype, int64_t tokens, int head_dim, int rotary_dim,
                 const int64_t* positions, int64_t positions_stride, const double* inv_freq, int axes,
                 const int32_t* sections_host, int interleaved, float scale, const void* q_weight, const void* k_weight,
                 int weight_dtype, float eps, int zero_centered, void* stream) {
    RopeArgs a = {};
    bool wide;
    if (const int rc = rope_args(a, wide, q, k, dtype, tokens, head_dim, rotary_dim, positions, positions_stride, inv_freq, axes,
                                 sections_host, interleaved, scale))
        return rc;
    if (weight_dtype != WL_DTYPE_F32 && weight_dtype != WL_DTYPE_BF16) return WL_EINVAL_DTYPE;
    const int size = weight_dtype == WL_DTYPE_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(q_weight) % size || reinterpret_cast<uintptr_t>(k_weight) % size) return WL_EINVAL_ALIGN;
    if (!(eps >= 0.0f && eps < __builtin_inff())) return WL_EINVAL_SHAPE;
    const NormArgs n = {q_weight, k_weight, eps, zero_centered ? 1.0f : 0.0f, weight_dtype == WL_DTYPE_BF16};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == WL_DTYPE_F32)
        wide ? launch_norm_rope<float, 4>(a, n, st) : launch_norm_rope<float, 1>(a, n, st);
    else
        wide ? launch_norm_rope<uint16_t, 8>(a, n, st) : launch_norm_rope<uint16_t, 1>(a, n, st);
    return launch_status();
}

}  // extern "C"
