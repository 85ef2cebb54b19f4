// Rotary positions with several axes (wl_rope).
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
    for (int j = threadIdx.x; j < a.half; j += kRopeThreads) {
        const double pos = static_cast<double>(a.positions[axis_of(a, j) * a.positions_stride + token]);
        const double turns = pos * a.inv_freq[j] * 0.15915494309189533577;  // 1 / (2 pi)
        float s, c;
        sincospif(static_cast<float>(2.0 * (turns - __builtin_rint(turns))), &s, &c);
        turn[j] = make_float2(a.scale * c, a.scale * s);
    }
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

}  // namespace
}  // namespace wl

using namespace wl;

extern "C" int wl_rope(const WlRopeTensor* q, const WlRopeTensor* k, int dtype, int64_t tokens, int head_dim, int rotary_dim,
                       const int64_t* positions, int64_t positions_stride, const double* inv_freq, int axes,
                       const int32_t* sections_host, int interleaved, float scale, void* stream) {
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
    RopeArgs a = {};
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
    const bool wide = a.half % vec == 0 && head_dim % vec == 0 && aligned16(q, size) && (!k || aligned16(k, size));
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == WL_DTYPE_F32)
        wide ? launch_rope<float, 4>(a, st) : launch_rope<float, 1>(a, st);
    else
        wide ? launch_rope<uint16_t, 8>(a, st) : launch_rope<uint16_t, 1>(a, st);
    return launch_status();
}
