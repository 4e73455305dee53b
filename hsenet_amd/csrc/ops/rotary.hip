// Rotary positions with several axes: point j of a head is turned by the angle positions[axis[j]] * freq[j].
//
// Bound: HBM.  q and k are read and written once; the angles of a token are shared by all of its heads, so a block makes the cosines and
// sines of its few tokens once, in LDS, and then streams the heads' rows past them with 16-byte accesses.
// The angle is a product in 64 bits, reduced to a fraction of a turn there (a position of 10^6 would leave an fp32 angle 0.06 rad off);
// the fraction, at most 1/2, is rounded to 32 bits and goes through sincospi.
#include "../common.h"
#include "../../../include/hsenet_ops.h"

namespace {

struct RotaryArgs {
    const void* x[2];
    void* y[2];
    const void* pos;
    const double* freq;
    const int* axis;
    long x_b[2], x_n[2], x_h[2], y_b[2], y_n[2], y_h[2];
    long pos_a, pos_b, pos_n;
    int N, tokens, heads0, heads, P, dh, pos_dtype, tpb;
    float inv_heads, inverse;
};

template <int DT> struct Elem;
template <> struct Elem<HS_PREC_BF16> {
    typedef bf16_t T;
    static __device__ __forceinline__ float get(T v) { return bf2f(v); }
    static __device__ __forceinline__ T put(float f) { return f2bf(f); }
};
template <> struct Elem<HS_PREC_F16> {
    typedef bf16_t T;
    static __device__ __forceinline__ float get(T v) { return h2f<true>(v); }
    static __device__ __forceinline__ T put(float f) { return f2h<true>(f); }
};
template <> struct Elem<HS_PREC_F32> {
    typedef float T;
    static __device__ __forceinline__ float get(T v) { return v; }
    static __device__ __forceinline__ T put(float f) { return f; }
};

// A row (one head of one token) is cut into items of VEC columns that one thread moves: with split halves, P / VEC items take VEC columns of
// the first half and the VEC facing them; interleaved, 2 P / VEC items take VEC / 2 neighbouring pairs; the columns behind follow as plain
// copies (none where a tensor is turned in place).
template <int DT, int VEC, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
    typedef typename Elem<DT>::T T;
    typedef __attribute__((ext_vector_type(VEC))) T V;
    extern __shared__ float2 cs[];                       // [tpb][P]: cosine, sine
    const int tok0 = blockIdx.x * a.tpb, ntok = min(a.tpb, a.tokens - tok0);
    const float inv_p = 1.0f / a.P;
    for (int i = threadIdx.x; i < ntok * a.P; i += 256) {
        int t = (int)((i + 0.5f) * inv_p);               // i / P (i < 2^16: the quotient's error is far under 0.5 / P)
        const int j = i - t * a.P;
        const long tok = tok0 + t, b = tok / a.N, n = tok - b * a.N;
        const long at = a.axis[j] * a.pos_a + b * a.pos_b + n * a.pos_n;
        const double pos = a.pos_dtype == HS_POS_I32 ? (double)((const int*)a.pos)[at]
                         : a.pos_dtype == HS_POS_I64 ? (double)((const long long*)a.pos)[at] : (double)((const float*)a.pos)[at];
        double turns = pos * a.freq[j] * 0.15915494309189533577;
        turns -= rint(turns);
        float s, c;
        sincospif(2.0f * (float)turns, &s, &c);
        cs[i] = make_float2(c, s * a.inverse);
    }
    __syncthreads();
    constexpr bool SINGLE = INTER && VEC == 1;           // rows of odd length: a pair is two single accesses
    const int turned = SINGLE ? a.P : INTER ? 2 * a.P / VEC : a.P / VEC;
    const int tail = (a.dh - 2 * a.P) / VEC, items = turned + tail;
    const int total = ntok * a.heads * items;
    const float inv_items = 1.0f / items;
    for (int i = threadIdx.x; i < total; i += 256) {
        const int row = (int)((i + 0.5f) * inv_items), it = i - row * items;
        const int t = (int)((row + 0.5f) * a.inv_heads);
        int h = row - t * a.heads;
        const int which = h >= a.heads0;
        h -= which ? a.heads0 : 0;
        const int tok = tok0 + t, b = tok / a.N, n = tok - b * a.N;
        const T* x = (const T*)a.x[which] + b * a.x_b[which] + n * a.x_n[which] + h * a.x_h[which];
        T* y = (T*)a.y[which] + b * a.y_b[which] + n * a.y_n[which] + h * a.y_h[which];
        const float2* w = cs + t * a.P;
        if (it >= turned) {
            const int col = 2 * a.P + (it - turned) * VEC;
            if (x != y) *(V*)(y + col) = *(const V*)(x + col);
        } else if constexpr (SINGLE) {
            const float2 r = w[it];
            const float p = Elem<DT>::get(x[2 * it]), q = Elem<DT>::get(x[2 * it + 1]);
            y[2 * it] = Elem<DT>::put(p * r.x - q * r.y);
            y[2 * it + 1] = Elem<DT>::put(p * r.y + q * r.x);
        } else if constexpr (INTER) {
            const V u = *(const V*)(x + it * VEC);
            V o;
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
                const float2 r = w[(it * VEC + e) >> 1];
                const float p = Elem<DT>::get(u[e]), q = Elem<DT>::get(u[e + 1]);
                o[e] = Elem<DT>::put(p * r.x - q * r.y);
                o[e + 1] = Elem<DT>::put(p * r.y + q * r.x);
            }
            *(V*)(y + it * VEC) = o;
        } else {
            const V u = *(const V*)(x + it * VEC), v = *(const V*)(x + a.P + it * VEC);
            V o, z;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float2 r = w[it * VEC + e];
                const float p = Elem<DT>::get(u[e]), q = Elem<DT>::get(v[e]);
                o[e] = Elem<DT>::put(p * r.x - q * r.y);
                z[e] = Elem<DT>::put(p * r.y + q * r.x);
            }
            *(V*)(y + it * VEC) = o;
            *(V*)(y + a.P + it * VEC) = z;
        }
    }
}

template <int DT, bool INTER>
void launch(const RotaryArgs& a, int vec, hipStream_t s) {
    const dim3 grid((a.tokens + a.tpb - 1) / a.tpb), block(256);
    const size_t lds = (size_t)a.tpb * a.P * sizeof(float2);
    constexpr int FULL = DT == HS_PREC_F32 ? 4 : 8;
    if (vec == FULL) hipLaunchKernelGGL((rotary_kernel<DT, FULL, INTER>), grid, block, lds, s, a);
    else if (vec == 2) hipLaunchKernelGGL((rotary_kernel<DT, 2, INTER>), grid, block, lds, s, a);
    else hipLaunchKernelGGL((rotary_kernel<DT, 1, INTER>), grid, block, lds, s, a);
}

}  // namespace

extern "C" int hs_rotary_axes(const hs_rotary_desc* d, const void* x0, void* y0, const void* x1, void* y1, const void* positions,
                              const double* freq, const int32_t* axis, void* stream) {
    if (!d || d->struct_size != sizeof(hs_rotary_desc) || !x0 || !y0 || !positions || !freq || !axis) return HS_ERR_ARG;
    if (d->dtype < 0 || d->dtype > 2 || d->pos_dtype < 0 || d->pos_dtype > 2) return HS_ERR_ARG;
    if (d->B < 1 || d->N < 1 || d->heads[0] < 1 || d->heads[1] < 0 || d->pairs < 1 || d->pairs > HS_ROTARY_MAX_PAIRS || d->axes < 1) return HS_ERR_SHAPE;
    if (d->dh < 2 * d->pairs || d->dh > 4096 || (int64_t)d->B * d->N > 0x7fffffff - 64) return HS_ERR_SHAPE;
    if (d->heads[1] && (!x1 || !y1)) return HS_ERR_ARG;
    const int heads = d->heads[0] + d->heads[1];
    if (heads > 4096 || (int64_t)heads * d->dh > (1 << 18)) return HS_ERR_SHAPE;      // a block's item numbers stay far inside fp32's whole numbers
    const int size = d->dtype == HS_PREC_F32 ? 4 : 2, full = 16 / size;
    RotaryArgs a = {};
    auto fits = [&](int vec) {
        if (d->interleaved ? (2 * d->pairs) % vec : d->pairs % vec) return false;
        if ((d->dh - 2 * d->pairs) % vec) return false;
        for (int i = 0; i < (d->heads[1] ? 2 : 1); ++i) {
            const void *x = i ? x1 : x0, *y = i ? y1 : y0;
            if (((uintptr_t)x | (uintptr_t)y) % (vec * size)) return false;
            for (int64_t s : {d->x_b[i], d->x_n[i], d->x_h[i], d->y_b[i], d->y_n[i], d->y_h[i]})
                if (s % vec) return false;
        }
        return true;
    };
    const int vec = fits(full) ? full : fits(2) ? 2 : 1;
    for (int i = 0; i < 2; ++i) {
        a.x[i] = i ? x1 : x0; a.y[i] = i ? y1 : y0;
        a.x_b[i] = d->x_b[i]; a.x_n[i] = d->x_n[i]; a.x_h[i] = d->x_h[i];
        a.y_b[i] = d->y_b[i]; a.y_n[i] = d->y_n[i]; a.y_h[i] = d->y_h[i];
    }
    a.pos = positions; a.freq = freq; a.axis = axis;
    a.pos_a = d->pos_a; a.pos_b = d->pos_b; a.pos_n = d->pos_n;
    a.N = d->N; a.tokens = d->B * d->N; a.heads0 = d->heads[0]; a.heads = heads; a.P = d->pairs; a.dh = d->dh; a.pos_dtype = d->pos_dtype;
    a.inv_heads = 1.0f / heads; a.inverse = d->inverse ? -1.0f : 1.0f;
    a.tpb = 1;
    hipStream_t s = (hipStream_t)stream;
    if (d->dtype == HS_PREC_BF16) d->interleaved ? launch<HS_PREC_BF16, true>(a, vec, s) : launch<HS_PREC_BF16, false>(a, vec, s);
    else if (d->dtype == HS_PREC_F16) d->interleaved ? launch<HS_PREC_F16, true>(a, vec, s) : launch<HS_PREC_F16, false>(a, vec, s);
    else d->interleaved ? launch<HS_PREC_F32, true>(a, vec, s) : launch<HS_PREC_F32, false>(a, vec, s);
    HS_CHECK_LAUNCH();
    return HS_OK;
}
