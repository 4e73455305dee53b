// Rotary positions with several axes: point j of a head is turned by the angle positions[axis[j]] * freq[j].
//
// Bound: HBM.  q and k are read and written once; the angles of a token are shared by all of its heads, so a block makes the cosines and
// sines of its few tokens once, in LDS, and then streams the heads' rows past them with 16-byte accesses: 4.4 to 5.3 TB/s over 8 to 16 volumes of 4097
// tokens, where a plain copy reaches 5.0.
// The angle is a product in 64 bits, reduced to a fraction of a turn there (a position of 10^6 would leave an fp32 angle 0.06 rad off);
// the fraction, at most 1/2, is rounded to 32 bits and goes through sincospi.
#include "../common.h"
#include <algorithm>
#include "../../../include/hsenet_ops.h"

namespace {

constexpr int MOST_TOKENS = 16, TARGET = 1024, MOST_STAGED = 512;     // of a block: tokens, vectors, vectors in LDS

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

enum { SPLIT, LINE, PAIRS, STAGED };

// A row (one head of one token) is cut into items of VEC columns that one thread moves.  SPLIT (halves, j and j + P): P / VEC items take VEC columns of
// the first half and the VEC facing them.  LINE (the same halves, where a row is a power of two of 16-byte vectors and turned whole): an item is one
// vector, so that a wave reads and writes whole lines, and the facing vector comes from the lane that holds it: 90 us against 94 for 16 x 4097 tokens of 24
// heads of 64 in bf16, 73 against 77 for 8 x 4097 of 20 heads of 128.  PAIRS (neighbours): an item is VEC / 2 pairs, the last ones maybe not to be turned.
// Columns behind the pairs follow as plain copies (none where a tensor is turned in place).  STAGED (halves whose P is no multiple of the vector): rows go
// through LDS, where a column's partner is read by itself: 8 x 4097 tokens of 24 heads of 64 with P = 29 in bf16 46 us, in single columns 134.
template <int DT, int VEC, int MODE>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
    typedef typename Elem<DT>::T T;
    typedef __attribute__((ext_vector_type(VEC))) T V;
    extern __shared__ float2 cs[];                       // [tpb][P]: cosine, sine
    __shared__ long at[MOST_TOKENS][4];                  // where each token's heads begin: x0, x1, y0, y1
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
    if (threadIdx.x < (unsigned)ntok) {
        const long tok = tok0 + threadIdx.x, b = tok / a.N, n = tok - b * a.N;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            at[threadIdx.x][i] = b * a.x_b[i] + n * a.x_n[i];
            at[threadIdx.x][2 + i] = b * a.y_b[i] + n * a.y_n[i];
        }
    }
    __syncthreads();
    if constexpr (MODE == STAGED) {
        constexpr int AT = MOST_STAGED / 256;
        __shared__ V stage[MOST_STAGED];
        const int items = a.dh / VEC, rows = ntok * a.heads, at_once = MOST_STAGED / items;
        const float inv_items = 1.0f / items;
        for (int r0 = 0; r0 < rows; r0 += at_once) {
            const int count = min(at_once, rows - r0) * items;
            V u[AT];
            T* y[AT];
            int it[AT], t[AT];
#pragma unroll
            for (int k = 0; k < AT; ++k) {
                const int i = threadIdx.x + k * 256;
                if (i >= count) continue;
                const int r = (int)((i + 0.5f) * inv_items), row = r0 + r;
                it[k] = i - r * items;
                t[k] = (int)((row + 0.5f) * a.inv_heads);
                int h = row - t[k] * a.heads;
                const int which = h >= a.heads0;
                h -= which ? a.heads0 : 0;
                u[k] = *(const V*)((const T*)(which ? a.x[1] : a.x[0]) + at[t[k]][which] + h * (which ? a.x_h[1] : a.x_h[0]) + it[k] * VEC);
                y[k] = (T*)(which ? a.y[1] : a.y[0]) + at[t[k]][2 + which] + h * (which ? a.y_h[1] : a.y_h[0]) + it[k] * VEC;
                stage[i] = u[k];
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < AT; ++k) {
                const int i = threadIdx.x + k * 256;
                if (i >= count) continue;
                const T* row = (const T*)(stage + (i - it[k]));
                V o;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const int c = it[k] * VEC + e, low = c < a.P;
                    const float2 r = cs[t[k] * a.P + min(low ? c : c - a.P, a.P - 1)];
                    const float own = Elem<DT>::get(u[k][e]), other = Elem<DT>::get(row[low ? c + a.P : c < 2 * a.P ? c - a.P : c]);
                    o[e] = c < 2 * a.P ? Elem<DT>::put(own * r.x + other * (low ? -r.y : r.y)) : u[k][e];
                }
                *(V*)y[k] = o;
            }
            __syncthreads();                                              // (the next rows go where these are)
        }
        return;
    }
    constexpr bool SINGLE = MODE == PAIRS && VEC == 1;           // rows of odd length: a pair is two single accesses
    const int turned = SINGLE ? a.P : MODE == SPLIT ? a.P / VEC : (2 * a.P + VEC - 1) / VEC;
    const int items = turned + (MODE == PAIRS && !SINGLE ? a.dh / VEC - turned : (a.dh - 2 * a.P) / VEC);
    const int total = ntok * a.heads * items;
    const float inv_items = 1.0f / items;
    // AT items of a thread at a time: their loads are all on the way before the first is used
    constexpr int AT = 2, W = SINGLE || MODE == SPLIT ? 2 : 1;                // vectors that an item reads
    for (int i0 = threadIdx.x; i0 < total; i0 += 256 * AT) {
        V u[AT][W];
        T* y[AT];
        int kind[AT], first[AT], second[AT];                              // 0: no item, 1: turned, 2: copied; columns; the angles' place
        const float2* w[AT];
#pragma unroll
        for (int k = 0; k < AT; ++k) {
            const int i = i0 + k * 256;
            kind[k] = 0;
            if (i >= total) continue;
            const int row = (int)((i + 0.5f) * inv_items), it = i - row * items;
            const int t = (int)((row + 0.5f) * a.inv_heads);
            int h = row - t * a.heads;
            const int which = h >= a.heads0;
            h -= which ? a.heads0 : 0;
            const T* x = (const T*)(which ? a.x[1] : a.x[0]) + at[t][which] + h * (which ? a.x_h[1] : a.x_h[0]);
            y[k] = (T*)(which ? a.y[1] : a.y[0]) + at[t][2 + which] + h * (which ? a.y_h[1] : a.y_h[0]);
            kind[k] = it < turned ? 1 : x != y[k] ? 2 : 0;
            first[k] = it < turned || (MODE == PAIRS && !SINGLE) ? (SINGLE ? 2 * it : it * VEC) : 2 * a.P + (it - turned) * VEC;
            second[k] = SINGLE ? first[k] + 1 : a.P + first[k];
            w[k] = cs + t * a.P + (SINGLE ? it : MODE == PAIRS ? 0 : MODE == LINE ? (it & (turned / 2 - 1)) * VEC : it * VEC);
            if (kind[k]) u[k][0] = *(const V*)(x + first[k]);
            if (W == 2 && kind[k] == 1) u[k][W - 1] = *(const V*)(x + second[k]);
        }
#pragma unroll
        for (int k = 0; k < AT; ++k) {
            V o, z;
            if constexpr (MODE == LINE) {
                typedef __attribute__((ext_vector_type(4))) int I;
                I v = __builtin_bit_cast(I, u[k][0]);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = __shfl_xor(v[e], turned / 2, 64);       // (a row's lanes take part together or not at all)
                z = __builtin_bit_cast(V, v);
            }
            if (kind[k] == 2) *(V*)(y[k] + first[k]) = u[k][0];
            if (kind[k] != 1) continue;
            if constexpr (MODE == LINE) {
                const float side = first[k] < a.P ? -1.0f : 1.0f;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float2 r = w[k][e];
                    o[e] = Elem<DT>::put(Elem<DT>::get(u[k][0][e]) * r.x + Elem<DT>::get(z[e]) * (side * r.y));
                }
            } else if constexpr (W == 1) {
                const int left = a.P - (first[k] >> 1);                   // pairs from here on
                const float2* r = w[k] + (first[k] >> 1);
                o = u[k][0];
                auto turn = [&](int e) {
                    const float p = Elem<DT>::get(u[k][0][e]), q = Elem<DT>::get(u[k][0][e + 1]);
                    o[e] = Elem<DT>::put(p * r[e >> 1].x - q * r[e >> 1].y);
                    o[e + 1] = Elem<DT>::put(p * r[e >> 1].y + q * r[e >> 1].x);
                };
                if (left >= VEC / 2) {
#pragma unroll
                    for (int e = 0; e < VEC; e += 2) turn(e);
                } else {
#pragma unroll
                    for (int e = 0; e < VEC - 2; e += 2)
                        if ((e >> 1) < left) turn(e);
                }
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float2 r = w[k][e];
                    const float p = Elem<DT>::get(u[k][0][e]), q = Elem<DT>::get(u[k][W - 1][e]);
                    o[e] = Elem<DT>::put(p * r.x - q * r.y);
                    z[e] = Elem<DT>::put(p * r.y + q * r.x);
                }
                *(V*)(y[k] + second[k]) = z;
            }
            *(V*)(y[k] + first[k]) = o;
        }
    }
}

template <int DT>
void launch(const RotaryArgs& a, int vec, int mode, hipStream_t s) {
    const dim3 grid((a.tokens + a.tpb - 1) / a.tpb), block(256);
    const size_t lds = (size_t)a.tpb * a.P * sizeof(float2);
    constexpr int FULL = DT == HS_PREC_F32 ? 4 : 8;
#define HS_ROT(VEC, MODE) hipLaunchKernelGGL((rotary_kernel<DT, VEC, MODE>), grid, block, lds, s, a)
    if (mode == LINE) HS_ROT(FULL, LINE);
    else if (mode == STAGED) HS_ROT(FULL, STAGED);
    else if (vec == FULL) { if (mode == PAIRS) HS_ROT(FULL, PAIRS); else HS_ROT(FULL, SPLIT); }
    else if (vec == 2) { if (mode == PAIRS) HS_ROT(2, PAIRS); else HS_ROT(2, SPLIT); }
    else { if (mode == PAIRS) HS_ROT(1, PAIRS); else HS_ROT(1, SPLIT); }
#undef HS_ROT
}

}  // namespace

extern "C" int hs_rotary_axes(const hs_rotary_desc* d, const void* x0, void* y0, const void* x1, void* y1, const void* positions,
                              const double* freq, const int32_t* axis, void* stream) {
    if (!d || d->struct_size != sizeof(hs_rotary_desc) || !x0 || !y0 || !positions || !freq || !axis) return HS_ERR_ARG;
    if (d->dtype < 0 || d->dtype > 2 || d->pos_dtype < 0 || d->pos_dtype > 2) return HS_ERR_ARG;
    if (d->B < 1 || d->N < 1 || d->heads[0] < 1 || d->heads[1] < 0 || d->pairs < 1 || d->pairs > HS_ROTARY_MAX_PAIRS || d->axes < 1) return HS_ERR_SHAPE;
    if (d->dh < 2 * d->pairs || d->dh > 4096 || (int64_t)d->B * d->N > 0x7fffffff - 64) return HS_ERR_SHAPE;
    if (d->heads[1] && (!x1 || !y1)) return HS_ERR_ARG;
    if (d->heads[0] > 4096 || d->heads[1] > 4096) return HS_ERR_SHAPE;
    const int heads = d->heads[0] + d->heads[1];
    if (heads > 4096 || (int64_t)heads * d->dh > (1 << 18)) return HS_ERR_SHAPE;      // a block's item numbers stay far inside fp32's whole numbers
    const int size = d->dtype == HS_PREC_F32 ? 4 : 2, full = 16 / size;
    RotaryArgs a = {};
    auto aligned = [&](int vec) {                                         // rows of whole vectors at whole vectors' places
        if (d->dh % vec) return false;
        for (int i = 0; i < (d->heads[1] ? 2 : 1); ++i) {
            const void *x = i ? x1 : x0, *y = i ? y1 : y0;
            if (((uintptr_t)x | (uintptr_t)y) % (vec * size)) return false;
            for (int64_t s : {d->x_b[i], d->x_n[i], d->x_h[i], d->y_b[i], d->y_n[i], d->y_h[i]})
                if (s % vec) return false;
        }
        return true;
    };
    const int P = d->pairs, vectors = d->dh / full;
    int vec = aligned(full) ? full : aligned(2) ? 2 : 1, mode = d->interleaved ? PAIRS : SPLIT;
    if (mode == SPLIT && vec == full && P % full == 0 && d->dh == 2 * P && vectors >= 2 && vectors <= 64 && !(vectors & (vectors - 1))) mode = LINE;
    if (mode == SPLIT && vec == full && P % full && vectors <= MOST_STAGED) mode = STAGED;
    if (mode == SPLIT && P % vec) vec = P % 2 == 0 ? 2 : 1;
    for (int i = 0; i < 2; ++i) {
        a.x[i] = i ? x1 : x0; a.y[i] = i ? y1 : y0;
        a.x_b[i] = d->x_b[i]; a.x_n[i] = d->x_n[i]; a.x_h[i] = d->x_h[i];
        a.y_b[i] = d->y_b[i]; a.y_n[i] = d->y_n[i]; a.y_h[i] = d->y_h[i];
    }
    a.pos = positions; a.freq = freq; a.axis = axis;
    a.pos_a = d->pos_a; a.pos_b = d->pos_b; a.pos_n = d->pos_n;
    a.N = d->N; a.tokens = d->B * d->N; a.heads0 = d->heads[0]; a.heads = heads; a.P = d->pairs; a.dh = d->dh; a.pos_dtype = d->pos_dtype;
    a.inv_heads = 1.0f / heads; a.inverse = d->inverse ? -1.0f : 1.0f;
    // tokens of a block: about TARGET vectors, while the grid still gives every CU several blocks
    const int items = mode == SPLIT ? (d->dh - 2 * P) / vec + 2 * (P / vec) : std::max(d->dh / vec, 1);
    a.tpb = std::max(1, std::min({TARGET / (heads * items), a.tokens / 2048, MOST_TOKENS}));
    if (a.tokens / a.tpb >= (1 << 24) - 1) return HS_ERR_SHAPE;                          // 2^32 threads
    hipStream_t s = (hipStream_t)stream;
    if (d->dtype == HS_PREC_BF16) launch<HS_PREC_BF16>(a, vec, mode, s);
    else if (d->dtype == HS_PREC_F16) launch<HS_PREC_F16>(a, vec, mode, s);
    else launch<HS_PREC_F32>(a, vec, mode, s);
    HS_CHECK_LAUNCH();
    return HS_OK;
}
