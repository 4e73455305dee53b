// AdamW over many tensors in one launch, moments in fp32 or in 8 bits.
//
// Bound: HBM.  Per element: p read and written, g read, both moments read and written: 28 bytes with fp32 everywhere, 16 (+ 16 bytes a block of
// 256 for the scales) with 8-bit moments.  125.8 M elements: fp32 659 us with fp32 moments, 388 with 8 bits; bf16 544 and 247: 5.1 to 5.3 TB/s (a plain
// copy: 5.0).  With 8-bit moments in bf16 the vector instructions come near the bytes: 4 elements a lane and correctly rounded roots, quotients and
// conversions took 394 us.  Accesses of 16 bytes, all of a block's in flight before the first is used.  The tensors' addresses travel in the kernel's arguments (no table in device memory that a later
// call could overwrite while an earlier one still reads it); a block finds its tensor by comparing its number with the tensors' first blocks, a lane
// each.  Half a wave owns one block of 256 elements, 8 a lane, so a block's scale is a maximum over 32 lanes and never leaves their registers.
#include "../common.h"
#include "../../../include/hsenet_ops.h"

namespace {

constexpr int BLOCK = HS_ADAMW_BLOCK;      // elements that share an 8-bit scale
constexpr int CHUNK = 16 * BLOCK;          // elements of a thread block
constexpr int TENSORS = 56;                // of one launch: 56 * 68 bytes + the rest stay under the 4 KiB of kernel arguments
constexpr int STEPS = 480;                 // step counters of one launch of the first kernel

struct Table {
    void* p[TENSORS]; const void* g[TENSORS]; void* m[TENSORS]; void* v[TENSORS];
    float* ms[TENSORS]; float* vs[TENSORS]; const int* step[TENSORS];
    long n[TENSORS];
    unsigned first[TENSORS + 1];           // first thread block of each tensor, and their number
    int count;
    float lr, beta1, beta2, rest1, rest2, eps, keep;       // rest = 1 - beta, keep = 1 - lr * weight_decay: differences taken in 64 bits
};
static_assert(sizeof(Table) <= 4000, "kernel arguments");
struct Steps { int* step[STEPS]; double beta1, beta2; int count; };

// one thread a tensor: raises the count t and leaves 1 / (1 - beta1^t) and 1 / sqrt(1 - beta2^t) beside it
__global__ void adamw_steps_kernel(Steps a) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= a.count) return;
    int* s = a.step[i];
    const int t = s[0] + 1;
    s[0] = t;
    ((float*)s)[1] = (float)(1.0 / (1.0 - pow(a.beta1, (double)t)));
    ((float*)s)[2] = (float)(1.0 / sqrt(1.0 - pow(a.beta2, (double)t)));
}

__device__ __forceinline__ int find_tensor(const Table& a) {
    const int lane = threadIdx.x & 63;
    const unsigned f = lane < a.count ? a.first[lane] : 0xffffffffu;
    return __popcll(__builtin_amdgcn_ballot_w64(f <= blockIdx.x)) - 1;
}

template <int DT> __device__ __forceinline__ float get1(const void* p, long i) {
    if constexpr (DT == HS_PREC_F32) return ((const float*)p)[i]; else return h2f<DT == HS_PREC_F16>(((const bf16_t*)p)[i]);
}
template <int DT> __device__ __forceinline__ void put1(void* p, long i, float f) {
    if constexpr (DT == HS_PREC_F32) ((float*)p)[i] = f; else ((bf16_t*)p)[i] = f2h<DT == HS_PREC_F16>(f);
}
template <int GAP> __device__ __forceinline__ long nth(long i, int e) { return i + (e >> 2) * GAP + (e & 3); }
// A lane's 8 elements of a tensor of n: two stretches of 4 that begin at i and GAP further, whole where its arrays are aligned for it, else one by one.
// In 16 bits they are side by side, one access of 16 bytes; in 32 bits each access of 16 bytes has its neighbours in the lanes beside it.
template <int DT, int GAP> __device__ __forceinline__ void get8(float (&r)[8], const void* p, long i, long n, bool whole) {
    if (whole) {
        if constexpr (DT == HS_PREC_F32) {
            const f32x4 x = *(const f32x4*)((const float*)p + i), y = *(const f32x4*)((const float*)p + i + GAP);
#pragma unroll
            for (int e = 0; e < 4; ++e) { r[e] = x[e]; r[4 + e] = y[e]; }
        } else {
            static_assert(GAP == 4, "one access");
            const u32x4 u = *(const u32x4*)((const bf16_t*)p + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) { r[2 * e] = unpack_lo<DT == HS_PREC_F16>(u[e]); r[2 * e + 1] = unpack_hi<DT == HS_PREC_F16>(u[e]); }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = nth<GAP>(i, e) < n ? get1<DT>(p, nth<GAP>(i, e)) : 0.f;
    }
}
template <int DT, int GAP> __device__ __forceinline__ void put8(void* p, long i, long n, bool whole, const float (&r)[8]) {
    if (whole) {
        if constexpr (DT == HS_PREC_F32) {
            *(f32x4*)((float*)p + i) = f32x4{r[0], r[1], r[2], r[3]};
            *(f32x4*)((float*)p + i + GAP) = f32x4{r[4], r[5], r[6], r[7]};
        } else {
            u32x4 u;
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = pack2h<DT == HS_PREC_F16>(r[2 * e], r[2 * e + 1]);
            *(u32x4*)((bf16_t*)p + i) = u;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) if (nth<GAP>(i, e) < n) put1<DT>(p, nth<GAP>(i, e), r[e]);
    }
}
template <int GAP> __device__ __forceinline__ u32x2 get_codes(const void* p, long i, long n, bool whole) {
    const unsigned char* c = (const unsigned char*)p;
    if (whole) return GAP == 4 ? *(const u32x2*)(c + i) : u32x2{*(const unsigned*)(c + i), *(const unsigned*)(c + i + GAP)};
    u32x2 r = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) if (nth<GAP>(i, e) < n) r[e >> 2] |= (unsigned)c[nth<GAP>(i, e)] << (8 * (e & 3));
    return r;
}
template <int GAP> __device__ __forceinline__ void put_codes(void* p, long i, long n, bool whole, u32x2 r) {
    unsigned char* c = (unsigned char*)p;
    if (whole) {
        if (GAP == 4) *(u32x2*)(c + i) = r;
        else { *(unsigned*)(c + i) = r[0]; *(unsigned*)(c + i + GAP) = r[1]; }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) if (nth<GAP>(i, e) < n) c[nth<GAP>(i, e)] = (unsigned char)(r[e >> 2] >> (8 * (e & 3)));
}
__device__ __forceinline__ void moments_of(float (&m)[8], float (&v)[8], u32x2 cm, u32x2 cv, float sm, float su) {
    sm *= 1.0f / (127 * 127);
    su *= 1.0f / (255 * 255);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float r = (float)(int)(signed char)(cm[e >> 2] >> (8 * (e & 3))), w = (float)((cv[e >> 2] >> (8 * (e & 3))) & 255u), u = su * (w * w);
        m[e] = sm * (r * fabsf(r));
        v[e] = u * u;
    }
}
// square root to a last place: the instruction takes what is below the normal numbers for 0
__device__ __forceinline__ float root(float x) {
    const bool tiny = x < 0x1p-96f;
    return __builtin_amdgcn_sqrtf(x * (tiny ? 0x1p64f : 1.0f)) * (tiny ? 0x1p-32f : 1.0f);
}
template <int CTRL> __device__ __forceinline__ unsigned moved(unsigned x) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true); }
// Largest of a block's values (all >= 0, or NaN) over its 32 lanes, and NaN where one of them is not finite: as whole numbers, the bits of what is not
// finite are larger than all others.
__device__ __forceinline__ float block_scale(const float (&a)[8]) {
    unsigned s = __builtin_bit_cast(unsigned, a[0]);
#pragma unroll
    for (int e = 1; e < 8; ++e) s = max(s, __builtin_bit_cast(unsigned, a[e]));
    s = max(s, moved<0xB1>(s));                                           // lanes that differ in bit 0, bit 1; the other 4 of 8; the other 8 of 16
    s = max(s, moved<0x4E>(s));
    s = max(s, moved<0x141>(s));
    s = max(s, moved<0x140>(s));
    s = max(s, (unsigned)__shfl_xor((int)s, 16, 64));
    return s < 0x7f800000u ? __builtin_bit_cast(float, s) : __builtin_nanf("");
}
// The nearest whole number of x f, below 2^22, in the low bits (two's complement) of a float whose last place is 1; and the low bytes of four of these.
__device__ __forceinline__ unsigned whole_bits(float x, float f) { return __builtin_bit_cast(unsigned, __builtin_fmaf(x, f, 12582912.0f)); }
__device__ __forceinline__ unsigned low_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
}

// A thread block's elements: two blocks of 256 for each half of a wave.
constexpr int TURNS = CHUNK / (256 * 8);
template <int DT> constexpr int GAP_OF = DT == HS_PREC_F32 ? BLOCK / 2 : 4;
struct Place { long i, blk; };
template <int GAP> __device__ __forceinline__ Place place_of(const Table& a, int k, int turn) {
    const long blk = (long)(blockIdx.x - a.first[k]) * (CHUNK / BLOCK) + turn * 8 + (threadIdx.x >> 5);
    return {blk * BLOCK + (threadIdx.x & 31) * (GAP == 4 ? 8 : 4), blk};
}

template <int DT, bool BITS8>
__global__ __launch_bounds__(256) void adamw_kernel(Table a) {
    const int k = find_tensor(a);
    void* p = a.p[k];
    const void* g = a.g[k];
    void *m = a.m[k], *v = a.v[k];
    const long n = a.n[k];
    constexpr int GAP = GAP_OF<DT>;
    const bool aligned = !((((uintptr_t)p | (uintptr_t)g) & 15) | (((uintptr_t)m | (uintptr_t)v) & (BITS8 ? 7 : 15)));
    float pv[TURNS][8], gv[TURNS][8], mv[TURNS][8], vv[TURNS][8], sm[TURNS], su[TURNS];
    u32x2 cm[TURNS], cv[TURNS];
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {                                     // everything is sent for before anything is used
        const Place at = place_of<GAP>(a, k, t);
        const bool whole = aligned && at.i + GAP + 4 <= n, some = at.blk * BLOCK < n;
        get8<DT, GAP>(pv[t], p, at.i, n, whole);
        get8<DT, GAP>(gv[t], g, at.i, n, whole);
        if constexpr (BITS8) {
            cm[t] = get_codes<GAP>(m, at.i, n, whole);
            cv[t] = get_codes<GAP>(v, at.i, n, whole);
            sm[t] = some ? a.ms[k][at.blk] : 0.f;
            su[t] = some ? a.vs[k][at.blk] : 0.f;
        } else {
            get8<HS_PREC_F32, GAP>(mv[t], m, at.i, n, whole);
            get8<HS_PREC_F32, GAP>(vv[t], v, at.i, n, whole);
        }
    }
    const float step_size = a.lr * ((const float*)a.step[k])[1], c2 = ((const float*)a.step[k])[2];
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {
        const Place at = place_of<GAP>(a, k, t);
        const bool whole = aligned && at.i + GAP + 4 <= n;
        float am[8], uv[8];
        if constexpr (BITS8) moments_of(mv[t], vv[t], cm[t], cv[t], sm[t], su[t]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            mv[t][e] = mv[t][e] * a.beta1 + gv[t][e] * a.rest1;
            vv[t][e] = vv[t][e] * a.beta2 + gv[t][e] * gv[t][e] * a.rest2;
            uv[e] = root(vv[t][e]);
            am[e] = fabsf(mv[t][e]);
            pv[t][e] = pv[t][e] * a.keep - step_size * mv[t][e] * __builtin_amdgcn_rcpf(uv[e] * c2 + a.eps);      // (to a last place)
        }
        put8<DT, GAP>(p, at.i, n, whole, pv[t]);
        if constexpr (BITS8) {
            const float Sm = block_scale(am), Su = block_scale(uv);
            const float im = Sm >= 0x1p-126f ? 1.0f / Sm : 0.f, iu = Su > 0.f ? 255.0f * 255 / Su : 0.f;      // (Su: 0 or at least 2^-75)
            unsigned wm[8], wv[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {                                 // (roots to a last place; what is not 0 is not taken for 0 in the second moment)
                wm[e] = whole_bits(copysignf(__builtin_amdgcn_sqrtf(am[e] * im), mv[t][e]), 127.0f);
                wv[e] = whole_bits(fmaxf(__builtin_amdgcn_sqrtf(uv[e] * iu), __builtin_amdgcn_fmed3f(uv[e] * 0x1p100f, 0.f, 1.0f)), 1.0f);
            }
            const u32x2 nm = {low_bytes(wm[0], wm[1], wm[2], wm[3]), low_bytes(wm[4], wm[5], wm[6], wm[7])};
            const u32x2 nv = {low_bytes(wv[0], wv[1], wv[2], wv[3]), low_bytes(wv[4], wv[5], wv[6], wv[7])};
            put_codes<GAP>(m, at.i, n, whole, nm);
            put_codes<GAP>(v, at.i, n, whole, nv);
            if ((threadIdx.x & 31) == 0 && at.i < n) { a.ms[k][at.blk] = Sm; a.vs[k][at.blk] = Su; }
        } else {
            put8<HS_PREC_F32, GAP>(m, at.i, n, whole, mv[t]);
            put8<HS_PREC_F32, GAP>(v, at.i, n, whole, vv[t]);
        }
    }
}

// the values that 8-bit moments stand for: m -> p of the table, v -> g
template <int DT>
__global__ __launch_bounds__(256) void adamw_moments_kernel(Table a) {
    const int k = find_tensor(a);
    void *om = a.p[k], *ov = (void*)a.g[k];
    const long n = a.n[k];
    constexpr int GAP = GAP_OF<DT>;
    const bool aligned = !((((uintptr_t)om | (uintptr_t)ov) & 15) | (((uintptr_t)a.m[k] | (uintptr_t)a.v[k]) & 7));
    u32x2 cm[TURNS], cv[TURNS];
    float sm[TURNS], su[TURNS];
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {
        const Place at = place_of<GAP>(a, k, t);
        const bool whole = aligned && at.i + GAP + 4 <= n, some = at.blk * BLOCK < n;
        cm[t] = get_codes<GAP>(a.m[k], at.i, n, whole);
        cv[t] = get_codes<GAP>(a.v[k], at.i, n, whole);
        sm[t] = some ? a.ms[k][at.blk] : 0.f;
        su[t] = some ? a.vs[k][at.blk] : 0.f;
    }
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {
        const Place at = place_of<GAP>(a, k, t);
        const bool whole = aligned && at.i + GAP + 4 <= n;
        float mv[8], vv[8];
        moments_of(mv, vv, cm[t], cv[t], sm[t], su[t]);
        put8<DT, GAP>(om, at.i, n, whole, mv);
        put8<DT, GAP>(ov, at.i, n, whole, vv);
    }
}

bool bad(const void* p, unsigned size) { return !p || (uintptr_t)p % size; }

// checks the entries, then launches `kernel` over them, TENSORS at a time
template <class F> int over_tables(const hs_adamw_tensor* t, int count, Table a, F launch) {
    for (int at = 0; at < count;) {
        a.count = 0;
        uint64_t blocks = 0;
        for (; at < count && a.count < TENSORS; ++at) {
            if (t[at].n == 0) continue;
            const uint64_t more = ((uint64_t)t[at].n + CHUNK - 1) / CHUNK;
            if (a.count && blocks + more >= 1u << 24) break;          // (256 threads each: below 2^32)
            const int k = a.count++;
            a.p[k] = t[at].p; a.g[k] = t[at].g; a.m[k] = t[at].m; a.v[k] = t[at].v;
            a.ms[k] = t[at].m_scale; a.vs[k] = t[at].v_scale; a.step[k] = t[at].step; a.n[k] = (long)t[at].n;
            a.first[k] = (unsigned)blocks;
            blocks += more;
        }
        if (!a.count) continue;
        a.first[a.count] = (unsigned)blocks;
        launch(a, dim3((unsigned)blocks));
        HS_CHECK_LAUNCH();
    }
    return HS_OK;
}

}  // namespace

extern "C" int hs_adamw_multi(const hs_adamw_tensor* t, int count, int dtype, int state_bits, double lr, double beta1, double beta2, double eps,
                              double weight_decay, void* stream) {
    if (!t || count < 1 || dtype < 0 || dtype > 2 || (state_bits != 8 && state_bits != 32)) return HS_ERR_ARG;
    if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0)) return HS_ERR_ARG;
    const unsigned size = dtype == HS_PREC_F32 ? 4 : 2;
    for (int i = 0; i < count; ++i) {
        if (t[i].n < 0 || t[i].n >= ((int64_t)CHUNK << 24) - CHUNK) return HS_ERR_SHAPE;
        if (bad(t[i].step, 16)) return HS_ERR_ARG;
        if (!t[i].n) continue;
        if (bad(t[i].p, size) || bad(t[i].g, size) || bad(t[i].m, state_bits / 8) || bad(t[i].v, state_bits / 8)) return HS_ERR_ARG;
        if (state_bits == 8 && (bad(t[i].m_scale, 4) || bad(t[i].v_scale, 4))) return HS_ERR_ARG;
    }
    hipStream_t s = (hipStream_t)stream;
    for (int at = 0; at < count;) {
        Steps a = {};
        a.beta1 = beta1; a.beta2 = beta2;
        for (; at < count && a.count < STEPS; ++at) a.step[a.count++] = t[at].step;
        hipLaunchKernelGGL(adamw_steps_kernel, dim3((a.count + 63) / 64), dim3(64), 0, s, a);
        HS_CHECK_LAUNCH();
    }
    Table a = {};
    a.lr = (float)lr; a.beta1 = (float)beta1; a.beta2 = (float)beta2; a.eps = (float)eps;
    a.rest1 = (float)(1 - beta1); a.rest2 = (float)(1 - beta2); a.keep = (float)(1 - lr * weight_decay);
    return over_tables(t, count, a, [&](const Table& a, dim3 grid) {
#define HS_ADAMW(DT)                                                                                          \
    do {                                                                                                      \
        if (state_bits == 8) hipLaunchKernelGGL((adamw_kernel<DT, true>), grid, dim3(256), 0, s, a);          \
        else hipLaunchKernelGGL((adamw_kernel<DT, false>), grid, dim3(256), 0, s, a);                         \
    } while (0)
        if (dtype == HS_PREC_BF16) HS_ADAMW(HS_PREC_BF16);
        else if (dtype == HS_PREC_F16) HS_ADAMW(HS_PREC_F16);
        else HS_ADAMW(HS_PREC_F32);
#undef HS_ADAMW
    });
}

extern "C" int hs_adamw_moments(const hs_adamw_tensor* t, int count, int out_dtype, void* stream) {
    if (!t || count < 1 || (out_dtype != HS_PREC_BF16 && out_dtype != HS_PREC_F32)) return HS_ERR_ARG;
    const unsigned size = out_dtype == HS_PREC_F32 ? 4 : 2;
    for (int i = 0; i < count; ++i) {
        if (t[i].n < 0 || t[i].n >= ((int64_t)CHUNK << 24) - CHUNK) return HS_ERR_SHAPE;
        if (!t[i].n) continue;
        if (bad(t[i].p, size) || bad(t[i].g, size) || bad(t[i].m, 1) || bad(t[i].v, 1) || bad(t[i].m_scale, 4) || bad(t[i].v_scale, 4)) return HS_ERR_ARG;
    }
    return over_tables(t, count, Table{}, [&](const Table& a, dim3 grid) {
        if (out_dtype == HS_PREC_F32) hipLaunchKernelGGL((adamw_moments_kernel<HS_PREC_F32>), grid, dim3(256), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL((adamw_moments_kernel<HS_PREC_BF16>), grid, dim3(256), 0, (hipStream_t)stream, a);
    });
}
