// AdamW over many tensors in one launch, moments in fp32 or in 8 bits.
//
// Bound: HBM.  Per element: p read and written, g read, both moments read and written: 28 bytes with fp32 everywhere, 16 (+ 16 bytes a block of
// 256 for the scales) with 8-bit moments.  The tensors' addresses travel in the kernel's arguments (no table in device memory that a later
// call could overwrite while an earlier one still reads it); a block finds its tensor by comparing its number with the tensors' first blocks, a lane
// each.  One wave owns one block of 256 elements, 4 a lane, so a block's scale is a maximum over the wave and never leaves its registers.
#include "../common.h"
#include "../../../include/hsenet_ops.h"

namespace {

constexpr int BLOCK = HS_ADAMW_BLOCK;      // elements that share an 8-bit scale
constexpr int CHUNK = 16 * BLOCK;          // elements of a thread block: 4 waves, 4 blocks of 256 each
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
// elements [i, i + 4) of a tensor of n: whole where the tensor's four arrays are aligned for it, else one by one
template <int DT> __device__ __forceinline__ f32x4 get4(const void* p, long i, long n, bool whole) {
    f32x4 r = {0.f, 0.f, 0.f, 0.f};
    if (whole) {
        if constexpr (DT == HS_PREC_F32) r = *(const f32x4*)((const float*)p + i);
        else {
            const u32x2 u = *(const u32x2*)((const bf16_t*)p + i);
            constexpr bool F = DT == HS_PREC_F16;
            r[0] = unpack_lo<F>(u[0]); r[1] = unpack_hi<F>(u[0]); r[2] = unpack_lo<F>(u[1]); r[3] = unpack_hi<F>(u[1]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (i + e < n) r[e] = get1<DT>(p, i + e);
    }
    return r;
}
template <int DT> __device__ __forceinline__ void put4(void* p, long i, long n, bool whole, f32x4 r) {
    if (whole) {
        if constexpr (DT == HS_PREC_F32) *(f32x4*)((float*)p + i) = r;
        else {
            u32x2 u;
            u[0] = pack2h<DT == HS_PREC_F16>(r[0], r[1]); u[1] = pack2h<DT == HS_PREC_F16>(r[2], r[3]);
            *(u32x2*)((bf16_t*)p + i) = u;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (i + e < n) put1<DT>(p, i + e, r[e]);
    }
}
__device__ __forceinline__ unsigned get_codes(const void* p, long i, long n, bool whole) {
    if (whole) return *(const unsigned*)((const unsigned char*)p + i);
    unsigned r = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) if (i + e < n) r |= (unsigned)((const unsigned char*)p)[i + e] << (8 * e);
    return r;
}
__device__ __forceinline__ void put_codes(void* p, long i, long n, bool whole, unsigned c) {
    if (whole) { *(unsigned*)((unsigned char*)p + i) = c; return; }
#pragma unroll
    for (int e = 0; e < 4; ++e) if (i + e < n) ((unsigned char*)p)[i + e] = (unsigned char)(c >> (8 * e));
}
__device__ __forceinline__ float m_of(float s, unsigned codes, int e) {
    const float r = (float)(int)(signed char)(codes >> (8 * e)) * (1.0f / 127.0f);
    return s * (r * fabsf(r));
}
__device__ __forceinline__ float u_of(float s, unsigned codes, int e) {
    const float r = (float)((codes >> (8 * e)) & 255u) * (1.0f / 255.0f);
    return s * (r * r);
}
// largest of a block's values (all >= 0, or NaN) over the wave, and NaN where one of them is not finite
__device__ __forceinline__ float block_scale(f32x4 a) {
    const float s = wave_max(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])));
    const float sum = (a[0] + a[1]) + (a[2] + a[3]);       // NaN exactly where one of them is (they are >= 0)
    return __builtin_amdgcn_ballot_w64(sum != sum) || !(s < __builtin_inff()) ? __builtin_nanf("") : s;
}

template <int DT, bool BITS8>
__global__ __launch_bounds__(256) void adamw_kernel(Table a) {
    const int k = find_tensor(a);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    void* p = a.p[k];
    const void* g = a.g[k];
    void *m = a.m[k], *v = a.v[k];
    const long n = a.n[k];
    const float c1 = ((const float*)a.step[k])[1], c2 = ((const float*)a.step[k])[2];
    constexpr unsigned PA = DT == HS_PREC_F32 ? 15 : 7, SA = BITS8 ? 3 : 15;
    const bool aligned = !((((uintptr_t)p | (uintptr_t)g) & PA) | (((uintptr_t)m | (uintptr_t)v) & SA));
    const float step_size = a.lr * c1;
    const long base = (long)(blockIdx.x - a.first[k]) * CHUNK;
#pragma unroll
    for (int it = 0; it < CHUNK / (4 * BLOCK); ++it) {
        const long blk = base / BLOCK + it * 4 + wave, i = blk * BLOCK + lane * 4;
        if (blk * BLOCK >= n) break;
        const bool whole = aligned && i + 4 <= n;
        f32x4 pv = get4<DT>(p, i, n, whole);
        const f32x4 gv = get4<DT>(g, i, n, whole);
        f32x4 mv, vv;
        if constexpr (BITS8) {
            const float sm = a.ms[k][blk], su = a.vs[k][blk];
            const unsigned cm = get_codes(m, i, n, whole), cv = get_codes(v, i, n, whole);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                mv[e] = m_of(sm, cm, e);
                const float u = u_of(su, cv, e);
                vv[e] = u * u;
            }
        } else {
            mv = get4<HS_PREC_F32>(m, i, n, whole);
            vv = get4<HS_PREC_F32>(v, i, n, whole);
        }
        f32x4 am, uv;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            mv[e] = mv[e] * a.beta1 + gv[e] * a.rest1;
            vv[e] = vv[e] * a.beta2 + gv[e] * gv[e] * a.rest2;
            uv[e] = sqrtf(vv[e]);
            am[e] = fabsf(mv[e]);
            pv[e] = pv[e] * a.keep - step_size * mv[e] / (uv[e] * c2 + a.eps);
        }
        put4<DT>(p, i, n, whole, pv);
        if constexpr (BITS8) {
            const float sm = block_scale(am), su = block_scale(uv);
            const float im = sm > 0.f ? 1.0f / sm : 0.f, iu = su > 0.f ? 1.0f / su : 0.f;
            unsigned cm = 0, cv = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = (int)fminf(rintf(sqrtf(am[e] * im) * 127.0f), 127.0f);
                cm |= (unsigned)((mv[e] < 0.f ? -c : c) & 255) << (8 * e);
                int u = (int)fminf(rintf(sqrtf(uv[e] * iu) * 255.0f), 255.0f);
                u = uv[e] > 0.f ? max(u, 1) : u;
                cv |= (unsigned)(u & 255) << (8 * e);
            }
            put_codes(m, i, n, whole, cm);
            put_codes(v, i, n, whole, cv);
            if (lane == 0) { a.ms[k][blk] = sm; a.vs[k][blk] = su; }
        } else {
            put4<HS_PREC_F32>(m, i, n, whole, mv);
            put4<HS_PREC_F32>(v, i, n, whole, vv);
        }
    }
}

// the values that 8-bit moments stand for: m -> p of the table, v -> g
template <int DT>
__global__ __launch_bounds__(256) void adamw_moments_kernel(Table a) {
    const int k = find_tensor(a);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    void *om = a.p[k], *ov = (void*)a.g[k];
    const long n = a.n[k];
    constexpr unsigned PA = DT == HS_PREC_F32 ? 15 : 7;
    const bool aligned = !((((uintptr_t)om | (uintptr_t)ov) & PA) | (((uintptr_t)a.m[k] | (uintptr_t)a.v[k]) & 3));
    const long base = (long)(blockIdx.x - a.first[k]) * CHUNK;
#pragma unroll
    for (int it = 0; it < CHUNK / (4 * BLOCK); ++it) {
        const long blk = base / BLOCK + it * 4 + wave, i = blk * BLOCK + lane * 4;
        if (blk * BLOCK >= n) break;
        const bool whole = aligned && i + 4 <= n;
        const float sm = a.ms[k][blk], su = a.vs[k][blk];
        const unsigned cm = get_codes(a.m[k], i, n, whole), cv = get_codes(a.v[k], i, n, whole);
        f32x4 mv, vv;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            mv[e] = m_of(sm, cm, e);
            const float u = u_of(su, cv, e);
            vv[e] = u * u;
        }
        put4<DT>(om, i, n, whole, mv);
        put4<DT>(ov, i, n, whole, vv);
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
            if (a.count && blocks + more > 0x7fffffffu) break;
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
        if (t[i].n < 0 || t[i].n > ((int64_t)1 << 42)) return HS_ERR_SHAPE;
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
        if (t[i].n < 0 || t[i].n > ((int64_t)1 << 42)) return HS_ERR_SHAPE;
        if (!t[i].n) continue;
        if (bad(t[i].p, size) || bad(t[i].g, size) || bad(t[i].m, 1) || bad(t[i].v, 1) || bad(t[i].m_scale, 4) || bad(t[i].v_scale, 4)) return HS_ERR_ARG;
    }
    return over_tables(t, count, Table{}, [&](const Table& a, dim3 grid) {
        if (out_dtype == HS_PREC_F32) hipLaunchKernelGGL((adamw_moments_kernel<HS_PREC_F32>), grid, dim3(256), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL((adamw_moments_kernel<HS_PREC_BF16>), grid, dim3(256), 0, (hipStream_t)stream, a);
    });
}
