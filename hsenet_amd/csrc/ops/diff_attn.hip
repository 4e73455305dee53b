// Differential attention, o = P1 v - lam P2 v with P_m = softmax(scale q_m k_m^T): forward, split forward for few queries, backward.
//
// As in attn.hip, the index that the second product sums over lies on the accumulator's row (register) axis, so a score tile is, rounded and
// packed, the next matrix instruction's operand as it stands:
//   forward  S_m^T[key][query] = K_m Q_m^T -> P_m^T ;            O_m^T[dv][query] += V^T P_m^T        (both maps read one V fragment)
//   dq       S_m^T, dP^T = V dO^T          -> dS_m^T = P_m^T (dP^T - D_m) ;  dQ_m^T[d][query] += K_m^T dS_m^T
//   dk, dv   S_m[query][key] = Q_m K_m^T, dP = dO V^T ;          dV^T[dv][key] += dO^T (P1 - lam P2) ;  dK_m^T[d][key] += Q_m^T dS_m
// with D_m = sum over keys of P_m dP = dO . O_m (O_m: the map's own output, kept by the forward pass).  dP is one product for both maps, and dV too.
// Tiles of 32 rows are staged in LDS images R (common.h: 128-byte rows, read by rows and by columns): d / 32 images of a head pair's two keys
// (queries) side by side and d / 32 of its values (dO).
// P and dS are rounded to the operands' 16 bits for the matrix products.  That is a choice for speed: P in two numbers of 16 bits, as the split forward takes it
// where bandwidth leaves the matrix pipe room, would make 32 of the whole forward's 40 matrix instructions a step (d = 64) products with V, instead of 16
// of 24.  With o's own rounding it leaves bf16 outputs of normally distributed inputs 2.5e-3 off (o's rounding alone: 1.7e-3), fp16 3.2e-4; P's error is relative
// to each map, so that it grows beside o where the maps cancel.  The maps' outputs are kept in 16 bits, and D is summed from them.  Scores, sums, statistics,
// D and all accumulators are fp32.
#include "../common.h"
#include "../attn_util.h"
#include <type_traits>
#include "../../../include/hsenet_ops.h"

namespace {

constexpr float LOG2E = 1.44269504088896341f;
constexpr float NONE = -1e30f;                 // running maximum before the first visible key
constexpr float HEADROOM = 8.0f;               // a running maximum is kept until a score passes it by this many powers of two
constexpr int SHIFT16 = 4;                     // fp16: P and dS of the backward pass are held times 2^4

typedef __attribute__((ext_vector_type(2))) float f32x2;
constexpr int MOST_CHUNKS = 512;               // of a row's keys

struct Args {
    const bf16_t *q, *k, *v, *go;
    const float* lam;
    const int *q_start, *kv_len;
    bf16_t *o, *maps;
    float* lse;                                // [B][H][hi of both maps, lo of both][Nq] (put_lse); hi = +inf: no visible key
    f32x4 *sums, *stats;                       // parts of the forward pass with their rows' (reference, sums); of dk and dv; of dq
    float *D, *x2, *rc;                        // backward: D_m [B][H][2][Nq], D_2 in full precision [B][H][Nq], constants of the rows (diff_rows_kernel)
    bf16_t *dq, *dk, *dv;
    float* part;                               // split forward: numerators, then (maximum, sum)
    long q_b, q_n, q_h, k_b, k_n, k_h, v_b, v_n, v_h, go_b, go_n, go_h;
    int B, Nq, Nk, H, Hkv, G, causal, q_start0, lam_stride, nsplit, chunk, tiles, parts, cuts;
    float c2, scale;                           // scale * log2(e), scale
};

// Blocks are dealt round the 8 XCDs; a contiguous range of them to each lets the blocks of a key head share one L2.
__device__ __forceinline__ int block_order() {
    const int nb = gridDim.x, id = blockIdx.x, q = nb >> 3, r = nb & 7, x = id & 7;
    return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (id >> 3);
}
__device__ __forceinline__ int first_pos(const Args& a, int b) {
    const int s = a.q_start ? a.q_start[b] : a.q_start0;
    return min(max(s, -(1 << 30)), 1 << 30);
}
// number of leading keys that some query sees: the others are not touched (a cache may hold anything there)
__device__ __forceinline__ int key_count(const Args& a, int b) {
    const int len = a.kv_len ? min(max(a.kv_len[b], 0), a.Nk) : a.Nk;
    return a.causal ? max(0, min(len, first_pos(a, b) + a.Nq)) : len;
}
// number of leading keys that query i sees
__device__ __forceinline__ int visible(const Args& a, int len, int start, int i) { return a.causal ? max(0, min(len, start + i + 1)) : len; }
// number of leading queries that the causal mask leaves no key: their rows may hold anything (a batch padded on the left)
__device__ __forceinline__ int blind(const Args& a, int start) { return a.causal ? min(max(0, -start), a.Nq) : 0; }

// ---- a tile: ROWS rows of [two heads of d | VC value columns], sent straight into LDS images ------------------------------------------------------
// A wave's instruction moves 8 rows of an image, 16 bytes a lane; the image's swizzle is applied to the source.  It is written out because its builtin
// makes the compiler wait for it in front of the next LDS read, whatever that reads: issue() only starts the transfers, landed() waits for this
// wave's; a barrier behind landed() makes a tile readable to the others.
// The compiler does not look into the text, so the text itself holds the five wait states between a vector instruction that writes a scalar register (the
// descriptor and the offset come out of v_readfirstlane) and a memory instruction that reads it; M0 needs one of them.
#define HS_LDS_DMA_WAITS "s_mov_b32 m0, %0\n\ts_nop 3\n\t"
template <int D, int VC, int ROWS, int NW> struct Dma {
    static constexpr int PAIRS = D / 32, IMAGES = PAIRS + VC / 64, GROUPS = ROWS / 8, PER = IMAGES * GROUPS / NW;
    static_assert(PER * NW == IMAGES * GROUPS && (NW == 1 || NW % GROUPS == 0), "whole pieces");
    static constexpr int BASES = NW == 1 ? 2 : 1;                         // a lone wave moves even and odd groups of 8 rows, whose swizzles differ
    const char *x, *y;                         // the next tile's first row
    long x_n, y_n, x_h;
    int wave, row, left;                       // rows left from there on
    unsigned vx[BASES], vy[BASES];             // byte offsets of the lane's chunk in image 0 of the pair and of the values
    __device__ __forceinline__ void init(int wave_, int lane, const bf16_t* x_, long x_n_, long x_h_, const bf16_t* y_, long y_n_, int first, int end) {
        x_n = x_n_ * 2; y_n = y_n_ * 2; x_h = x_h_ * 2; wave = wave_;
        start(x_, y_, first, end);
        row = wave % GROUPS * 8 + (lane >> 3);
#pragma unroll
        for (int i = 0; i < BASES; ++i) {
            const int ch = (lane & 7) ^ swzR(row + 8 * i);
            vx[i] = (unsigned)(row * x_n + (D == 32 ? (ch >> 2) * x_h + (ch & 3) * 16 : ch * 16));
            vy[i] = (unsigned)(row * y_n + ch * 16);
        }
    }
    __device__ __forceinline__ void start(const bf16_t* x_, const bf16_t* y_, int first, int end) {
        x = (const char*)x_ + first * x_n;
        y = (const char*)y_ + first * y_n;
        left = end - first;
    }
    __device__ __forceinline__ void skip(int rows) {
        x += rows * x_n;
        y += rows * y_n;
        left -= rows;
    }
    static __device__ __forceinline__ u32x4 resource(const char* p) {
        const unsigned long long a = (unsigned long long)p;
        return u32x4{(unsigned)__builtin_amdgcn_readfirstlane((unsigned)a), (unsigned)__builtin_amdgcn_readfirstlane((unsigned)(a >> 32)), HS_MAX_RECORDS, 0x00020000u};
    }
    __device__ __forceinline__ void issue(unsigned lds) const { send<0, PER>(lds); }
    // pieces FROM to TO of the tile; rows at or behind `end` become zeros, and are not touched
    template <int FROM, int TO> __device__ __forceinline__ void send(unsigned lds) const {
        const u32x4 rx = resource(x), ry = resource(y);
#pragma unroll
        for (int i = FROM; i < TO; ++i) {
            const int g = i * NW + wave, image = g / GROUPS, group = g % GROUPS, more = NW == 1 ? group * 8 : 0;
            const bool pair = image < PAIRS;
            const int im = pair ? image : image - PAIRS;
            unsigned off = pair ? vx[BASES == 2 ? i & 1 : 0] : vy[BASES == 2 ? i & 1 : 0];
            off = row + more < left ? off : HS_OOB_OFF;
            const unsigned so = (unsigned)(pair ? more * x_n + (D == 32 ? 0 : D == 64 ? im * x_h : (im >> 1) * x_h + (im & 1) * 128) : more * y_n + im * 128);
            const unsigned at = lds + image * (ROWS * 128) + group * 1024;
            asm volatile(HS_LDS_DMA_WAITS "buffer_load_dwordx4 %1, %2, %3 offen lds"
                         :: "s"(__builtin_amdgcn_readfirstlane(at)), "v"(off), "s"(pair ? rx : ry), "s"(__builtin_amdgcn_readfirstlane(so)) : "memory");
        }
    }
    template <int LEFT = 0> static __device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(%0)" :: "i"(LEFT) : "memory"); }
};
// Where a lane's fragments lie in a tile: every fragment is one of these 8 addresses plus a constant, which becomes the LDS instruction's offset.
struct Lane {
    unsigned row[4], col[2][2];
    __device__ __forceinline__ void init(const char* smem, int lane) {
        const int h = lane >> 5, c = lane & 31, g = lane >> 4, p = lane & 3, q = (lane >> 2) & 3;
        const unsigned at = lds_addr(smem);
#pragma unroll
        for (int j = 0; j < 4; ++j) row[j] = at + offR(c, 2 * j + h);
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            const int col_ = d * 32 + 16 * (g & 1) + 4 * p;
            col[d][0] = at + offR(4 * h + q, col_ >> 3) + 8 * (p & 1);
            col[d][1] = at + offR(4 * h + q + 8, col_ >> 3) + 8 * (p & 1);
        }
    }
    __device__ __forceinline__ Lane at(unsigned off) const {
        Lane r = *this;
#pragma unroll
        for (int j = 0; j < 4; ++j) { r.row[j] += off; r.col[j >> 1][j & 1] += off; }
        return r;
    }
    // 16 columns from col_ of row lane % 32; 16 rows from r0, 32 columns from col_
    template <int ROWS> __device__ __forceinline__ bf16x8 rows16(int col_) const {
        return *(LDS_PTR(const bf16x8))(__UINTPTR_TYPE__)(row[(col_ & 63) >> 4] + (col_ >> 6) * (ROWS * 128));
    }
    template <int ROWS> __device__ __forceinline__ bf16x8 cols32(int r0, int col_) const {
        const unsigned o = (col_ >> 6) * (ROWS * 128) + r0 * 128;
        const int d = (col_ >> 5) & 1;
        return cat4(__builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(bf16x4))(__UINTPTR_TYPE__)(col[d][0] + o)),
                    __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(bf16x4))(__UINTPTR_TYPE__)(col[d][1] + o)));
    }
};
// Waits for the loads so far.  The compiler counts a loop's first pass into all others: operands still on their way at the loop's entry would make
// every pass wait for the newest loads, the next tile's.
__device__ __forceinline__ void arrived() { __builtin_amdgcn_s_waitcnt(0x0F70); }
__device__ __forceinline__ bf16x8 load8(const bf16_t* p) { return *(const bf16x8*)p; }
template <bool F16> __device__ __forceinline__ void store4(bf16_t* p, float a, float b, float c, float d) {
    u32x2 u;
    u[0] = pack2h<F16>(a, b); u[1] = pack2h<F16>(c, d);
    *(u32x2*)p = u;
}
// the rows (columns of the accumulators) of NB accumulators, times mul, to 32 NB consecutive columns
template <bool F16, int NB> __device__ __forceinline__ void store_rows(bf16_t* p, const f32x16 (&acc)[NB], float mul, int h) {
#pragma unroll
    for (int db = 0; db < NB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            store4<F16>(p + db * 32 + 8 * g + 4 * h, acc[db][4 * g] * mul, acc[db][4 * g + 1] * mul, acc[db][4 * g + 2] * mul, acc[db][4 * g + 3] * mul);
}
template <int NB> __device__ __forceinline__ void clear(f32x16 (&acc)[NB]) {
#pragma unroll
    for (int i = 0; i < NB; ++i) acc[i] = zero16();
}

// One map's softmax over 32 keys of a query is taken against a reference m: the largest score so far up to HEADROOM.  It moves,
// and l and the numerators with it, only when a score passes it by more, which after the first tiles is rare; any reference gives the same
// quotient.  It is one number for both halves of a query's lanes (they hold different keys of one product).
// The numerators are divided by the sum of P as rounded for their product, so that a query of few keys gets their values' average with no error of P's;
// a backward pass wants the sum of P itself (SUMS 2).
template <int SUMS, int NB>
__device__ __forceinline__ void follow_max(const f32x16& s, float c2, float& m, float (&l)[SUMS], f32x16 (&o)[NB]) {
    float mx = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
    mx *= c2;
    if (__builtin_amdgcn_ballot_w64(mx > m + HEADROOM)) {
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float mn = fmaxf(m, ceilf(mx)), alpha = __builtin_amdgcn_exp2f(m - mn);
#pragma unroll
        for (int i = 0; i < SUMS; ++i) l[i] *= alpha;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][r] *= alpha;
            __builtin_amdgcn_sched_barrier(0);
        }
        m = mn;
    }
}
// the reference that the first 32 keys of a row give
__device__ __forceinline__ float first_max(const f32x16& s, float c2) {
    float mx = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
    mx *= c2;
    return fmaxf(NONE, ceilf(fmaxf(mx, __shfl_xor(mx, 32, 64))));
}
template <bool F16> __device__ __forceinline__ float add2(unsigned pair, float sum) {      // sum + both halves, in fp32
    typedef __attribute__((ext_vector_type(2))) __bf16 b2;
    typedef __attribute__((ext_vector_type(2))) _Float16 h2;
    if constexpr (F16) return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, pair), h2{(_Float16)1.f, (_Float16)1.f}, sum, false);
    else return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, pair), b2{(__bf16)1.f, (__bf16)1.f}, sum, false);
}
// numerators, in s as they are and in p rounded for the product
template <bool F16>
__device__ __forceinline__ void softmax_weights(f32x16& s, float c2, float m, bf16x8 (&p)[2]) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c2, -m));
    p[0] = pack8<F16>(s, 0); p[1] = pack8<F16>(s, 1);
}
// numerators in two numbers of 16 bits, value and what its rounding left, and their sum
template <bool F16>
__device__ __forceinline__ void two_part_weights(f32x16& s, float c2, float m, float& l, bf16x8 (&p)[2], bf16x8 (&rest)[2]) {
    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c2, -m));
        part[r & 3] += s[r];
    }
    l += (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
    for (int sp = 0; sp < 2; ++sp) {
        p[sp] = pack8<F16>(s, sp);
        const u32x4 w = __builtin_bit_cast(u32x4, p[sp]);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[8 * sp + e] -= e & 1 ? unpack_hi<F16>(w[e >> 1]) : unpack_lo<F16>(w[e >> 1]);
        rest[sp] = pack8<F16>(s, sp);
    }
}
__device__ __forceinline__ float exp2_neg(float x) { return __builtin_amdgcn_exp2f(-x); }
// What the backward pass needs of a row's softmax: P = 2^(c2 s - hi - lo), hi whole (the reference m is), 0 <= lo < 1.  One fp32 number of their sum's
// size would put a common error of 5e-7 on all of a row's P, which the sum that is lam's gradient would keep.
__device__ __forceinline__ void put_lse(float* p, long next, float m, float l) {
    const int e = l > 0.f && l < __builtin_inff() ? __builtin_amdgcn_frexp_expf(l) - 1 : 0;
    p[0] = l == 0.f ? __builtin_inff() : m + (float)e;
    p[next] = l == 0.f ? 0.f : __builtin_amdgcn_logf(__builtin_amdgcn_ldexpf(l, -e));
}

// The parts of a step of one wave's 32 queries against 32 keys: both maps' scores, their softmax (lim: visible keys of the lane's query, counted from
// the step's first; mask: some of the 32 may not be visible), the products with V.
template <int D, bool F16, int ROWS>
__device__ __forceinline__ void scores(const Lane& f, const bf16x8 (&qf)[2][D / 16], f32x16 (&s)[2]) {
    constexpr int N = D / 8, AHEAD = 4;                                   // fragments are read AHEAD products before their use
    bf16x8 x[AHEAD];
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) x[n] = f.template rows16<ROWS>(n * 16);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int i = n / (D / 16), ks = n % (D / 16);
        s[i] = mfma32<F16>(x[n % AHEAD], qf[i][ks], ks ? s[i] : zero16());
        if (n + AHEAD < N) x[n % AHEAD] = f.template rows16<ROWS>((n + AHEAD) * 16);
        __builtin_amdgcn_sched_barrier(0);
    }
}
// scores of both maps and dP: the tile's columns are [keys | values] against q and dO
template <int D, bool F16, int ROWS>
__device__ __forceinline__ void scores_dp(const Lane& f, const bf16x8 (&qf)[2][D / 16], const bf16x8 (&gf)[D / 8], f32x16 (&s)[2], f32x16& dp) {
    constexpr int N = D / 4, AHEAD = 4;
    bf16x8 x[AHEAD];
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) x[n] = f.template rows16<ROWS>(n * 16);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int i = n / (D / 16), ks = n % (D / 16);
        if (i < 2) s[i & 1] = mfma32<F16>(x[n % AHEAD], qf[i & 1][ks], ks ? s[i & 1] : zero16());
        else dp = mfma32<F16>(x[n % AHEAD], gf[n - D / 8], n > D / 8 ? dp : zero16());
        if (n + AHEAD < N) x[n % AHEAD] = f.template rows16<ROWS>((n + AHEAD) * 16);
        __builtin_amdgcn_sched_barrier(0);
    }
}
__device__ __forceinline__ void mask_keys(f32x16 (&s)[2], int lim, int h) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[i][r] = acc_row(r, h) < lim ? s[i][r] : -__builtin_inff();
}
template <bool F16> __device__ __forceinline__ void pack2maps(const f32x16 (&s)[2], bf16x8 (&p)[2][2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int sp = 0; sp < 2; ++sp) p[i][sp] = pack8<F16>(s[i], sp);
}
// The sums of a step's numerators (short ones, which l takes up: it runs over thousands of keys): of the rounded ones, that o is divided by, and with
// SUMS = 2 of those in s.
template <bool F16, int SUMS> __device__ __forceinline__ void add_weights(const bf16x8 (&p)[2][2], const f32x16 (&s)[2], float (&part)[2], float (&whole)[2]) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int i = 0; i < 2; ++i) part[i] = add2<F16>(__builtin_bit_cast(u32x4, p[i][e >> 2])[e & 3], part[i]);
    if (SUMS == 2)
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int i = 0; i < 2; ++i) whole[i] += s[i][r];
}
template <int SUMS> __device__ __forceinline__ void take_up(float (&l)[2][SUMS], const float (&part)[2], const float (&whole)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i][0] += part[i];
        if (SUMS == 2) l[i][SUMS - 1] += whole[i];
    }
}
// the products with V, and the sums while the first fragments are on their way
template <int D, bool F16, int ROWS, int NB, int SUMS>
__device__ __forceinline__ void values(const Lane& f, const bf16x8 (&p)[2][2], const f32x16 (&s)[2], f32x16 (&o1)[NB], f32x16 (&o2)[NB], float (&l)[2][SUMS]) {
    constexpr int N = 2 * NB, AHEAD = 4;
    bf16x8 x[AHEAD];
    float part[2] = {0.f, 0.f}, whole[2] = {0.f, 0.f};
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) x[n] = f.template cols32<ROWS>(16 * (n / NB), 2 * D + n % NB * 32);
    __builtin_amdgcn_sched_barrier(0);
    add_weights<F16, SUMS>(p, s, part, whole);
    if (SUMS == 1) take_up(l, part, whole);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int sp = n / NB, db = n % NB, q = n + AHEAD;
        o1[db] = mfma32<F16>(x[n % AHEAD], p[0][sp], o1[db]);
        o2[db] = mfma32<F16>(x[n % AHEAD], p[1][sp], o2[db]);
        if (q < N) x[n % AHEAD] = f.template cols32<ROWS>(16 * (q / NB), 2 * D + q % NB * 32);
        __builtin_amdgcn_sched_barrier(0);
    }
    if (SUMS == 2) take_up(l, part, whole);                     // (here it costs fewer registers)
}

// ---- the phases of a sweep -----------------------------------------------------------------------------------------------------------------------
// The forward, dq and dk,dv sweeps share one scheme: a wave keeps 32 rows of its own and a tile of 32 rows streams past a step.  A step is a vector phase (the
// softmax weights of the step) and a matrix phase (the products that the weights go into, then the next step's scores), a barrier behind each.
// At d = 32 and 64 a block has 8 waves; w and w + 4 share a SIMD, and the later four run half a step behind: while one works on the vector units, the
// other has the matrix pipe (left to themselves both do the same thing at the same time).  The vector phase is the longer one: sums of what it made, that
// nobody waits for, are taken in the matrix phase (forward at d = 64: 4 % faster with one sum a map, 12 % with two).  At d = 128 a SIMD's registers hold one
// wave only; nothing alternates there, the barrier behind the matrix phase goes (2 to 4 %: with a fourth buffer, the one that is sent to was left before the
// barrier of the step before), and the forward pass has a kernel of its own.
// Tile t is first read in the matrix phase of step t - 1 and left in step t's, half a step later by the later waves: it is sent for in step t - LEAD
// into the buffer of tile t - BUFS.
template <int D> struct Sweep {
    static constexpr bool PAIRED = D < 128;
    static constexpr int NW = PAIRED ? 8 : 4, ROWS = 32, TILE = ROWS * D * 8, BUFS = PAIRED ? 5 : 4, LEAD = PAIRED ? 3 : 2, OWN = NW * 32;
    static __device__ __forceinline__ void fall_behind(int wave) { if (PAIRED && wave >= NW / 2) __syncthreads(); }
    static __device__ __forceinline__ void wait_for_late(int wave) { if (PAIRED && wave < NW / 2) __syncthreads(); }
    static __device__ __forceinline__ int next(int buf) { return buf == BUFS - 1 ? 0 : buf + 1; }
    // The waits for a wave's own transfers.  Paired: at the start of a vector phase, all of them (tile j + LEAD - 1, sent for a step ago, and the next one is
    // sent for behind the wait).  Alone, at its end, all but the youngest tile's PER instructions, or all where the list has ended; the choice is made
    // inside the instruction text, since a branch of the program here costs copies of the accumulators.
    template <class DMA> static __device__ __forceinline__ void before_vector() { if (PAIRED) DMA::landed(); }
    template <class DMA> static __device__ __forceinline__ void behind_vector(bool more) {
        if (!PAIRED)
            asm volatile("s_cmp_eq_u32 %0, 0\n\ts_cbranch_scc1 .Lland_all%=\n\ts_waitcnt vmcnt(%1)\n\ts_branch .Lland_done%=\n"
                         ".Lland_all%=:\n\ts_waitcnt vmcnt(0)\n.Lland_done%=:"
                         :: "s"(__builtin_amdgcn_readfirstlane((int)more)), "i"(DMA::PER) : "memory", "scc");
    }
};

// ---- forward ----------------------------------------------------------------------------------------------------------------------------------
// 12 d operations a visible pair and head, both maps' products with V apart.  Bound: the matrix and vector instructions together (53 and 42 % of a SIMD's
// cycles, at a clock that the power cap holds at 2.2 GHz).  16 heads of 64 on 4, 8192 causal tokens: 364 us, 1.14 PFLOP/s.  2 x 4097 tokens of 6 heads: 168 us,
// 183 with the maps kept: 204 blocks on 256 CUs, and 12 of these hold one row each, at the time of a full one.
// CUT: a block takes one of a.cuts parts of its keys, and diff_fwd_join_kernel puts them together.
template <int D, bool F16, bool KEEP, bool CUT>
__global__ __launch_bounds__(Sweep<D>::NW * 64, Sweep<D>::PAIRED ? 2 : 1) void diff_fwd_kernel(Args a) {
    typedef Sweep<D> S;
    static_assert(S::PAIRED, "d = 128: diff_fwd_wide_kernel");
    constexpr int ROWS = S::ROWS, TILE = S::TILE, NW = S::NW, NB = D / 16;
    extern __shared__ __attribute__((aligned(16))) char smem[];           // BUFS tiles
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, c = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nblk = (a.Nq + NW * 32 - 1) / (NW * 32);
    int id = block_order();
    const int blk = nblk - 1 - id % nblk;                                 // under a causal mask the last queries have most to do: first
    id /= nblk;
    const int head = id % a.H;
    id /= a.H;
    const int b = CUT ? id % a.B : id, part = CUT ? id / a.B : 0, kvh = head / a.G;
    const int len = key_count(a, b), start = first_pos(a, b);
    const int q0 = blk * (NW * 32) + wave * 32, query = q0 + c;
    const int kend = visible(a, len, start, min(blk * (NW * 32) + NW * 32, a.Nq) - 1);
    const int all = (kend + ROWS - 1) / ROWS, j0 = CUT ? all * part / a.cuts : 0, nj = CUT ? all * (part + 1) / a.cuts - j0 : all;     // tiles of 32 keys
    const int lim = visible(a, len, start, query) - j0 * ROWS, lim_lo = visible(a, len, start, q0) - j0 * ROWS;

    Lane fl;
    fl.init(smem, lane);
    const unsigned lds0 = lds_addr(smem);
    Dma<D, 2 * D, ROWS, NW> dma;
    const bf16_t *kp = a.k + b * a.k_b + 2 * kvh * a.k_h, *vp = a.v + b * a.v_b + kvh * a.v_h;
    dma.init(wave, lane, kp, a.k_n, a.k_h, vp, a.v_n, j0 * ROWS, len);
    for (int t = 0; t < min(S::LEAD, nj); ++t) { dma.issue(lds0 + t * TILE); dma.skip(ROWS); }
    bf16x8 qf[2][D / 16];
    {
        const bf16_t* qp = a.q + b * a.q_b + (long)min(query, a.Nq - 1) * a.q_n + 2 * head * a.q_h + 8 * h;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) qf[i][ks] = load8(qp + i * a.q_h + ks * 16);
    }
    constexpr int SUMS = KEEP ? 2 : 1;
    float m[2], l[2][SUMS];
    f32x16 o1[NB], o2[NB], s[2];
    // The reference that scores are taken against is the largest of the first 32 keys' (a query that sees any key sees the first), and stays: a maximum
    // a step would be a fifth of the vector instructions that bound this loop.  Where a sum shows that later scores passed it so far that P leaves the
    // range (fp16: 2^15, P itself; bf16: 2^40, which leaves 2^87 for the values), the block starts again and keeps a running maximum.
    for (bool running = false;; running = true) {
        if (running) {
            dma.start(kp, vp, j0 * ROWS, len);
            for (int t = 0; t < min(S::LEAD, nj); ++t) { dma.issue(lds0 + t * TILE); dma.skip(ROWS); }
        }
        m[0] = m[1] = NONE;
        l[0][0] = l[1][0] = l[0][SUMS - 1] = l[1][SUMS - 1] = 0.f;
        clear(o1); clear(o2);
        arrived();
        dma.landed();
        __syncthreads();
        scores<D, F16, ROWS>(fl, qf, s);                                  // (without a tile, or behind the last: of what lies there, not used)
        S::fall_behind(wave);
        int buf = 0, ahead = S::LEAD;                                     // the step's buffer, and the one to send to
        for (int j = 0; j < nj; ++j) {
            S::template before_vector<decltype(dma)>();
            if (j + S::LEAD < nj) dma.issue(lds0 + ahead * TILE);
            dma.skip(ROWS);
            ahead = S::next(ahead);
            if (j * 32 + 32 > lim_lo) mask_keys(s, lim - j * 32, h);
            if (j == 0 || running) {
                follow_max(s[0], a.c2, m[0], l[0], o1);
                follow_max(s[1], a.c2, m[1], l[1], o2);
            }
            bf16x8 p[2][2];
            softmax_weights<F16>(s[0], a.c2, m[0], p[0]);
            softmax_weights<F16>(s[1], a.c2, m[1], p[1]);
            S::template behind_vector<decltype(dma)>(j + S::LEAD < nj);
            __syncthreads();
            __builtin_amdgcn_s_setprio(1);
            values<D, F16, ROWS>(fl.at(buf * TILE), p, s, o1, o2, l);
            buf = S::next(buf);
            scores<D, F16, ROWS>(fl.at(buf * TILE), qf, s);
            __builtin_amdgcn_s_setprio(0);
            __syncthreads();
        }
        S::wait_for_late(wave);
        constexpr float MOST = F16 ? 32768.f : 1.0995116e12f;
        if (running || !__syncthreads_or(!(l[0][0] < MOST && l[1][0] < MOST))) break;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < SUMS; ++k) l[i][k] += __shfl_xor(l[i][k], 32, 64);
    if (CUT) {                                                            // [part][32 rows][map, 32 columns][a lane's 4 at a time]; (reference, sums) a row and map
        const long tile = (((long)part * a.B + b) * a.H + head) * nblk * NW + blk * NW + wave;
        f32x4* to = a.sums + tile * (2 * NB * 256) + lane;
#pragma unroll
        for (int n = 0; n < 2 * NB; ++n) {
            const f32x16& x = n < NB ? o1[n % NB] : o2[n % NB];
#pragma unroll
            for (int i = 0; i < 4; ++i) to[n * 256 + i * 64] = f32x4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
        }
        a.stats[tile * 64 + lane] = f32x4{h ? m[1] : m[0], h ? l[1][0] : l[0][0], h ? l[1][SUMS - 1] : l[0][SUMS - 1], 0.f};
        return;
    }
    if (query >= a.Nq) return;
    const float lam = a.lam[head * a.lam_stride];
    float inv[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        inv[i] = l[i][0] > 0.f ? 1.0f / l[i][0] : l[i][0] == 0.f ? 0.f : l[i][0];      // (a NaN stays one)
    }
    const long row = ((long)b * a.Nq + query) * a.H + head, at = row * 2 * D;
    if (KEEP) {
        store_rows<F16>(a.maps + at, o1, inv[0], h);
        store_rows<F16>(a.maps + (long)a.B * a.Nq * a.H * 2 * D + at, o2, inv[1], h);
        float* ls = a.lse + ((long)b * a.H + head) * 4 * a.Nq + query;
        if (h == 0) {
            put_lse(ls, 2 * a.Nq, m[0], l[0][SUMS - 1]);
            put_lse(ls + a.Nq, 2 * a.Nq, m[1], l[1][SUMS - 1]);
        }
    }
    const float w2 = lam * inv[1];
#pragma unroll
    for (int db = 0; db < NB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o1[db][r] = __builtin_fmaf(-w2, o2[db][r], o1[db][r] * inv[0]);
    store_rows<F16>(a.o + at, o1, 1.0f, h);
}

// the parts of a forward pass put together: a wave 32 rows by 32 columns of both maps
template <int D, bool F16, bool KEEP>
__global__ __launch_bounds__(256) void diff_fwd_join_kernel(Args a) {
    constexpr int NB = D / 16, NW = Sweep<D>::NW;
    const int lane = threadIdx.x & 63, h = lane >> 5, c = lane & 31, nq = (a.Nq + Sweep<D>::OWN - 1) / Sweep<D>::OWN * NW;
    const long piece = (long)blockIdx.x * 4 + (threadIdx.x >> 6), tile = piece / NB, tiles = (long)a.B * a.H * nq;
    if (tile >= tiles) return;
    const int db = piece % NB, query = (int)(tile % nq) * 32 + c, head = tile / nq % a.H;
    const long b = tile / nq / a.H;
    if (query >= a.Nq) return;
    float M[2] = {NONE, NONE}, l[2] = {0.f, 0.f}, whole[2] = {0.f, 0.f};
    for (int p = 0; p < a.cuts; ++p)
#pragma unroll
        for (int i = 0; i < 2; ++i) M[i] = fmaxf(M[i], a.stats[(p * tiles + tile) * 64 + i * 32 + c][0]);
    f32x16 x[2][1] = {{zero16()}, {zero16()}};
    for (int p = 0; p < a.cuts; ++p)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f32x4 st = a.stats[(p * tiles + tile) * 64 + i * 32 + c];
            const float w = __builtin_amdgcn_exp2f(st[0] - M[i]);
            l[i] += w * st[1];
            whole[i] += w * st[2];
            const f32x4* from = a.sums + ((p * tiles + tile) * 2 + i) * (NB * 256) + db * 256 + lane;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 t = from[g * 64];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[i][0][4 * g + e] += w * t[e];
            }
        }
    const long at = ((b * a.Nq + query) * a.H + head) * 2 * D + db * 32;
    float inv[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        inv[i] = l[i] > 0.f ? 1.0f / l[i] : l[i] == 0.f ? 0.f : l[i];      // (a NaN stays one)
        if (KEEP) store_rows<F16>(a.maps + i * (long)a.B * a.Nq * a.H * 2 * D + at, x[i], inv[i], h);
        if (KEEP && db == 0 && h == i) put_lse(a.lse + ((b * a.H + head) * 4 + i) * a.Nq + query, 2 * a.Nq, M[i], whole[i]);
    }
    const float w2 = a.lam[head * a.lam_stride] * inv[1];
#pragma unroll
    for (int r = 0; r < 16; ++r) x[0][0][r] = __builtin_fmaf(-w2, x[1][0][r], x[0][0][r] * inv[0]);
    store_rows<F16>(a.o + at, x[0], 1.0f, h);
}

// one map's scores at d = 128
template <bool F16, int ROWS> __device__ __forceinline__ void one_score(const Lane& f, const bf16x8 (&qf)[8], f32x16& s) {
    constexpr int AHEAD = 4;
    bf16x8 x[AHEAD];
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) x[n] = f.template rows16<ROWS>(n * 16);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < 8; ++n) {
        s = mfma32<F16>(x[n % AHEAD], qf[n], n ? s : zero16());
        if (n + AHEAD < 8) x[n % AHEAD] = f.template rows16<ROWS>((n + AHEAD) * 16);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// Forward pass at d = 128: one map after the other.  Both maps' numerators are half of a lane's registers; map 1's outputs wait there, finished, while map 2's
// are made.  A SIMD holds one wave, so nothing alternates, and a step needs one barrier: the tile sent for in step j goes where tile j - 2 was, which all
// waves have left by the barrier of step j - 1.  2 x 4096 tokens of 4 heads: 241 us, 252 with the maps kept,
// 0.86 PFLOP/s (both maps at once in two blocks of half the values, each with all scores: 390 and 412).
struct Wide { static constexpr int D = 128, W = 256, ROWS = 32, NW = Sweep<128>::NW, OWN = Sweep<128>::OWN, BUFS = 4, LEAD = 2, TILE = ROWS * (D + W) * 2; };
template <bool F16, bool KEEP>
__global__ __launch_bounds__(Wide::NW * 64, 1) void diff_fwd_wide_kernel(Args a) {
    typedef Wide S;
    constexpr int ROWS = S::ROWS, TILE = S::TILE, NB = S::W / 32, SUMS = KEEP ? 2 : 1;
    extern __shared__ __attribute__((aligned(16))) char smem[];           // BUFS tiles: a map's keys, two images, and the values, four
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, c = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nblk = (a.Nq + S::OWN - 1) / S::OWN;
    int id = block_order();
    const int blk = nblk - 1 - id % nblk;
    id /= nblk;
    const int head = id % a.H, b = id / a.H, kvh = head / a.G;
    const int len = key_count(a, b), start = first_pos(a, b);
    const int q0 = blk * S::OWN + wave * 32, query = q0 + c;
    const int kend = visible(a, len, start, min(blk * S::OWN + S::OWN, a.Nq) - 1);
    const int lim = visible(a, len, start, query), lim_lo = visible(a, len, start, q0);
    const int nj = (kend + ROWS - 1) / ROWS;
    Lane fl;
    fl.init(smem, lane);
    const unsigned lds0 = lds_addr(smem);
    typedef Dma<64, S::W, ROWS, S::NW> Tiles;                             // (128 columns of one map: two images of 64, 64 columns apart)
    Tiles dma;
    const bf16_t *kp = a.k + b * a.k_b + 2 * kvh * a.k_h, *vp = a.v + b * a.v_b + kvh * a.v_h;
    dma.init(wave, lane, kp, a.k_n, 64, vp, a.v_n, 0, len);
    const float lam = a.lam[head * a.lam_stride];
    const long row = ((long)b * a.Nq + query) * a.H + head, at = row * S::W;
    f32x16 done[NB];
#pragma unroll
    for (int map = 0; map < 2; ++map) {
        bf16x8 qf[S::D / 16];
        const bf16_t* qp = a.q + b * a.q_b + (long)min(query, a.Nq - 1) * a.q_n + (2 * head + map) * a.q_h + 8 * h;
#pragma unroll
        for (int ks = 0; ks < S::D / 16; ++ks) qf[ks] = load8(qp + ks * 16);
        float m, l[SUMS];
        f32x16 o[NB], s;
        // With a fixed reference of a row's scores or a running one (see diff_fwd_kernel).  Two loops: numerators that a step may have to rescale do not
        // stay in the accumulation registers, which costs 128 copies a step.
        auto sweep = [&](auto kind) {
            constexpr bool RUNNING = decltype(kind)::value;
            dma.start(kp + map * a.k_h, vp, 0, len);
            for (int t = 0; t < min(S::LEAD, nj); ++t) { dma.issue(lds0 + t * TILE); dma.skip(ROWS); }
            m = NONE;
            l[0] = l[SUMS - 1] = 0.f;
            clear(o);
            arrived();
            dma.landed();
            __syncthreads();
            one_score<F16, ROWS>(fl, qf, s);                              // (without a tile, or behind the last: of what lies there, not used)
            int buf = 0, ahead = S::LEAD;
            for (int j = 0; j < nj; ++j) {
                if (j + S::LEAD < nj) dma.issue(lds0 + ahead * TILE);
                dma.skip(ROWS);
                ahead = (ahead + 1) & (S::BUFS - 1);
                if (j * 32 + 32 > lim_lo)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = acc_row(r, h) < lim - j * 32 ? s[r] : -__builtin_inff();
                if (RUNNING) follow_max(s, a.c2, m, l, o);
                else if (j == 0) m = first_max(s, a.c2);
                bf16x8 p[2];
                softmax_weights<F16>(s, a.c2, m, p);
                float part[2] = {0.f, 0.f}, whole[2] = {0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 8; ++e) part[e & 1] = add2<F16>(__builtin_bit_cast(u32x4, p[e >> 2])[e & 3], part[e & 1]);
                l[0] += part[0] + part[1];
                if (KEEP) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) whole[r & 1] += s[r];
                    l[SUMS - 1] += whole[0] + whole[1];
                }
                Sweep<128>::behind_vector<Tiles>(j + S::LEAD < nj);
                __syncthreads();
                const Lane f = fl.at(buf * TILE);
                buf = (buf + 1) & (S::BUFS - 1);
                constexpr int N = 2 * NB, AHEAD = 4;
                bf16x8 x[AHEAD];
#pragma unroll
                for (int n = 0; n < AHEAD; ++n) x[n] = f.template cols32<ROWS>(16 * (n / NB), S::D + n % NB * 32);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    o[n % NB] = mfma32<F16>(x[n % AHEAD], p[n / NB], o[n % NB]);
                    if (n + AHEAD < N) x[n % AHEAD] = f.template cols32<ROWS>(16 * ((n + AHEAD) / NB), S::D + (n + AHEAD) % NB * 32);
                    __builtin_amdgcn_sched_barrier(0);
                }
                one_score<F16, ROWS>(fl.at(buf * TILE), qf, s);
            }
            return __syncthreads_or(!(l[0] < (F16 ? 32768.f : 1.0995116e12f)));
        };
        if (sweep(std::false_type())) sweep(std::true_type());
#pragma unroll
        for (int k = 0; k < SUMS; ++k) l[k] += __shfl_xor(l[k], 32, 64);
        const float inv = l[0] > 0.f ? 1.0f / l[0] : l[0] == 0.f ? 0.f : l[0];      // (a NaN stays one)
        if (KEEP && query < a.Nq) {
            store_rows<F16>(a.maps + map * (long)a.B * a.Nq * a.H * S::W + at, o, inv, h);
            if (h == 0) put_lse(a.lse + (((long)b * a.H + head) * 4 + map) * a.Nq + query, 2 * a.Nq, m, l[SUMS - 1]);
        }
        const float w2 = lam * inv;
#pragma unroll
        for (int db = 0; db < NB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) done[db][r] = map ? __builtin_fmaf(-w2, o[db][r], done[db][r]) : o[db][r] * inv;
    }
    if (query < a.Nq) store_rows<F16>(a.o + at, done, 1.0f, h);
}

// ---- split forward: few queries against many keys ------------------------------------------------------------------------------------------
// HBM-bound: K and V are read once for all query heads of a key head.  The 32 columns of a wave's matrix products are 16 rows, (head of the group, query)
// pairs, under both maps: column c is map c / 16 of row c % 16.  q K^T is made of both maps for all columns, and each column keeps its own; the softmax and
// the products with V then go over both maps at once.  A block takes one chunk of the keys, each of its waves every NW-th tile of 32 keys through LDS of
// its own (no barrier in the loop): the next tile's keys are sent for when the scores have been read, its values behind the products with V, so that
// half a tile a wave is always on its way.  Bandwidth leaves the matrix pipe room enough to take P in two numbers of 16 bits, value and what its rounding
// left, so that o is rounded once, at its end.  The waves' numerators are joined in LDS, and the chunks' by diff_join_kernel; with one chunk the result is
// written at once.  Measured: one query of 16 entries on 16384 keys (16 heads on 4 of 64) 108 us with the join, 5.0 TB/s; entries of 0 to 16384 keys 70 us,
// the kernel itself 53, the time of its bytes; 1 entry on 30000 keys 15; 64 entries on 1000 keys 29 us, 4.5 TB/s.
template <int D> struct SplitOf { static constexpr int NW = 4, TILE = 32 * 4 * D * 2; };

template <int D, bool F16, bool KEEP>
__global__ __launch_bounds__(SplitOf<D>::NW * 64, D == 128 ? 1 : 2) void diff_split_kernel(Args a) {
    constexpr int ROWS = 32, NW = SplitOf<D>::NW, TILE = SplitOf<D>::TILE, W = 2 * D, NB = W / 32, NT = NW * 64, PER = 4 * W / NT;
    extern __shared__ __attribute__((aligned(16))) char smem[];           // a tile a wave; then the waves' numerators
    __shared__ float wm[NW][32], wl[NW][32], total[32];
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, c = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int id = blockIdx.x;
    const int split = id % a.nsplit; id /= a.nsplit;
    const int tile = id % a.tiles; id /= a.tiles;
    const int kvh = id % a.Hkv, b = id / a.Hkv;
    const int len = key_count(a, b), start = first_pos(a, b), rows = a.G * a.Nq, here = min(16, rows - tile * 16), RT = min(16, rows);
    const int k0 = split * a.chunk;
    if (k0 >= len && a.nsplit > 1) return;                                // (the join reads the chunks that begin inside len alone)
    const int R = min(tile * 16 + (c & 15), rows - 1), head = kvh * a.G + R / a.Nq, query = R % a.Nq;
    bf16x8 qf[2][D / 16];
    {
        const bf16_t* qp = a.q + b * a.q_b + query * a.q_n + 2 * head * a.q_h + 8 * h;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) qf[i][ks] = load8(qp + i * a.q_h + ks * 16);
    }
    const int lim = visible(a, len, start, query);
    int k1 = min(lim, k0 + a.chunk), lim_lo = lim;                        // end of the chunk's keys that some row sees; keys that every row sees
#pragma unroll
    for (int i = 8; i > 0; i >>= 1) {
        k1 = max(k1, __shfl_xor(k1, i, 64));
        lim_lo = min(lim_lo, __shfl_xor(lim_lo, i, 64));
    }
    k1 = __builtin_amdgcn_readfirstlane(k1);
    lim_lo = __builtin_amdgcn_readfirstlane(lim_lo);

    typedef Dma<D, W, ROWS, 1> Tiles;
    constexpr int KEYS = Tiles::PAIRS * Tiles::GROUPS, ALL = Tiles::PER;  // a tile's pieces: keys, then values
    char* const own = smem + wave * TILE;
    const unsigned at = lds_addr(own);
    Lane f;
    f.init(own, lane);
    Tiles dma;
    dma.init(0, lane, a.k + b * a.k_b + 2 * kvh * a.k_h, a.k_n, a.k_h, a.v + b * a.v_b + kvh * a.v_h, a.v_n, k0 + wave * ROWS, k1);
    dma.issue(at);
    float m = NONE, l[1] = {0.f};
    f32x16 o[NB];
    clear(o);
    arrived();
    for (int t = k0 + wave * ROWS; t < k1; t += NW * ROWS) {
        f32x16 s[2];
        Tiles::template landed<ALL - KEYS>();
        scores<D, F16, ROWS>(f, qf, s);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                // (the reads of the keys are over)
        dma.skip(NW * ROWS);
        dma.template send<0, KEYS>(at);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[0][r] = c < 16 ? s[0][r] : s[1][r];
        if (t + ROWS > lim_lo)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[0][r] = acc_row(r, h) < lim - t ? s[0][r] : -__builtin_inff();
        bf16x8 p[2], rest[2];
        follow_max(s[0], a.c2, m, l, o);
        two_part_weights<F16>(s[0], a.c2, m, l[0], p, rest);
        Tiles::template landed<KEYS>();
        constexpr int N = 2 * NB, AHEAD = 4;
        bf16x8 x[AHEAD];
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) x[n] = f.template cols32<ROWS>(16 * (n / NB), W + n % NB * 32);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            o[n % NB] = mfma32<F16>(x[n % AHEAD], p[n / NB], o[n % NB]);
            o[n % NB] = mfma32<F16>(x[n % AHEAD], rest[n / NB], o[n % NB]);
            if (n + AHEAD < N) x[n % AHEAD] = f.template cols32<ROWS>(16 * ((n + AHEAD) / NB), W + (n + AHEAD) % NB * 32);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                // (and of the values)
        dma.template send<KEYS, ALL>(at);
    }
    Tiles::landed();                                                      // (the numerators go where the tiles were)
    if (h == 0) wm[wave][c] = m;
    l[0] += __shfl_xor(l[0], 32, 64);
    if (h == 0) wl[wave][c] = l[0];
    __syncthreads();
    const long slot = ((long)(b * a.Hkv + kvh) * a.tiles + tile) * a.nsplit + split;
    f32x4* num = (f32x4*)smem;                                            // [wave][32][W / 4], vectors exchanged within 8 by the row's number
    float M = NONE;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, wm[w][c]);
    const float mine = __builtin_amdgcn_exp2f(m - M);
    if ((c & 15) < here) {
#pragma unroll
        for (int db = 0; db < NB; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                num[(wave * 32 + c) * (W / 4) + ((db * 8 + 2 * g + h) ^ (c & 7))] =
                    f32x4{o[db][4 * g] * mine, o[db][4 * g + 1] * mine, o[db][4 * g + 2] * mine, o[db][4 * g + 3] * mine};
        if (tid < 32) {
            float L = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) L += wl[w][c] * __builtin_amdgcn_exp2f(wm[w][c] - M);
            total[c] = L;
            if (a.nsplit > 1) ((f32x2*)a.part)[(slot * 2 + (c >> 4)) * RT + (c & 15)] = f32x2{M, L};
            else if (KEEP) put_lse(a.lse + (((long)b * a.H + head) * 4 + (c >> 4)) * a.Nq + query, 2 * a.Nq, M, L);
        }
    }
    __syncthreads();
    f32x4* part = (f32x4*)a.part + (long)a.B * a.Hkv * a.tiles * a.nsplit * RT;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int r = (e * NT + tid) / (W / 4), at4 = (e * NT + tid) % (W / 4);
        if (r >= here) continue;
        f32x4 x[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[i] = num[(i * 16 + r) * (W / 4) + (at4 ^ (r & 7))];
#pragma unroll
            for (int w = 1; w < NW; ++w) x[i] += num[(w * 32 + i * 16 + r) * (W / 4) + (at4 ^ (r & 7))];
        }
        if (a.nsplit > 1) {
            part[((slot * 2 + 0) * RT + r) * (W / 4) + at4] = x[0];
            part[((slot * 2 + 1) * RT + r) * (W / 4) + at4] = x[1];
            continue;
        }
        const int jh = kvh * a.G + (tile * 16 + r) / a.Nq, jq = (tile * 16 + r) % a.Nq;
        const long row = ((long)b * a.Nq + jq) * a.H + jh;
        const float jl = a.lam[jh * a.lam_stride];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float L = total[i * 16 + r];
            x[i] *= L > 0.f ? 1.0f / L : L == 0.f ? 0.f : L;              // (a NaN stays one)
            if (KEEP) store4<F16>(a.maps + (i * (long)a.B * a.Nq * a.H + row) * W + at4 * 4, x[i][0], x[i][1], x[i][2], x[i][3]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) x[0][k] = __builtin_fmaf(-jl, x[1][k], x[0][k]);
        store4<F16>(a.o + row * W + at4 * 4, x[0][0], x[0][1], x[0][2], x[0][3]);
    }
}

// Joins the chunks of a row (latency: 5 to 6 us), a block each: the chunks' weights first, then their numerators, D threads for the 4 D numbers of one chunk.
template <int D, bool F16>
__global__ __launch_bounds__(256) void diff_join_kernel(Args a) {
    constexpr int W = 2 * D, TOGETHER = 256 / D;
    __shared__ float weight[2][MOST_CHUNKS], top[2][4], sum[2][4];
    __shared__ f32x4 num[256];
    const int tid = threadIdx.x, wave = tid >> 6;
    const int query = blockIdx.x % a.Nq, head = blockIdx.x / a.Nq % a.H, b = blockIdx.x / a.Nq / a.H;
    const int kvh = head / a.G, R = (head % a.G) * a.Nq + query, RT = min(16, a.G * a.Nq);
    const int n = (key_count(a, b) + a.chunk - 1) / a.chunk;              // <= nsplit
    const long slot = ((long)(b * a.Hkv + kvh) * a.tiles + (R >> 4)) * a.nsplit, slots = (long)a.B * a.Hkv * a.tiles * a.nsplit;
    const f32x2* stats = (const f32x2*)a.part + slot * 2 * RT + (R & 15);
    const f32x4* part = (const f32x4*)a.part + slots * RT + (slot * 2 * RT + (R & 15)) * (W / 4);
    float M[2] = {NONE, NONE};
    for (int s = tid; s < n; s += 256)
#pragma unroll
        for (int i = 0; i < 2; ++i) M[i] = fmaxf(M[i], weight[i][s] = stats[(s * 2 + i) * RT][0]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        M[i] = wave_max(M[i]);
        if ((tid & 63) == 0) top[i][wave] = M[i];
    }
    __syncthreads();
    float L[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i) M[i] = fmaxf(fmaxf(top[i][0], top[i][1]), fmaxf(top[i][2], top[i][3]));
    for (int s = tid; s < n; s += 256)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float w = __builtin_amdgcn_exp2f(weight[i][s] - M[i]);
            weight[i][s] = w;
            L[i] += w * stats[(s * 2 + i) * RT][1];
        }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        L[i] = wave_sum(L[i]);
        if ((tid & 63) == 0) sum[i][wave] = L[i];
    }
    __syncthreads();
    const int item = tid % D, map = item / (D / 2), first = tid / D;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    const f32x4* x = part + map * RT * (W / 4) + item % (D / 2);
#pragma unroll 4
    for (int s = first; s < n; s += TOGETHER) acc += weight[map][s] * x[(long)s * 2 * RT * (W / 4)];
    num[tid] = acc;
    __syncthreads();
    if (tid >= W) return;
    const long row = ((long)b * a.Nq + query) * a.H + head;
    float out[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        out[i] = 0.f;
#pragma unroll
        for (int g = 0; g < TOGETHER; ++g) out[i] += ((const float*)num)[g * 4 * D + i * W + tid];
        const float S = (sum[i][0] + sum[i][1]) + (sum[i][2] + sum[i][3]);
        out[i] *= S > 0.f ? 1.0f / S : S == 0.f ? 0.f : S;                // (a NaN stays one)
        if (a.maps) a.maps[(i * (long)a.B * a.Nq * a.H + row) * W + tid] = f2h<F16>(out[i]);
        if (a.maps && tid == 0) put_lse(a.lse + (((long)b * a.H + head) * 4 + i) * a.Nq + query, 2 * a.Nq, M[i], S);
    }
    a.o[row * W + tid] = f2h<F16>(__builtin_fmaf(-a.lam[head * a.lam_stride], out[1], out[0]));
}

// ---- backward ----------------------------------------------------------------------------------------------------------------------------------
// D_m = dO . O_m, 2 d / 8 lanes a row (HBM-bound: three tensors once), and from it the constants of a row that the dk, dv sweep reads, 32 rows together:
// the scores' offsets of both maps (the second with lam's size in it), -D_1 and sign(lam) (D_2 - D_1).  They are counted from the first query that sees a
// key; rows behind the last have P = 0.
template <int D, bool F16>
__global__ __launch_bounds__(256) void diff_rows_kernel(Args a) {
    constexpr int LANES = D / 4;
    const int qt = (a.Nq + 31) / 32;
    const long id = ((long)blockIdx.x * 256 + threadIdx.x) / LANES;       // (b, query of whole tiles, head)
    const int part = threadIdx.x % LANES;
    if (id >= (long)a.B * qt * 32 * a.H) return;                          // (whole groups of LANES leave)
    const long rows = (long)a.B * a.Nq * a.H;
    const int head = id % a.H, place = id / a.H % (qt * 32), b = id / a.H / (qt * 32);
    const int start = first_pos(a, b), query = place + blind(a, start);
    float d[2] = {0.f, 0.f};
    if (query < a.Nq) {
        const u32x4 g = *(const u32x4*)(a.go + b * a.go_b + query * a.go_n + head * a.go_h + part * 8);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const u32x4 o = *(const u32x4*)(a.maps + (i * rows + ((long)b * a.Nq + query) * a.H + head) * 2 * D + part * 8);
#pragma unroll
            for (int e = 0; e < 4; ++e) d[i] += unpack_lo<F16>(g[e]) * unpack_lo<F16>(o[e]) + unpack_hi<F16>(g[e]) * unpack_hi<F16>(o[e]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int s = LANES / 2; s > 0; s >>= 1) d[i] += __shfl_xor(d[i], s, 64);
    if (part) return;
    const long bh = (long)b * a.H + head;
    float e[2] = {__builtin_inff(), __builtin_inff()};
    const float lam = a.lam[head * a.lam_stride];
    if (query < a.Nq) {
        constexpr float UP = F16 ? SHIFT16 : 0;
        const float* ls = a.lse + bh * 4 * a.Nq + query;
        e[0] = ls[0] + (ls[2 * a.Nq] - UP);
        e[1] = ls[a.Nq] + (ls[3 * a.Nq] - UP) - __builtin_amdgcn_logf(fabsf(lam));
        float* p = a.D + bh * 2 * a.Nq + query;
        p[0] = d[0];
        p[a.Nq] = d[1];
    }
    float* r = a.rc + (bh * qt + (place >> 5)) * 128 + (place & 31);
    r[0] = -e[0] / a.c2; r[32] = -e[1] / a.c2; r[64] = -d[0]; r[96] = copysignf(1.0f, lam) * (d[1] - d[0]);
}

// dQ: queries stay, keys stream.  Bound as the forward pass is; 2 x 4097 tokens of 6 heads of 64: 186 us, 155 GFLOP, 0.83 PFLOP/s on 204 of the 256 CUs.
template <int D, bool F16, bool CUT>
__global__ __launch_bounds__(Sweep<D>::NW * 64, Sweep<D>::PAIRED ? 2 : 1) void diff_dq_kernel(Args a) {
    typedef Sweep<D> S;
    constexpr int ROWS = S::ROWS, TILE = S::TILE, NW = S::NW, NQ = D / 32;
    extern __shared__ __attribute__((aligned(16))) char smem[];           // BUFS tiles
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, c = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nblk = (a.Nq + NW * 32 - 1) / (NW * 32);
    int id = block_order();
    const int blk = nblk - 1 - id % nblk;
    id /= nblk;
    const int head = id % a.H;
    id /= a.H;
    const int b = CUT ? id % a.B : id, part = CUT ? id / a.B : 0, kvh = head / a.G;
    const int len = key_count(a, b), start = first_pos(a, b);
    const int q0 = blk * (NW * 32) + wave * 32, query = q0 + c, qrow = min(query, a.Nq - 1);
    const int kend = visible(a, len, start, min(blk * (NW * 32) + NW * 32, a.Nq) - 1);
    const int all = (kend + ROWS - 1) / ROWS, j0 = CUT ? all * part / a.cuts : 0, nj = CUT ? all * (part + 1) / a.cuts - j0 : all;     // tiles of 32 keys
    const int lim = visible(a, len, start, query) - j0 * ROWS, lim_lo = visible(a, len, start, q0) - j0 * ROWS;

    Lane fl;
    fl.init(smem, lane);
    const unsigned lds0 = lds_addr(smem);
    Dma<D, 2 * D, ROWS, NW> dma;
    dma.init(wave, lane, a.k + b * a.k_b + 2 * kvh * a.k_h, a.k_n, a.k_h, a.v + b * a.v_b + kvh * a.v_h, a.v_n, j0 * ROWS, len);
    for (int t = 0; t < min(S::LEAD, nj); ++t) { dma.issue(lds0 + t * TILE); dma.skip(ROWS); }
    bf16x8 qf[2][D / 16], gf[D / 8];
    {
        const bf16_t* qp = a.q + b * a.q_b + qrow * a.q_n + 2 * head * a.q_h + 8 * h;
        const bf16_t* gp = a.go + b * a.go_b + qrow * a.go_n + head * a.go_h + 8 * h;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) qf[i][ks] = load8(qp + i * a.q_h + ks * 16);
#pragma unroll
        for (int ks = 0; ks < D / 8; ++ks) gf[ks] = load8(gp + ks * 16);
    }
    constexpr float UP = F16 ? SHIFT16 : 0;
    const long bh = (long)b * a.H + head;
    const float* ls = a.lse + bh * 4 * a.Nq + qrow;
    const float hi0 = ls[0] - UP, hi1 = ls[a.Nq] - UP;                    // (P comes out times 2^lo)
    const float D0 = a.D[bh * 2 * a.Nq + qrow], D1 = a.D[(bh * 2 + 1) * a.Nq + qrow];
    // bf16: 2^lo is taken off the sums at the end.  fp16: off dP - D, so that dS is packed as 2^4 P (dP - D), as it is for dk
    const float un0 = exp2_neg(ls[2 * a.Nq]), un1 = exp2_neg(ls[3 * a.Nq]), Du0 = D0 * un0, Du1 = D1 * un1;
    float x2 = 0.f;
    f32x16 dq[2][NQ], s[2], dp;
    clear(dq[0]); clear(dq[1]);
    arrived();
    dma.landed();
    __syncthreads();
    scores_dp<D, F16, ROWS>(fl, qf, gf, s, dp);
    S::fall_behind(wave);
    int buf = 0, ahead = S::LEAD;
    for (int j = 0; j < nj; ++j) {
        S::template before_vector<decltype(dma)>();
        if (j + S::LEAD < nj) dma.issue(lds0 + ahead * TILE);
        dma.skip(ROWS);
        ahead = S::next(ahead);
        if (j * 32 + 32 > lim_lo) mask_keys(s, lim - j * 32, h);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][r], a.c2, -hi0));
            const float p2 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[1][r], a.c2, -hi1));
            s[0][r] = p1 * (F16 ? __builtin_fmaf(dp[r], un0, -Du0) : dp[r] - D0);
            s[1][r] = p2 * (F16 ? __builtin_fmaf(dp[r], un1, -Du1) : dp[r] - D1);
        }
        bf16x8 ds[2][2];
        pack2maps<F16>(s, ds);
        S::template behind_vector<decltype(dma)>(j + S::LEAD < nj);
        __syncthreads();
        __builtin_amdgcn_s_setprio(1);
        {
            const Lane f = fl.at(buf * TILE);
            float part[2] = {0.f, 0.f};
            constexpr int N = 4 * NQ, AHEAD = 4;                          // (map, sixteen keys, 32 columns)
            auto frag = [&](int n) { return f.template cols32<ROWS>(16 * (n / NQ % 2), n / (2 * NQ) * D + n % NQ * 32); };
            bf16x8 x[AHEAD];
#pragma unroll
            for (int n = 0; n < AHEAD; ++n) x[n] = frag(n);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                f32x16& acc = dq[n / (2 * NQ)][n % NQ];
                acc = mfma32<F16>(x[n % AHEAD], ds[n / (2 * NQ)][n / NQ % 2], acc);
#pragma unroll
                for (int e = 16 / N * n; e < 16 / N * (n + 1); ++e) part[e & 1] += s[1][e];        // (beside a matrix instruction: see values())
                if (n + AHEAD < N) x[n % AHEAD] = frag(n + AHEAD);
                __builtin_amdgcn_sched_barrier(0);
            }
            x2 += part[0] + part[1];
        }
        buf = S::next(buf);
        scores_dp<D, F16, ROWS>(fl.at(buf * TILE), qf, gf, s, dp);
        __builtin_amdgcn_s_setprio(0);
        if (S::PAIRED) __syncthreads();
    }
    S::wait_for_late(wave);
    x2 += __shfl_xor(x2, 32, 64);
    if (CUT) {                                                            // [part][32 rows][32 columns][a lane's 4 at a time]; [part][row]
        const long tile = (((long)part * a.B + b) * a.H + head) * nblk * NW + blk * NW + wave;
        f32x4* to = a.sums + tile * (2 * NQ * 256) + lane;
#pragma unroll
        for (int n = 0; n < 2 * NQ; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x16& x = dq[n / NQ][n % NQ];
                to[n * 256 + i * 64] = f32x4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
            }
        if (h == 0) ((float*)a.stats)[tile * 32 + c] = x2;
        return;
    }
    if (query >= a.Nq) return;
    const float down0 = F16 ? 1.0f / (1 << SHIFT16) : un0, down1 = F16 ? 1.0f / (1 << SHIFT16) : un1;
    const bool sees = visible(a, len, start, query) > 0;
    if (!sees) { clear(dq[0]); clear(dq[1]); }                            // (whatever its q and dO hold)
    // D_2 = sum P2 dP = D_1' + sum P2 (dP - D_1'), whatever D_1' is that stands for it in the row's dS (sum P2 = 1)
    if (h == 0) a.x2[bh * a.Nq + query] = sees ? x2 * down1 + D1 : 0.f;
    bf16_t* p = a.dq + (((long)b * a.Nq + query) * a.H + head) * 2 * D;
    store_rows<F16>(p, dq[0], a.scale * down0, h);
    store_rows<F16>(p + D, dq[1], -a.lam[head * a.lam_stride] * a.scale * down1, h);
}

// the sum of dq's parts, in their order: a wave 32 rows by 32 columns of [dq1 | dq2]
template <int D, bool F16>
__global__ __launch_bounds__(256) void diff_dq_join_kernel(Args a) {
    constexpr int NQ = D / 32, PER = 2 * NQ, NW = Sweep<D>::NW;
    const int lane = threadIdx.x & 63, h = lane >> 5, c = lane & 31, nq = (a.Nq + Sweep<D>::OWN - 1) / Sweep<D>::OWN * NW;
    const long piece = (long)blockIdx.x * 4 + (threadIdx.x >> 6), tile = piece / PER, tiles = (long)a.B * a.H * nq;
    if (tile >= tiles) return;
    const int n = piece % PER, query = (int)(tile % nq) * 32 + c, head = tile / nq % a.H;
    const long b = tile / nq / a.H, bh = b * a.H + head;
    if (query >= a.Nq) return;
    f32x16 x[1] = {zero16()};
    float x2 = 0.f;
    for (int p = 0; p < a.cuts; ++p) {
        const f32x4* from = a.sums + ((p * tiles + tile) * PER + n) * 256 + lane;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 t = from[i * 64];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[0][4 * i + e] += t[e];
        }
        x2 += ((const float*)a.stats)[(p * tiles + tile) * 32 + c];
    }
    const float* ls = a.lse + bh * 4 * a.Nq + query;
    const float down0 = F16 ? 1.0f / (1 << SHIFT16) : exp2_neg(ls[2 * a.Nq]), down1 = F16 ? 1.0f / (1 << SHIFT16) : exp2_neg(ls[3 * a.Nq]);      // (see there)
    const bool sees = visible(a, key_count(a, b), first_pos(a, b), query) > 0;
    if (!sees) clear(x);
    if (n == 0 && h == 0) a.x2[bh * a.Nq + query] = sees ? x2 * down1 + a.D[(bh * 2 + 1) * a.Nq + query] : 0.f;
    store_rows<F16>(a.dq + ((b * a.Nq + query) * a.H + head) * 2 * D + n * 32, x, n < NQ ? a.scale * down0 : -a.lam[head * a.lam_stride] * a.scale * down1, h);
}

// dK, dV: keys stay, the queries of every head of the group stream.  With the constants of a row (row_constants)
//   P1 = 2^(c2 (s1 - e1)),  P2' = |lam| P2 = 2^(c2 (s2 - e2)),  dP' = dP - D_1 (the accumulators start from -e1, -e2, -D_1),
//   dS1 = P1 dP',  dS2 = sign(lam) P2' (D_2 - D_1 - dP')
template <bool F16>
__device__ __forceinline__ void dkv_weights(const float* rc, int h, float c2, float sign, f32x16 (&s)[2], const f32x16& dp, bf16x8 (&pc)[2], bf16x8 (&ds)[2][2]) {
    f32x16 p;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const f32x4 dd = *(const f32x4*)(rc + 96 + 8 * g + 4 * h);        // rows of registers 4 g .. 4 g + 3
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 4 * g + e;
            const float p1 = __builtin_amdgcn_exp2f(s[0][r] * c2), p2 = __builtin_amdgcn_exp2f(s[1][r] * c2);
            p[r] = __builtin_fmaf(p2, -sign, p1);
            s[0][r] = p1 * dp[r];
            s[1][r] = p2 * __builtin_fmaf(dp[r], -sign, dd[e]);
        }
    }
    pc[0] = pack8<F16>(p, 0); pc[1] = pack8<F16>(p, 1);
    pack2maps<F16>(s, ds);
}
__device__ __forceinline__ f32x16 row_start(const float* rc, int h) {
    f32x16 d;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const f32x4 t = *(const f32x4*)(rc + 8 * g + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) d[4 * g + e] = t[e];
    }
    return d;
}
__device__ __forceinline__ void mask_queries(f32x16 (&s)[2], int vis, int h) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[i][r] = acc_row(r, h) >= vis ? s[i][r] : -__builtin_inff();
}

// At d = 64 the wave's keys lie in LDS and its values in registers: all of both would leave the fragments no room in the 256 registers of two waves
// a SIMD.
// Bound: the matrix phase (32 products, 52 fragment reads of LDS: 1600 cycles) and the vector phase (1600) of a step alike.  2 x 4097 tokens of 6 heads of 64: 260 us,
// 206 GFLOP, 0.79 PFLOP/s on 204 of the 256 CUs.
template <int D, bool F16, bool CUT>
__global__ __launch_bounds__(Sweep<D>::NW * 64, Sweep<D>::PAIRED ? 2 : 1) void diff_dkv_kernel(Args a) {
    typedef Sweep<D> S;
    constexpr int ROWS = S::ROWS, TILE = S::TILE, NW = S::NW, KEYS = S::OWN, NBUF = S::BUFS, NEVER = 0x7fffffff, NQ = D / 32;
    constexpr bool KLDS = D == 64;
    extern __shared__ __attribute__((aligned(16))) char smem[];           // NBUF tiles, NBUF row constants, the block's keys
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, c = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nblk = (a.Nk + KEYS - 1) / KEYS;
    int id = block_order();
    const int blk = id % nblk;                                            // under a causal mask the first keys have most to do: first
    id /= nblk;
    const int kvh = id % a.Hkv;
    id /= a.Hkv;
    const int b = CUT ? id % a.B : id, part = CUT ? id / a.B : 0;
    const int len = key_count(a, b), skip = blind(a, first_pos(a, b)), start = first_pos(a, b) + skip, Nq = a.Nq - skip;
    const int kb = blk * KEYS, k0 = kb + wave * 32, key = k0 + c;
    // Queries are counted from the first that sees a key: the others' rows are not touched.  First query that sees the block's first key; the tiles of a
    // head begin at its tile
    const int t0 = (a.causal ? max(0, kb - start) : 0) / ROWS, qt = (Nq + ROWS - 1) / ROWS;
    // the block's list of tiles, head by head, and its part of it
    const int per = kb < len ? max(0, qt - t0) : 0, all = per * a.G;
    const int j0 = CUT ? (int)((long)all * part / a.parts) : 0, nj = CUT ? (int)((long)all * (part + 1) / a.parts) - j0 : all;
    const int g0 = CUT && per ? j0 / per : 0, first = CUT && per ? t0 + j0 % per : t0;
    // first query row that sees a key (NEVER: the key does not count)
    auto sees = [&](int key) { return key >= len ? NEVER : a.causal ? key - start : -(1 << 30); };
    const int vis = sees(key), vis_all = sees(k0 + 31);

    const unsigned lds0 = lds_addr(smem);
    float* const rc = (float*)(smem + NBUF * TILE);                       // [NBUF][-e1, -e2, -D_1, sign (D_2 - D_1)][32]
    char* const own = smem + NBUF * (TILE + 512) + wave * (32 * D * 4);
    Lane fl, ol;
    fl.init(smem, lane);
    ol.init(own, lane);
    Dma<D, 2 * D, ROWS, NW> dma;
    int sg = g0, st = first, sbuf = 0;                                    // what is sent next
    const char* srow = nullptr;                                           // the tile's row constants
    auto head_start = [&]() {
        const int head = kvh * a.G + sg;
        dma.start(a.q + b * a.q_b + skip * a.q_n + 2 * head * a.q_h, a.go + b * a.go_b + skip * a.go_n + head * a.go_h, st * ROWS, Nq);
        srow = (const char*)(a.rc + (((long)b * a.H + head) * ((a.Nq + ROWS - 1) / ROWS) + st) * 128) + wave * 256;
    };
    dma.init(wave, lane, a.q, a.q_n, a.q_h, a.go, a.go_n, 0, 0);
    if (!CUT || nj > 0) head_start();
    auto send = [&]() {
        dma.issue(lds0 + sbuf * TILE);
        if (wave < 2) {
            const u32x4 r = Dma<D, 2 * D, ROWS, NW>::resource(srow);
            asm volatile(HS_LDS_DMA_WAITS "buffer_load_dword %1, %2, 0 offen lds"
                         :: "s"(__builtin_amdgcn_readfirstlane(lds0 + NBUF * TILE + sbuf * 512 + wave * 256)), "v"(lane * 4), "s"(r) : "memory");
        }
        sbuf = S::next(sbuf);
        dma.skip(ROWS);
        srow += 512;
        if (++st == qt) {
            st = t0;
            if (++sg < a.G) head_start();
        }
    };
    for (int t = 0; t < min(S::LEAD, nj); ++t) send();
    bf16x8 kf[2][D / 16], vf[D / 8];
    {
        // (keys that do not count are not touched: their rows are cleared, so that nothing they hold can come through a product)
        const bf16x8 none = {0, 0, 0, 0, 0, 0, 0, 0};
        const long krow = min(key, a.Nk - 1);
        const bf16_t* kp = a.k + b * a.k_b + krow * a.k_n + 2 * kvh * a.k_h + 8 * h;
        const bf16_t* vp = a.v + b * a.v_b + krow * a.v_n + kvh * a.v_h + 8 * h;
        const bool counts = key < len;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
                bf16x8 x = none;
                if (counts) x = load8(kp + i * a.k_h + ks * 16);
                const int col = i * D + ks * 16;
                if (KLDS) *(bf16x8*)(own + (col >> 6) * (32 * 128) + offR(c, ((col & 63) >> 3) + h)) = x;
                else kf[i][ks] = x;
            }
#pragma unroll
        for (int ks = 0; ks < D / 8; ++ks) { vf[ks] = none; if (counts) vf[ks] = load8(vp + ks * 16); }
    }
    f32x16 dk[2][NQ], dv[2 * NQ], s[2], dp;
    clear(dk[0]); clear(dk[1]); clear(dv);
    auto next_scores = [&](int buf) {
        const Lane f = fl.at(buf * TILE);
        constexpr int N = D / 4, AHEAD = KLDS ? 2 : 4;
        s[0] = row_start(rc + buf * 128, h);
        s[1] = row_start(rc + buf * 128 + 32, h);
        dp = row_start(rc + buf * 128 + 64, h);
        bf16x8 x[AHEAD], y[AHEAD];
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) { x[n] = f.template rows16<ROWS>(n * 16); if (KLDS) y[n] = ol.template rows16<32>(n * 16); }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = n / (D / 16), ks = n % (D / 16);
            if (i < 2) s[i & 1] = mfma32<F16>(x[n % AHEAD], KLDS ? y[n % AHEAD] : kf[i & 1][ks], s[i & 1]);
            else dp = mfma32<F16>(x[n % AHEAD], vf[n - D / 8], dp);
            if (n + AHEAD < N) {
                x[n % AHEAD] = f.template rows16<ROWS>((n + AHEAD) * 16);
                if (KLDS && n + AHEAD < D / 8) y[n % AHEAD] = ol.template rows16<32>((n + AHEAD) * 16);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    arrived();
    dma.landed();
    __syncthreads();
    next_scores(0);                                                       // (without a tile, or behind the last: of what lies there, not used)
    S::fall_behind(wave);
    int buf = 0, g = g0, tq = first;
    float sign = copysignf(1.0f, a.lam[(kvh * a.G + (CUT && nj > 0 ? g0 : 0)) * a.lam_stride]);
    for (int j = 0; j < nj; ++j) {
        S::template before_vector<decltype(dma)>();
        if (j + S::LEAD < nj) send();
        if (tq * ROWS < vis_all) mask_queries(s, vis == NEVER ? NEVER : vis - tq * ROWS, h);
        bf16x8 pc[2], ds[2][2];
        dkv_weights<F16>(rc + buf * 128, h, a.c2, sign, s, dp, pc, ds);
        S::template behind_vector<decltype(dma)>(j + S::LEAD < nj);
        __syncthreads();
        __builtin_amdgcn_s_setprio(1);
        {
            const Lane f = fl.at(buf * TILE);
            constexpr int N = 8 * NQ, AHEAD = 4;                          // (sixteen queries, 32 columns of [q1 | q2 | dO])
            auto frag = [&](int n) { return f.template cols32<ROWS>(16 * (n / (4 * NQ)), n % (4 * NQ) * 32); };
            bf16x8 x[AHEAD];
#pragma unroll
            for (int n = 0; n < AHEAD; ++n) x[n] = frag(n);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int sp = n / (4 * NQ), cb = n % (4 * NQ);
                f32x16& acc = cb < 2 * NQ ? dk[cb / NQ % 2][cb % NQ] : dv[cb < 2 * NQ ? 0 : cb - 2 * NQ];
                acc = mfma32<F16>(x[n % AHEAD], cb < 2 * NQ ? ds[cb / NQ % 2][sp] : pc[sp], acc);
                if (n + AHEAD < N) x[n % AHEAD] = frag(n + AHEAD);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        buf = S::next(buf);
        if (++tq == qt) {
            tq = t0;
            if (++g < a.G) sign = copysignf(1.0f, a.lam[(kvh * a.G + g) * a.lam_stride]);
        }
        next_scores(buf);
        __builtin_amdgcn_s_setprio(0);
        if (S::PAIRED) __syncthreads();
    }
    S::wait_for_late(wave);
    if (CUT) {                                                            // [part][32 keys][32 columns][a lane's 4 at a time], for diff_dkv_join_kernel
        f32x4* to = a.sums + ((((long)part * a.B + b) * a.Hkv + kvh) * nblk * NW + blk * NW + wave) * (4 * NQ * 256) + lane;
#pragma unroll
        for (int n = 0; n < 4 * NQ; ++n) {
            const f32x16& x = n < 2 * NQ ? dk[n / NQ % 2][n % NQ] : dv[n < 2 * NQ ? 0 : n - 2 * NQ];
#pragma unroll
            for (int i = 0; i < 4; ++i) to[n * 256 + i * 64] = f32x4{x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
        }
        return;
    }
    if (key >= a.Nk) return;
    const float down = F16 ? 1.0f / (1 << SHIFT16) : 1.0f;
    const long row = ((long)b * a.Nk + key) * a.Hkv + kvh;
    store_rows<F16>(a.dv + row * 2 * D, dv, down, h);
    store_rows<F16>(a.dk + row * 2 * D, dk[0], a.scale * down, h);
    store_rows<F16>(a.dk + row * 2 * D + D, dk[1], a.scale * down, h);
}

// the sum of the parts of dk and dv, in their order: a wave 32 keys by 32 columns of [dk1 | dk2 | dv]
template <int D, bool F16>
__global__ __launch_bounds__(256) void diff_dkv_join_kernel(Args a) {
    constexpr int NQ = D / 32, PER = 4 * NQ;
    const int lane = threadIdx.x & 63, h = lane >> 5, nk = (a.Nk + Sweep<D>::OWN - 1) / Sweep<D>::OWN * Sweep<D>::NW;
    const long piece = (long)blockIdx.x * 4 + (threadIdx.x >> 6), pieces = (long)a.B * a.Hkv * nk * PER;
    if (piece >= pieces) return;
    const int n = piece % PER, key = (int)(piece / PER % nk) * 32 + (lane & 31), kvh = piece / PER / nk % a.Hkv;
    const long b = piece / PER / nk / a.Hkv;
    if (key >= a.Nk) return;
    const f32x4* from = a.sums + piece * 256 + lane;
    f32x16 x[1] = {zero16()};
    for (int p = 0; p < a.parts; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 t = from[p * pieces * 256 + i * 64];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[0][4 * i + e] += t[e];
        }
    const float down = F16 ? 1.0f / (1 << SHIFT16) : 1.0f;
    const long row = ((b * a.Nk + key) * a.Hkv + kvh) * 2 * D;
    if (n < 2 * NQ) store_rows<F16>(a.dk + row + n * 32, x, a.scale * down, h);
    else store_rows<F16>(a.dv + row + n * 32 - 2 * D, x, down, h);
}

// dlam[h] = - sum over entries and queries of D_2 (all heads for one shared lam): a block each, in a fixed order, summed in 64 bits; a thread has
// eight loads on their way at a time
__global__ __launch_bounds__(1024) void diff_dlam_kernel(Args a, float* dlam) {
    __shared__ double red[1024];
    const int h0 = a.lam_stride ? blockIdx.x : 0;
    const long run = (long)(a.lam_stride ? 1 : a.H) * a.Nq, n = run * a.B;                   // an entry's stretch of D_2; all of them
    double s = 0;
    for (long i0 = threadIdx.x; i0 < n; i0 += 8 * 1024) {
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const long i = i0 + k * 1024, b = i / run;
            x[k] = i < n ? a.x2[(b * a.H + h0) * a.Nq + (i - b * run)] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) s += x[k];
    }
    red[threadIdx.x] = s;
    __syncthreads();
    for (int w = 512; w > 0; w >>= 1) {
        if ((int)threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x == 0) dlam[blockIdx.x] = (float)-red[0];
}

// ---- host --------------------------------------------------------------------------------------------------------------------------------------
int check(const hs_diff_attn_desc* d, bool backward) {
    if (!d || d->struct_size != sizeof(hs_diff_attn_desc)) return HS_ERR_ARG;
    if (d->dtype != HS_PREC_BF16 && d->dtype != HS_PREC_F16) return HS_ERR_ARG;
    if (!(d->scale > 1e-30f) || !(d->scale < 1e6f) || d->lam_stride < 0) return HS_ERR_ARG;      // (diff_rows_kernel divides by it)
    if (d->B < 1 || d->Nq < 1 || d->Nk < 1 || d->H < 1 || d->Hkv < 1 || d->H % d->Hkv) return HS_ERR_SHAPE;
    if (d->d != 32 && d->d != 64 && d->d != 128) return HS_ERR_SHAPE;
    if (d->Nq > (1 << 28) || d->Nk > (1 << 28) || d->H > (1 << 16)) return HS_ERR_SHAPE;
    if ((int64_t)d->B * d->H > ((int64_t)1 << 36) / ((int64_t)d->Nq + d->Nk)) return HS_ERR_SHAPE;
    // every launch stays under 2^32 threads: the sweeps have 512 for 256 rows or 256 for 64 or 128, the rows' constants d / 4 for one (split_of sees to the
    // split forward, 256 for 16)
    if ((int64_t)d->B * d->H * (((int64_t)(d->Nq > d->Nk ? d->Nq : d->Nk) + 127) / 128) >= (1 << 22)) return HS_ERR_SHAPE;
    if (backward && (int64_t)d->B * d->H * (((int64_t)d->Nq + 31) / 32) * 8 * d->d >= (int64_t)1 << 32) return HS_ERR_SHAPE;
    for (int64_t s : {d->q_b, d->q_n, d->q_h, d->k_b, d->k_n, d->k_h, d->v_b, d->v_n, d->v_h})
        if (s < 0 || (s & 7)) return HS_ERR_SHAPE;
    for (int64_t s : {d->q_n, d->q_h, d->k_n, d->k_h, d->v_n, d->v_h, backward ? d->go_n : 0, backward ? d->go_h : 0})
        if (s > (1 << 24)) return HS_ERR_SHAPE;                            // a tile's 32 rows lie inside a buffer descriptor's 2 GiB
    if (backward)
        for (int64_t s : {d->go_b, d->go_n, d->go_h})
            if (s < 0 || (s & 7)) return HS_ERR_SHAPE;
    return HS_OK;
}
bool misaligned(const void* p, unsigned n = 16) { return !p || (uintptr_t)p % n; }

struct Split { int tiles, nsplit, chunk; };
constexpr int SPARSE = 128, WANT = 1024, LEAST = 512;       // blocks (two rounds even out ragged entries: 70 us against 78 with one); keys of a chunk (4 tiles a wave)
// Parts that a sweep is cut into.  A round of blocks (one a CU) takes `tiles` microseconds; cutting costs each block another start, a second kernel, and
// `traffic` of a microsecond for a part's sums of a block written and read.  The forward pass gives the time that it measured (whole_of).  The backward sweeps
// are taken at one microsecond a tile of 32 rows at every width, less than they measure (full rounds: dq 1.4 at d = 64 and 1.8 at 128, dk, dv 2.1 and 2.8), so that
// they are cut later than would pay.  Whole / cut in us: forward, 4096 tokens of 4 heads of 64 136 / 74, causal
// 137 / 64; 2048 causal tokens of 8 heads 72 / 46; 512 queries of 16 heads on 8192 keys 135 / 75; the backward pass with dq cut, the same four but the last:
// 253 / 172, 242 / 159, 145 / 107.
struct Cuts { int parts; double time; };
Cuts cuts_of(int64_t blocks, double tiles, double start, double traffic) {
    Cuts best = {1, 0};
    for (int p = 1; p <= 16; ++p) {
        const double time = (double)((blocks * p + 255) / 256) * (tiles / p + start) + (p > 1 ? 6 + traffic * (double)blocks * p : 0);
        if (p == 1 || time < best.time) best = {p, time};
    }
    return best;
}
int own_of(const hs_diff_attn_desc* d) { return d->d == 128 ? Sweep<128>::OWN : Sweep<64>::OWN; }
int64_t blocks_of(const hs_diff_attn_desc* d) { return (int64_t)d->B * d->H * ((d->Nq + own_of(d) - 1) / own_of(d)); }
// the whole forward pass, in us: at d = 32, 64 and 128 0.8, 1.06 and twice 0.92 a tile (at d = 128 not cut)
Cuts whole_of(const hs_diff_attn_desc* d) {
    const double time = (double)((d->Nk + 31) / 32) * (d->d == 32 ? 0.8 : d->d == 64 ? 1.06 : 1.84);
    if (d->d == 128) return {1, (double)((blocks_of(d) + 255) / 256) * (time + 4)};
    return cuts_of(blocks_of(d), time, 3, 0.09 * d->d / 64);
}
// Whether the split forward runs, and how it cuts the keys.  The whole forward needs the time of one block over all (its part of the) keys for each round of
// blocks on the 256 CUs, full or not; the split forward's time goes with its tiles, wherever they come from.  Measured with 16 query heads on 4 key heads of
// 64, 8192 keys, whole (not cut) / split in us: 1 entry, 16 queries 256 / 18; 16 entries, 16 queries 343 / 116, 32 (512 tiles) 328 / 205, 64 (1024 tiles)
// 317 / 352, 128 334 / 488.  8 on 2 of 128, 16 entries, 512 / 2048 keys: 32 queries (256 tiles) 36, 116 / 27, 74, 64 (512 tiles) 37, 117 / 36, 107.
Split split_of(const hs_diff_attn_desc* d) {
    const int64_t rows = (int64_t)(d->H / d->Hkv) * d->Nq, tiles = (rows + 15) / 16, blocks = (int64_t)d->B * d->Hkv * tiles;
    const double time = (d->d == 128 ? 0.0019 : 0.00135) * (double)blocks * (double)((d->Nk + 31) / 32);      // us beside 8 of start and join
    if (time > 4 && time + 8 > whole_of(d).time) return {0, 0, 0};          // (small calls take launches either way, and the split forward rounds less)
    if (blocks >= 1 << 24) return {0, 0, 0};                                // (a block of 256 threads for each 16 rows: a launch ends at 2^32)
    const int64_t want = std::min<int64_t>((WANT + blocks - 1) / blocks, MOST_CHUNKS);
    // (a grid that leaves most CUs idle anyway takes half as long chunks, unless one would do without the join: 1 entry, 2000 keys 12 -> 11 us)
    const int64_t least = d->Nk > LEAST && blocks * ((d->Nk + LEAST - 1) / LEAST) <= SPARSE ? LEAST / 2 : LEAST;
    const int64_t chunk = std::max<int64_t>(((d->Nk + want - 1) / want + 127) / 128 * 128, least);
    return {(int)tiles, (int)((d->Nk + chunk - 1) / chunk), (int)chunk};
}
// bytes of the parts' sums of a forward pass, and of all that it needs
size_t cut_bytes(const hs_diff_attn_desc* d, int cuts) { return cuts > 1 ? (size_t)cuts * blocks_of(d) * own_of(d) * (size_t)d->d * 16 : 0; }
size_t forward_bytes(const hs_diff_attn_desc* d, const Split& s, int cuts) {
    const size_t rows = std::min<int64_t>(16, (int64_t)(d->H / d->Hkv) * d->Nq);
    if (!s.nsplit) return cuts > 1 ? cut_bytes(d, cuts) + (size_t)cuts * blocks_of(d) * own_of(d) * 32 : 0;
    return s.nsplit > 1 ? (size_t)d->B * d->Hkv * s.tiles * s.nsplit * 2 * rows * (2 * d->d + 2) * 4 : 0;
}
// Parts that the dk, dv sweep's list of tiles is cut into.  Backward pass whole / cut in us: 8192 causal tokens, 16 heads of 64 on 1: 5904 / 1216, on 4:
// 1850 / 1225; 4 x 512 tokens, 12 on 4: 130 / 107; 2 x 4097 tokens, 6 on 6 (204 blocks): not cut.
int parts_of(const hs_diff_attn_desc* d) {
    return cuts_of((int64_t)d->B * d->Hkv * ((d->Nk + own_of(d) - 1) / own_of(d)), (double)(d->H / d->Hkv) * ((d->Nq + 31) / 32), 4, 0.07).parts;
}
size_t rows_bytes(const hs_diff_attn_desc* d) { return (size_t)d->B * d->H * ((size_t)d->Nq * 12 + (size_t)((d->Nq + 31) / 32) * 512); }
// parts of the dq sweep's keys (see cuts_of)
int cuts_of_dq(const hs_diff_attn_desc* d) { return cuts_of(blocks_of(d), (double)((d->Nk + 31) / 32), 4, 0.045 * d->d / 64).parts; }
// Behind the rows' numbers lie dq's parts (sums, then a number a row), and, when these have been put together, those of dk and dv.
size_t sums_at(const hs_diff_attn_desc* d) { return (rows_bytes(d) + 255) / 256 * 256; }
size_t dq_bytes(const hs_diff_attn_desc* d, int cuts) { return cuts > 1 ? (size_t)cuts * blocks_of(d) * own_of(d) * (size_t)d->d * 8 : 0; }
size_t backward_bytes(const hs_diff_attn_desc* d) {
    const size_t own = own_of(d), p = parts_of(d), c = cuts_of_dq(d);
    const size_t kv = p > 1 ? p * d->B * d->Hkv * ((d->Nk + own - 1) / own) * own * d->d * 16 : 0, q = c > 1 ? dq_bytes(d, c) + c * blocks_of(d) * own * 4 : 0;
    return kv || q ? sums_at(d) + std::max(kv, q) : rows_bytes(d);
}
Args args_of(const hs_diff_attn_desc* d) {
    Args a = {};
    a.q_b = d->q_b; a.q_n = d->q_n; a.q_h = d->q_h; a.k_b = d->k_b; a.k_n = d->k_n; a.k_h = d->k_h;
    a.v_b = d->v_b; a.v_n = d->v_n; a.v_h = d->v_h; a.go_b = d->go_b; a.go_n = d->go_n; a.go_h = d->go_h;
    a.B = d->B; a.Nq = d->Nq; a.Nk = d->Nk; a.H = d->H; a.Hkv = d->Hkv; a.G = d->H / d->Hkv;
    a.causal = d->causal; a.q_start0 = d->q_start0; a.lam_stride = d->lam_stride;
    a.scale = d->scale; a.c2 = d->scale * LOG2E;
    return a;
}
template <class K> void launch(K kernel, int64_t grid, int threads, size_t lds, hipStream_t s, const Args& a) {
    if (lds > 60000) (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), lds, s, a);
}
template <int D, bool F16, bool KEEP> void forward(const Args& a, const Split& sp, hipStream_t s) {
    typedef Sweep<D> S;
    if (sp.nsplit) {
        typedef SplitOf<D> P;
        launch(diff_split_kernel<D, F16, KEEP>, (int64_t)a.B * a.Hkv * sp.tiles * sp.nsplit, P::NW * 64, (size_t)P::NW * P::TILE, s, a);
        if (sp.nsplit > 1) launch(diff_join_kernel<D, F16>, (int64_t)a.B * a.H * a.Nq, 256, 0, s, a);
        return;
    }
    const int64_t blocks = (int64_t)a.B * a.H * ((a.Nq + S::OWN - 1) / S::OWN);
    if constexpr (D == 128) launch(diff_fwd_wide_kernel<F16, KEEP>, blocks, Wide::NW * 64, (size_t)Wide::BUFS * Wide::TILE, s, a);
    else if (a.cuts == 1) launch(diff_fwd_kernel<D, F16, KEEP, false>, blocks, S::NW * 64, (size_t)S::BUFS * S::TILE, s, a);
    else {
        launch(diff_fwd_kernel<D, F16, KEEP, true>, blocks * a.cuts, S::NW * 64, (size_t)S::BUFS * S::TILE, s, a);
        launch(diff_fwd_join_kernel<D, F16, KEEP>, blocks * S::NW * (D / 16) / 4, 256, 0, s, a);
    }
}
template <int D, bool F16> void backward(const Args& a, hipStream_t s) {
    typedef Sweep<D> S;
    constexpr int LANES = D / 4;
    launch(diff_rows_kernel<D, F16>, ((int64_t)a.B * ((a.Nq + 31) / 32 * 32) * a.H * LANES + 255) / 256, 256, 0, s, a);
    const int64_t rows = (int64_t)a.B * a.H * ((a.Nq + S::OWN - 1) / S::OWN);
    if (a.cuts == 1) launch(diff_dq_kernel<D, F16, false>, rows, S::NW * 64, (size_t)S::BUFS * S::TILE, s, a);
    else {
        launch(diff_dq_kernel<D, F16, true>, rows * a.cuts, S::NW * 64, (size_t)S::BUFS * S::TILE, s, a);
        launch(diff_dq_join_kernel<D, F16>, rows * S::NW * (D / 16) / 4, 256, 0, s, a);
    }
    const int64_t blocks = (int64_t)a.B * a.Hkv * ((a.Nk + S::OWN - 1) / S::OWN);
    const size_t lds = (size_t)S::BUFS * (S::TILE + 512) + (D == 64 ? S::OWN * D * 4 : 0);
    if (a.parts == 1) return launch(diff_dkv_kernel<D, F16, false>, blocks, S::NW * 64, lds, s, a);
    launch(diff_dkv_kernel<D, F16, true>, blocks * a.parts, S::NW * 64, lds, s, a);
    launch(diff_dkv_join_kernel<D, F16>, blocks * S::NW * (D / 32), 256, 0, s, a);
}
#define HS_BY_TYPE(call)                                                               \
    do {                                                                               \
        const bool f16 = d->dtype == HS_PREC_F16;                                      \
        if (d->d == 32) { if (f16) call(32, true); else call(32, false); }             \
        else if (d->d == 64) { if (f16) call(64, true); else call(64, false); }        \
        else { if (f16) call(128, true); else call(128, false); }                      \
    } while (0)

}  // namespace

extern "C" size_t hs_diff_attn_fwd_ws_bytes(const hs_diff_attn_desc* d) { return check(d, false) == HS_OK ? forward_bytes(d, split_of(d), whole_of(d).parts) : 0; }
extern "C" size_t hs_diff_attn_bwd_ws_bytes(const hs_diff_attn_desc* d) { return check(d, false) == HS_OK ? backward_bytes(d) : 0; }

extern "C" int hs_diff_attn_fwd(const hs_diff_attn_desc* d, const void* q, const void* k, const void* v, const float* lam, const int32_t* q_start,
                                const int32_t* kv_len, void* o, void* maps, float* lse, void* ws, size_t ws_bytes, void* stream) {
    const int rc = check(d, false);
    if (rc != HS_OK) return rc;
    if (!q || !k || !v || !o || !lam || !maps != !lse) return HS_ERR_ARG;
    if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(o) || (maps && misaligned(maps))) return HS_ERR_SHAPE;
    const Split sp = split_of(d);
    const int cuts = whole_of(d).parts;
    const size_t need = forward_bytes(d, sp, cuts);
    if (need && (misaligned(ws) || ws_bytes < need)) return HS_ERR_SHAPE;
    Args a = args_of(d);
    a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.lam = lam; a.q_start = q_start; a.kv_len = kv_len;
    a.o = (bf16_t*)o; a.maps = (bf16_t*)maps; a.lse = lse; a.part = (float*)ws;
    a.tiles = sp.tiles; a.nsplit = sp.nsplit; a.chunk = sp.chunk;
    a.cuts = cuts; a.sums = (f32x4*)ws; a.stats = (f32x4*)((char*)ws + cut_bytes(d, cuts));
    hipStream_t s = (hipStream_t)stream;
#define CALL(D, F) maps ? forward<D, F, true>(a, sp, s) : forward<D, F, false>(a, sp, s)
    HS_BY_TYPE(CALL);
#undef CALL
    HS_CHECK_LAUNCH();
    return HS_OK;
}

extern "C" int hs_diff_attn_bwd(const hs_diff_attn_desc* d, const void* q, const void* k, const void* v, const float* lam, const int32_t* q_start,
                                const int32_t* kv_len, const void* d_o, const void* maps, const float* lse, void* dq, void* dk, void* dv,
                                float* dlam, void* ws, size_t ws_bytes, void* stream) {
    const int rc = check(d, true);
    if (rc != HS_OK) return rc;
    if (!q || !k || !v || !lam || !d_o || !maps || !lse || !dq || !dk || !dv || !dlam || !ws) return HS_ERR_ARG;
    for (const void* p : {q, k, v, d_o, maps, (const void*)dq, (const void*)dk, (const void*)dv, (const void*)ws})
        if (misaligned(p)) return HS_ERR_SHAPE;
    if (ws_bytes < backward_bytes(d)) return HS_ERR_SHAPE;
    Args a = args_of(d);
    a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.go = (const bf16_t*)d_o; a.lam = lam;
    a.q_start = q_start; a.kv_len = kv_len; a.maps = (bf16_t*)maps; a.lse = (float*)lse;
    a.D = (float*)ws; a.x2 = a.D + (size_t)d->B * d->H * 2 * d->Nq;
    a.rc = a.x2 + (size_t)d->B * d->H * d->Nq;
    a.parts = parts_of(d); a.cuts = cuts_of_dq(d);
    a.sums = (f32x4*)((char*)ws + sums_at(d)); a.stats = (f32x4*)((char*)a.sums + dq_bytes(d, a.cuts));
    a.dq = (bf16_t*)dq; a.dk = (bf16_t*)dk; a.dv = (bf16_t*)dv;
    hipStream_t s = (hipStream_t)stream;
#define CALL(D, F) backward<D, F>(a, s)
    HS_BY_TYPE(CALL);
#undef CALL
    HS_CHECK_LAUNCH();
    hipLaunchKernelGGL(diff_dlam_kernel, dim3(a.lam_stride ? a.H : 1), dim3(1024), 0, s, a, dlam);
    HS_CHECK_LAUNCH();
    return HS_OK;
}
