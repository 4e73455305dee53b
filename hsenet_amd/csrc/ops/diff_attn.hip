// Differential attention, o = P1 v - lam P2 v with P_m = softmax(scale q_m k_m^T): forward, split forward for few queries, backward.
//
// As in attn.hip, the index that the second product sums over lies on the accumulator's row (register) axis, so a score tile is, rounded and
// packed, the next matrix instruction's operand as it stands:
//   forward  S_m^T[key][query] = K_m Q_m^T -> P_m^T ;            O_m^T[dv][query] += V^T P_m^T        (both maps read one V fragment)
//   dq       S_m^T, dP^T = V dO^T          -> dS_m^T = P_m^T (dP^T - D_m) ;  dQ_m^T[d][query] += K_m^T dS_m^T
//   dk, dv   S_m[query][key] = Q_m K_m^T, dP = dO V^T ;          dV^T[dv][key] += dO^T (P1 - lam P2) ;  dK_m^T[d][key] += Q_m^T dS_m
// with D_m = sum over keys of P_m dP = dO . O_m (O_m: the map's own output, kept by the forward pass).  dP is one product for both maps, and dV too.
// Tiles of 64 rows are staged in LDS images R (common.h: 128-byte rows, read by rows and by columns): d / 32 images of a head pair's two keys
// (queries) side by side and d / 32 of its values (dO).
#include "../common.h"
#include "../attn_util.h"
#include "../../../include/hsenet_ops.h"

namespace {

constexpr float LOG2E = 1.44269504088896341f;
constexpr float NONE = -1e30f;                 // running maximum before the first visible key
constexpr float HEADROOM = 8.0f;               // a running maximum is kept until a score passes it by this many powers of two
constexpr int SHIFT16 = 4;                     // fp16: P and dS of the backward pass are held times 2^4

struct Args {
    const bf16_t *q, *k, *v, *go;
    const float* lam;
    const int *q_start, *kv_len;
    bf16_t *o, *maps;
    float* lse;                                // [B][H][hi of both maps, lo of both][Nq] (put_lse); hi = +inf: no visible key
    float *D, *x2;                             // backward: D_m [B][H][2][Nq], D_2 in full precision [B][H][Nq]
    bf16_t *dq, *dk, *dv;
    float* part;                               // split forward: numerators, then (maximum, sum)
    long q_b, q_n, q_h, k_b, k_n, k_h, v_b, v_n, v_h, go_b, go_n, go_h;
    int B, Nq, Nk, H, Hkv, G, causal, q_start0, lam_stride, nsplit, chunk, tiles;
    float c2, scale;                           // scale * log2(e), scale
};

// Blocks are dealt round the 8 XCDs; a contiguous range of them to each lets the blocks of a key head share one L2.
__device__ __forceinline__ int block_order() {
    const int nb = gridDim.x, id = blockIdx.x, q = nb >> 3, r = nb & 7, x = id & 7;
    return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (id >> 3);
}
__device__ __forceinline__ int key_count(const Args& a, int b) { return a.kv_len ? min(max(a.kv_len[b], 0), a.Nk) : a.Nk; }
__device__ __forceinline__ int first_pos(const Args& a, int b) {
    const int s = a.q_start ? a.q_start[b] : a.q_start0;
    return min(max(s, -(1 << 30)), 1 << 30);
}
// number of leading keys that query i sees
__device__ __forceinline__ int visible(const Args& a, int len, int start, int i) { return a.causal ? max(0, min(len, start + i + 1)) : len; }

// ---- a tile: ROWS rows of [two heads of d | 2d] columns, through registers into LDS images ------------------------------------------------
// A thread always moves the same 16-byte column chunk, so its source is one pointer and one row stride.
template <int D, int ROWS, int NT> struct Stage {
    static constexpr int CH = D / 2, PER = ROWS * CH / NT, STEP = NT / CH, BASES = STEP < 16 ? 16 / STEP : 1;
    const char* src;
    long stride;
    int row, dst[BASES];                       // (image R's swizzle repeats every 16 rows)
    u32x4 r[PER];
    __device__ __forceinline__ void init(int tid, const bf16_t* x, long x_n, long x_h, const bf16_t* y, long y_n) {
        const int cc = tid % CH, col = cc * 8;
        row = tid / CH;
        const bool pair = cc < CH / 2;
        src = (const char*)(pair ? x + (col / D) * x_h + col % D : y + (col - 2 * D));
        stride = (pair ? x_n : y_n) * 2;
#pragma unroll
        for (int i = 0; i < BASES; ++i) dst[i] = (cc >> 3) * (ROWS * 128) + offR(row + i * STEP, cc & 7);
    }
    __device__ __forceinline__ void load(int first, int end) {       // rows at or behind `end` become zeros, and are not touched
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int n = first + row + i * STEP;
            r[i] = u32x4{0u, 0u, 0u, 0u};
            if (n < end) r[i] = *(const u32x4*)(src + n * stride);
        }
    }
    __device__ __forceinline__ void write(char* lds) const {
#pragma unroll
        for (int i = 0; i < PER; ++i) *(u32x4*)(lds + dst[i % BASES] + i / BASES * BASES * STEP * 128) = r[i];
    }
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

// One map's softmax over 32 keys of a query: s becomes 2^(c2 s - m).  m, the reference, is the largest score so far up to HEADROOM: it moves,
// and l and the numerators with it, only when a score passes it by more, which after the first tiles is rare; any reference gives the same
// quotient.  It is one number for both halves of a query's lanes (they hold different keys of one product).
template <int NB>
__device__ __forceinline__ void softmax_step(f32x16& s, float c2, float& m, float& l, f32x16 (&o)[NB]) {
    float mx = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
    mx *= c2;
    if (__builtin_amdgcn_ballot_w64(mx > m + HEADROOM)) {
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float mn = fmaxf(m, ceilf(mx)), alpha = __builtin_amdgcn_exp2f(m - mn);
        l *= alpha;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][r] *= alpha;
            __builtin_amdgcn_sched_barrier(0);
        }
        m = mn;
    }
    float part[4] = {0.f, 0.f, 0.f, 0.f};                                 // short sums first: l runs over thousands of keys
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c2, -m));
        s[r] = p;
        part[r & 3] += p;
    }
    l += (part[0] + part[1]) + (part[2] + part[3]);
}
// What the backward pass needs of a row's softmax: P = 2^(c2 s - hi - lo), hi whole (the reference m is), 0 <= lo < 1.  One fp32 number of their sum's
// size would put a common error of 5e-7 on all of a row's P, which the sum that is lam's gradient would keep.
__device__ __forceinline__ void put_lse(float* p, long next, float m, float l) {
    const int e = l > 0.f && l < __builtin_inff() ? __builtin_amdgcn_frexp_expf(l) - 1 : 0;
    p[0] = l == 0.f ? __builtin_inff() : m + (float)e;
    p[next] = l == 0.f ? 0.f : __builtin_amdgcn_logf(__builtin_amdgcn_ldexpf(l, -e));
}

// both maps of one wave's 32 queries against the 32 keys whose rows start at r0 of the tile; lim: visible keys of the lane's query, counted from
// the tile's first row; MASK: some of them may not be visible
template <int D, bool F16, int ROWS>
__device__ __forceinline__ void forward_step(const Lane& f, int r0, bool mask, int lim, int h, float c2, const bf16x8 (&qf)[2][D / 16], float (&m)[2],
                                             float (&l)[2], f32x16 (&o1)[D / 16], f32x16 (&o2)[D / 16]) {
    f32x16 s[2] = {zero16(), zero16()};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) s[i] = mfma32<F16>(f.template rows16<ROWS>(i * D + ks * 16), qf[i][ks], s[i]);
    if (mask) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[i][r] = r0 + acc_row(r, h) < lim ? s[i][r] : -__builtin_inff();
    }
    softmax_step(s[0], c2, m[0], l[0], o1);
    softmax_step(s[1], c2, m[1], l[1], o2);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int sp = 0; sp < 2; ++sp) {
        const bf16x8 p1 = pack8<F16>(s[0], sp), p2 = pack8<F16>(s[1], sp);
#pragma unroll
        for (int db = 0; db < D / 16; ++db) {
            const bf16x8 vf = f.template cols32<ROWS>(16 * sp, 2 * D + db * 32);
            o1[db] = mfma32<F16>(vf, p1, o1[db]);
            o2[db] = mfma32<F16>(vf, p2, o2[db]);
        }
    }
}

// ---- forward: a block is NW waves of 32 queries of one head ------------------------------------------------------------------------------
template <int D, bool F16, int NW>
__global__ __launch_bounds__(NW * 64, D == 128 ? 1 : 2) void diff_fwd_kernel(Args a) {
    constexpr int ROWS = D == 128 ? 32 : 64, TILE = ROWS * D * 8, NT = NW * 64, NB = D / 16;
    extern __shared__ __attribute__((aligned(16))) char smem[];           // two tiles
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, c = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nblk = (a.Nq + NW * 32 - 1) / (NW * 32);
    int id = block_order();
    const int blk = nblk - 1 - id % nblk;                                 // under a causal mask the last queries have most to do: first
    id /= nblk;
    const int head = id % a.H, b = id / a.H, kvh = head / a.G;
    const int len = key_count(a, b), start = first_pos(a, b);
    const int q0 = blk * (NW * 32) + wave * 32, query = q0 + c;
    const int kend = visible(a, len, start, min(blk * (NW * 32) + NW * 32, a.Nq) - 1);
    const int lim = visible(a, len, start, query), lim_lo = visible(a, len, start, q0), lim_hi = visible(a, len, start, min(q0 + 31, a.Nq - 1));
    const int nt = (kend + ROWS - 1) / ROWS;

    bf16x8 qf[2][D / 16];
    {
        const bf16_t* qp = a.q + b * a.q_b + (long)min(query, a.Nq - 1) * a.q_n + 2 * head * a.q_h + 8 * h;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) qf[i][ks] = load8(qp + i * a.q_h + ks * 16);
    }
    float m[2] = {NONE, NONE}, l[2] = {0.f, 0.f};
    f32x16 o1[NB], o2[NB];
    clear(o1); clear(o2);
    Lane fl;
    fl.init(smem, lane);
    Stage<D, ROWS, NT> st;
    st.init(tid, a.k + b * a.k_b + 2 * kvh * a.k_h, a.k_n, a.k_h, a.v + b * a.v_b + kvh * a.v_h, a.v_n);
    if (nt > 0) {
        st.load(0, len);
        st.write(smem);
    }
    __syncthreads();
    for (int t = 0; t < nt; ++t) {
        if (t + 1 < nt) st.load((t + 1) * ROWS, len);
        const int k0 = t * ROWS;
        if (q0 < a.Nq) {
            const bool mask = k0 + ROWS > lim_lo;
#pragma unroll 1
            for (int r0 = 0; r0 < min(ROWS, lim_hi - k0); r0 += 32)
                forward_step<D, F16, ROWS>(fl.at((t & 1) * TILE + r0 * 128), r0, mask, lim - k0, h, a.c2, qf, m, l, o1, o2);
        }
        if (t + 1 < nt) st.write(smem + ((t + 1) & 1) * TILE);
        __syncthreads();
    }
    if (query >= a.Nq) return;
    const float lam = a.lam[head * a.lam_stride];
    float inv[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor(l[i], 32, 64);
        inv[i] = l[i] > 0.f ? 1.0f / l[i] : l[i] == 0.f ? 0.f : l[i];      // (a NaN stays one)
    }
    const long row = ((long)b * a.Nq + query) * a.H + head;
    if (a.maps) {
        store_rows<F16>(a.maps + row * 2 * D, o1, inv[0], h);
        store_rows<F16>(a.maps + ((long)a.B * a.Nq * a.H + row) * 2 * D, o2, inv[1], h);
        float* ls = a.lse + ((long)b * a.H + head) * 4 * a.Nq + query;
        if (h == 0) {
            put_lse(ls, 2 * a.Nq, m[0], l[0]);
            put_lse(ls + a.Nq, 2 * a.Nq, m[1], l[1]);
        }
    }
    const float w2 = lam * inv[1];
#pragma unroll
    for (int db = 0; db < NB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o1[db][r] = o1[db][r] * inv[0] - w2 * o2[db][r];
    store_rows<F16>(a.o + row * 2 * D, o1, 1.0f, h);
}

// ---- split forward: few queries against many keys ------------------------------------------------------------------------------------------
// HBM-bound: K and V are read once for all query heads of a key head.  A wave's 32 rows are (head of the group, query) pairs; a block takes one
// chunk of the keys, each of its waves every NW-th tile of 32 keys through LDS of its own (no barrier in the loop).  The waves' numerators are
// joined in LDS, and the chunks' by diff_join_kernel; with one chunk the result is written at once.
template <int D, bool F16, int NW>
__global__ __launch_bounds__(NW * 64, 1) void diff_split_kernel(Args a) {
    constexpr int ROWS = 32, TILE = ROWS * D * 8, NB = D / 16, NT = NW * 64, PER = 32 * 2 * D / NT;
    extern __shared__ __attribute__((aligned(16))) char smem[];           // NW tiles; then the waves' numerators of one map
    __shared__ float wm[2][NW][32], wl[2][NW][32];
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, c = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int id = blockIdx.x;
    const int split = id % a.nsplit; id /= a.nsplit;
    const int tile = id % a.tiles; id /= a.tiles;
    const int kvh = id % a.Hkv, b = id / a.Hkv;
    const int len = key_count(a, b), start = first_pos(a, b), rows = a.G * a.Nq;
    const int k0 = split * a.chunk;
    if (k0 >= len && a.nsplit > 1) return;                                // (the join reads the chunks that begin inside len alone)
    const int R = tile * 32 + c, Rc = min(R, rows - 1);
    const int head = kvh * a.G + Rc / a.Nq, query = Rc % a.Nq;
    const int lim = visible(a, len, start, query);
    int k1 = min(lim, k0 + a.chunk);                                      // end of the chunk's keys that some row of the tile sees
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) k1 = max(k1, __shfl_xor(k1, i, 64));
    k1 = __builtin_amdgcn_readfirstlane(k1);

    bf16x8 qf[2][D / 16];
    {
        const bf16_t* qp = a.q + b * a.q_b + query * a.q_n + 2 * head * a.q_h + 8 * h;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) qf[i][ks] = load8(qp + i * a.q_h + ks * 16);
    }
    float m[2] = {NONE, NONE}, l[2] = {0.f, 0.f};
    f32x16 o[2][NB];
    clear(o[0]); clear(o[1]);
    Lane fl;
    fl.init(smem, lane);
    Stage<D, ROWS, 64> st;
    st.init(lane, a.k + b * a.k_b + 2 * kvh * a.k_h, a.k_n, a.k_h, a.v + b * a.v_b + kvh * a.v_h, a.v_n);
    char* lds = smem + wave * TILE;
    int t = k0 + wave * ROWS;
    constexpr bool AHEAD = D < 128;                                       // (at d = 128 the next tile does not fit the registers beside the numerators)
    if (AHEAD && t < k1) st.load(t, len);
    for (; t < k1; t += NW * ROWS) {
        if (!AHEAD) st.load(t, len);
        st.write(lds);
        if (AHEAD && t + NW * ROWS < k1) st.load(t + NW * ROWS, len);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        forward_step<D, F16, ROWS>(fl.at(wave * TILE), 0, true, lim - t, h, a.c2, qf, m, l, o[0], o[1]);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor(l[i], 32, 64);
        if (h == 0) { wm[i][wave][c] = m[i]; wl[i][wave][c] = l[i]; }
    }
    float first[PER];
    const float lam = a.lam[head * a.lam_stride];
    // a thread joins PER columns of one row: row = tid % 32, columns from (tid / 32) PER
    const int jr = tid & 31, jc = (tid >> 5) * PER, JR = tile * 32 + jr;
    const long slot = (((long)(b * a.Hkv + kvh) * a.tiles + tile) * a.nsplit + split) * 2;
    float* stats = a.part + (long)a.B * a.Hkv * a.tiles * a.nsplit * 2 * 32 * (2 * D);
    float* num = (float*)smem;                                            // [wave][2 D][32]
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        __syncthreads();
        float M = NONE;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, wm[i][w][c]);
        const float f = __builtin_amdgcn_exp2f(m[i] - M);
#pragma unroll
        for (int db = 0; db < NB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) num[(wave * 2 * D + db * 32 + acc_row(r, h)) * 32 + c] = o[i][db][r] * f;
        __syncthreads();
        M = NONE;
        float L = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, wm[i][w][jr]);
#pragma unroll
        for (int w = 0; w < NW; ++w) L += wl[i][w][jr] * __builtin_amdgcn_exp2f(wm[i][w][jr] - M);
        const float inv = L > 0.f ? 1.0f / L : L == 0.f ? 0.f : L;
        if (JR < rows && a.nsplit > 1 && jc == 0) {
            stats[((slot + i) * 32 + jr) * 2] = M;
            stats[((slot + i) * 32 + jr) * 2 + 1] = L;
        }
        const int jh = kvh * a.G + min(JR, rows - 1) / a.Nq, jq = min(JR, rows - 1) % a.Nq;
        const long row = ((long)b * a.Nq + jq) * a.H + jh;
        const float jl = a.lam[jh * a.lam_stride];
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            float x = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) x += num[(w * 2 * D + jc + e) * 32 + jr];
            if (JR >= rows) continue;
            if (a.nsplit > 1) a.part[((slot + i) * 32 + jr) * (2 * D) + jc + e] = x;
            else {
                x *= inv;
                if (a.maps) a.maps[(i * (long)a.B * a.Nq * a.H + row) * 2 * D + jc + e] = f2h<F16>(x);
                if (i == 0) first[e] = x; else a.o[row * 2 * D + jc + e] = f2h<F16>(first[e] - jl * x);
            }
        }
        if (JR < rows && a.nsplit == 1 && a.maps && jc == 0)
            put_lse(a.lse + (((long)b * a.H + jh) * 4 + i) * a.Nq + jq, 2 * a.Nq, M, L);
    }
    (void)lam;
}

// joins the chunks of a row: a wave each
template <int D, bool F16>
__global__ __launch_bounds__(256) void diff_join_kernel(Args a) {
    constexpr int PER = 2 * D / 64;
    const int lane = threadIdx.x & 63;
    const long id = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= (long)a.B * a.H * a.Nq) return;
    const int query = id % a.Nq, head = id / a.Nq % a.H, b = id / a.Nq / a.H;
    const int kvh = head / a.G, R = (head % a.G) * a.Nq + query;
    const int n = (key_count(a, b) + a.chunk - 1) / a.chunk;              // <= nsplit
    const long slot = (((long)(b * a.Hkv + kvh) * a.tiles + (R >> 5)) * a.nsplit) * 2;
    const float* stats = a.part + (long)a.B * a.Hkv * a.tiles * a.nsplit * 2 * 32 * (2 * D) + (slot * 32 + (R & 31)) * 2;
    const float* num = a.part + (slot * 32 + (R & 31)) * (2 * D) + lane * PER;
    float out[2][PER];
    const long row = ((long)b * a.Nq + query) * a.H + head;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float M = NONE, L = 0.f;
        for (int s = lane; s < n; s += 64) M = fmaxf(M, stats[(s * 2 + i) * 64]);
        M = wave_max(M);
#pragma unroll
        for (int e = 0; e < PER; ++e) out[i][e] = 0.f;
        for (int s = 0; s < n; ++s) {
            const float w = __builtin_amdgcn_exp2f(stats[(s * 2 + i) * 64] - M);
            L += w * stats[(s * 2 + i) * 64 + 1];
            const float* x = num + (long)(s * 2 + i) * 32 * (2 * D);
#pragma unroll
            for (int e = 0; e < PER; ++e) out[i][e] += w * x[e];
        }
        const float inv = L > 0.f ? 1.0f / L : L == 0.f ? 0.f : L;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            out[i][e] *= inv;
            if (a.maps) a.maps[(i * (long)a.B * a.Nq * a.H + row) * 2 * D + lane * PER + e] = f2h<F16>(out[i][e]);
        }
        if (a.maps && lane == 0) put_lse(a.lse + (((long)b * a.H + head) * 4 + i) * a.Nq + query, 2 * a.Nq, M, L);
    }
    const float lam = a.lam[head * a.lam_stride];
#pragma unroll
    for (int e = 0; e < PER; ++e) a.o[row * 2 * D + lane * PER + e] = f2h<F16>(out[0][e] - lam * out[1][e]);
}

// ---- backward ----------------------------------------------------------------------------------------------------------------------------------
// D_m = dO . O_m: 2 d / 8 lanes a row (HBM-bound: three tensors once)
template <int D, bool F16>
__global__ __launch_bounds__(256) void diff_rows_kernel(Args a) {
    constexpr int LANES = D / 4;
    const long id = ((long)blockIdx.x * 256 + threadIdx.x) / LANES;       // (b, query, head)
    const int part = threadIdx.x % LANES;
    const long rows = (long)a.B * a.Nq * a.H;
    float d[2] = {0.f, 0.f};
    if (id < rows) {
        const int head = id % a.H, query = id / a.H % a.Nq, b = id / a.H / a.Nq;
        const u32x4 g = *(const u32x4*)(a.go + b * a.go_b + query * a.go_n + head * a.go_h + part * 8);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const u32x4 o = *(const u32x4*)(a.maps + (i * rows + id) * 2 * D + part * 8);
#pragma unroll
            for (int e = 0; e < 4; ++e) d[i] += unpack_lo<F16>(g[e]) * unpack_lo<F16>(o[e]) + unpack_hi<F16>(g[e]) * unpack_hi<F16>(o[e]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int s = LANES / 2; s > 0; s >>= 1) d[i] += __shfl_xor(d[i], s, 64);
    if (id < rows && part == 0) {
        const int head = id % a.H, query = id / a.H % a.Nq, b = id / a.H / a.Nq;
        float* p = a.D + ((long)b * a.H + head) * 2 * a.Nq + query;
        p[0] = d[0];
        p[a.Nq] = d[1];
    }
}

// dQ: queries stay, keys stream
template <int D, bool F16, int ROWS>
__device__ __forceinline__ void dq_step(const Lane& f, int r0, bool mask, int lim, int h, float c2, const bf16x8 (&qf)[2][D / 16], const bf16x8 (&gf)[D / 8],
                                        const float (&lse)[2], const float (&Dr)[2], float& x2, f32x16 (&dq1)[D / 32], f32x16 (&dq2)[D / 32]) {
    f32x16 s[2] = {zero16(), zero16()}, dp = zero16();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) s[i] = mfma32<F16>(f.template rows16<ROWS>(i * D + ks * 16), qf[i][ks], s[i]);
#pragma unroll
    for (int ks = 0; ks < D / 8; ++ks) dp = mfma32<F16>(f.template rows16<ROWS>(2 * D + ks * 16), gf[ks], dp);
    if (mask) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[i][r] = r0 + acc_row(r, h) < lim ? s[i][r] : -__builtin_inff();
    }
    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][r], c2, -lse[0]));
        const float p2 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[1][r], c2, -lse[1]));
        part[r & 3] = __builtin_fmaf(p2, dp[r], part[r & 3]);
        s[0][r] = p1 * (dp[r] - Dr[0]);
        s[1][r] = p2 * (dp[r] - Dr[1]);
    }
    x2 += (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
    for (int sp = 0; sp < 2; ++sp) {
        const bf16x8 d1 = pack8<F16>(s[0], sp), d2 = pack8<F16>(s[1], sp);
#pragma unroll
        for (int db = 0; db < D / 32; ++db) {
            dq1[db] = mfma32<F16>(f.template cols32<ROWS>(16 * sp, db * 32), d1, dq1[db]);
            dq2[db] = mfma32<F16>(f.template cols32<ROWS>(16 * sp, D + db * 32), d2, dq2[db]);
        }
    }
}

template <int D, bool F16, int NW>
__global__ __launch_bounds__(NW * 64, D == 128 ? 1 : 2) void diff_dq_kernel(Args a) {
    constexpr int ROWS = 64, TILE = ROWS * D * 8, NT = NW * 64;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, c = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nblk = (a.Nq + NW * 32 - 1) / (NW * 32);
    int id = block_order();
    const int blk = nblk - 1 - id % nblk;
    id /= nblk;
    const int head = id % a.H, b = id / a.H, kvh = head / a.G;
    const int len = key_count(a, b), start = first_pos(a, b);
    const int q0 = blk * (NW * 32) + wave * 32, query = q0 + c, qrow = min(query, a.Nq - 1);
    const int kend = visible(a, len, start, min(blk * (NW * 32) + NW * 32, a.Nq) - 1);
    const int lim = visible(a, len, start, query), lim_lo = visible(a, len, start, q0), lim_hi = visible(a, len, start, min(q0 + 31, a.Nq - 1));
    const int nt = (kend + ROWS - 1) / ROWS;
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
    const float lse[2] = {ls[0] - UP, ls[a.Nq] - UP};                     // (P comes out times 2^lo: taken off the sums at the end)
    const float unlo[2] = {__builtin_amdgcn_exp2f(-ls[2 * a.Nq]), __builtin_amdgcn_exp2f(-ls[3 * a.Nq])};
    const float Dr[2] = {a.D[bh * 2 * a.Nq + qrow], a.D[(bh * 2 + 1) * a.Nq + qrow]};
    float x2 = 0.f;
    f32x16 dq1[D / 32], dq2[D / 32];
    clear(dq1); clear(dq2);
    Lane fl;
    fl.init(smem, lane);
    Stage<D, ROWS, NT> st;
    st.init(tid, a.k + b * a.k_b + 2 * kvh * a.k_h, a.k_n, a.k_h, a.v + b * a.v_b + kvh * a.v_h, a.v_n);
    if (nt > 0) {
        st.load(0, len);
        st.write(smem);
    }
    __syncthreads();
    for (int t = 0; t < nt; ++t) {
        if (t + 1 < nt) st.load((t + 1) * ROWS, len);
        const int k0 = t * ROWS;
        if (q0 < a.Nq) {
            const bool mask = k0 + ROWS > lim_lo;
#pragma unroll 1
            for (int r0 = 0; r0 < min(ROWS, lim_hi - k0); r0 += 32)
                dq_step<D, F16, ROWS>(fl.at((t & 1) * TILE + r0 * 128), r0, mask, lim - k0, h, a.c2, qf, gf, lse, Dr, x2, dq1, dq2);
        }
        if (t + 1 < nt) st.write(smem + ((t + 1) & 1) * TILE);
        __syncthreads();
    }
    if (query >= a.Nq) return;
    const float down = F16 ? 1.0f / (1 << SHIFT16) : 1.0f, mul = a.scale * down;
    x2 += __shfl_xor(x2, 32, 64);
    if (h == 0) a.x2[bh * a.Nq + query] = x2 * down * unlo[1];
    bf16_t* p = a.dq + (((long)b * a.Nq + query) * a.H + head) * 2 * D;
    store_rows<F16>(p, dq1, mul * unlo[0], h);
    store_rows<F16>(p + D, dq2, -a.lam[head * a.lam_stride] * mul * unlo[1], h);
}

// dK, dV: keys stay, the queries of every head of the group stream.  At d = 128 the accumulators of both do not fit a lane's registers: two
// blocks then, one for dV (WHAT 1), one for dK (WHAT 2); else one for both (WHAT 3).
template <int D, bool F16, int ROWS, int WHAT>
__device__ __forceinline__ void dkv_step(const Lane& f, const float* rc, int r0, bool mask, int vis, int h, float c2, float lam, const bf16x8 (&kf)[2][D / 16],
                                         const bf16x8 (&vf)[D / 8], f32x16 (&dk1)[D / 32], f32x16 (&dk2)[D / 32], f32x16 (&dv)[D / 16]) {
    f32x16 s[2] = {zero16(), zero16()}, dp = zero16();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) s[i] = mfma32<F16>(f.template rows16<ROWS>(i * D + ks * 16), kf[i][ks], s[i]);
    if (WHAT & 2) {
#pragma unroll
        for (int ks = 0; ks < D / 8; ++ks) dp = mfma32<F16>(f.template rows16<ROWS>(2 * D + ks * 16), vf[ks], dp);
    }
    if (mask) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[i][r] = r0 + acc_row(r, h) >= vis ? s[i][r] : -__builtin_inff();
    }
    f32x16 pc;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int at = r0 + 8 * g + 4 * h;                                // rows of registers 4 g .. 4 g + 3
        const f32x4 e1 = *(const f32x4*)(rc + at), e2 = *(const f32x4*)(rc + ROWS + at);
        f32x4 d1, d2;
        if (WHAT & 2) { d1 = *(const f32x4*)(rc + 2 * ROWS + at); d2 = *(const f32x4*)(rc + 3 * ROWS + at); }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = 4 * g + e;
            float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][r], c2, -e1[e]));
            float p2 = lam * __builtin_amdgcn_exp2f(__builtin_fmaf(s[1][r], c2, -e2[e]));
            pc[r] = p1 - p2;
            if (WHAT & 2) {
                s[0][r] = p1 * (dp[r] - d1[e]);
                s[1][r] = p2 * (d2[e] - dp[r]);
            }
        }
    }
#pragma unroll
    for (int sp = 0; sp < 2; ++sp) {
        if (WHAT & 1) {
            const bf16x8 p = pack8<F16>(pc, sp);
#pragma unroll
            for (int db = 0; db < D / 16; ++db) dv[db] = mfma32<F16>(f.template cols32<ROWS>(16 * sp, 2 * D + db * 32), p, dv[db]);
        }
        if (WHAT & 2) {
            const bf16x8 d1 = pack8<F16>(s[0], sp), d2 = pack8<F16>(s[1], sp);
#pragma unroll
            for (int db = 0; db < D / 32; ++db) {
                dk1[db] = mfma32<F16>(f.template cols32<ROWS>(16 * sp, db * 32), d1, dk1[db]);
                dk2[db] = mfma32<F16>(f.template cols32<ROWS>(16 * sp, D + db * 32), d2, dk2[db]);
            }
        }
    }
}

template <int D, bool F16, int NW, int WHAT>
__global__ __launch_bounds__(NW * 64, 1) void diff_dkv_kernel(Args a) {
    constexpr int ROWS = 64, TILE = ROWS * D * 8, NT = NW * 64;
    extern __shared__ __attribute__((aligned(16))) char smem[];           // two tiles
    __shared__ __attribute__((aligned(16))) float rc[2][4 * ROWS];        // the tile's rows: lse of both maps, D of both
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5, c = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nblk = (a.Nk + NW * 32 - 1) / (NW * 32);
    int id = block_order();
    const int blk = id % nblk;                                            // under a causal mask the first keys have most to do: first
    id /= nblk;
    const int kvh = id % a.Hkv, b = id / a.Hkv;
    const int len = key_count(a, b), start = first_pos(a, b);
    const int kb = blk * (NW * 32), k0 = kb + wave * 32, key = k0 + c, krow = min(key, a.Nk - 1);
    // first query that sees the block's first key; the tiles of a head begin at its tile
    const int qfirst = a.causal ? max(0, kb - start) : 0;
    const int t0 = qfirst / ROWS, per = kb < len ? max(0, (a.Nq + ROWS - 1) / ROWS - t0) : 0, nt = per * a.G;
    // query rows that see the lane's key: those from vis on (none where the key does not count)
    const int vis = key >= len ? 0x7fffffff : a.causal ? key - start : -(1 << 30);
    const int vis_all = k0 + 31 >= len ? 0x7fffffff : a.causal ? k0 + 31 - start : -(1 << 30);      // ... that see all of the wave's
    const int vis_any = k0 >= len ? 0x7fffffff : a.causal ? k0 - start : -(1 << 30);

    bf16x8 kf[2][D / 16], vf[D / 8];
    {
        // (keys that do not count are not touched: their rows are cleared, so that nothing they hold can come through a product)
        const bf16x8 none = {0, 0, 0, 0, 0, 0, 0, 0};
        const bf16_t* kp = a.k + b * a.k_b + krow * a.k_n + 2 * kvh * a.k_h + 8 * h;
        const bf16_t* vp = a.v + b * a.v_b + krow * a.v_n + kvh * a.v_h + 8 * h;
        const bool counts = key < len;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) { kf[i][ks] = none; if (counts) kf[i][ks] = load8(kp + i * a.k_h + ks * 16); }
        if (WHAT & 2) {
#pragma unroll
            for (int ks = 0; ks < D / 8; ++ks) { vf[ks] = none; if (counts) vf[ks] = load8(vp + ks * 16); }
        }
    }
    f32x16 dk1[D / 32], dk2[D / 32], dv[D / 16];
    clear(dk1); clear(dk2); clear(dv);
    constexpr float UP = F16 ? SHIFT16 : 0;
    Lane fl;
    fl.init(smem, lane);
    Stage<D, ROWS, NT> st;
    float rr[4 * ROWS / NT];
    auto fetch = [&](int t) {
        const int head = kvh * a.G + t / per, q0 = (t0 + t % per) * ROWS;
        st.init(tid, a.q + b * a.q_b + 2 * head * a.q_h, a.q_n, a.q_h, a.go + b * a.go_b + head * a.go_h, a.go_n);
        st.load(q0, a.Nq);
        const long bh = ((long)b * a.H + head) * a.Nq;
#pragma unroll
        for (int i = 0; i < 4 * ROWS / NT; ++i) {
            const int j = i * NT + tid, which = j / ROWS, n = q0 + j % ROWS;
            rr[i] = which < 2 ? __builtin_inff() : 0.f;                   // a row behind the last: P = 0
            if (n < a.Nq) rr[i] = which < 2 ? a.lse[bh * 4 + which * a.Nq + n] + (a.lse[bh * 4 + (2 + which) * a.Nq + n] - UP) : a.D[bh * 2 + (which - 2) * a.Nq + n];
        }
    };
    auto put = [&](int s) {
        st.write(smem + s * TILE);
#pragma unroll
        for (int i = 0; i < 4 * ROWS / NT; ++i) rc[s][i * NT + tid] = rr[i];
    };
    if (nt > 0) {
        fetch(0);
        put(0);
    }
    __syncthreads();
    for (int t = 0; t < nt; ++t) {
        const float* r = rc[t & 1];
        if (t + 1 < nt) fetch(t + 1);
        const int q0 = (t0 + t % per) * ROWS;
        const float lam = a.lam[(kvh * a.G + t / per) * a.lam_stride];
        const bool mask = q0 < vis_all;
        const int v = vis == 0x7fffffff ? vis : vis - q0;
#pragma unroll 1
        for (int r0 = 0; r0 < ROWS; r0 += 32)
            if (q0 + r0 + 31 >= vis_any) dkv_step<D, F16, ROWS, WHAT>(fl.at((t & 1) * TILE + r0 * 128), r, r0, mask, v, h, a.c2, lam, kf, vf, dk1, dk2, dv);
        if (t + 1 < nt) put((t + 1) & 1);
        __syncthreads();
    }
    if (key >= a.Nk) return;
    const float down = F16 ? 1.0f / (1 << SHIFT16) : 1.0f;
    const long row = ((long)b * a.Nk + key) * a.Hkv + kvh;
    if (WHAT & 1) store_rows<F16>(a.dv + row * 2 * D, dv, down, h);
    if (WHAT & 2) {
        store_rows<F16>(a.dk + row * 2 * D, dk1, a.scale * down, h);
        store_rows<F16>(a.dk + row * 2 * D + D, dk2, a.scale * down, h);
    }
}

// dlam[h] = - sum over entries and queries of D_2 (all heads for one shared lam): a block each, in a fixed order, summed in 64 bits
__global__ __launch_bounds__(256) void diff_dlam_kernel(Args a, float* dlam) {
    __shared__ double red[256];
    const int h0 = a.lam_stride ? blockIdx.x : 0, nh = a.lam_stride ? 1 : a.H;
    double s = 0;
    for (int b = 0; b < a.B; ++b)
        for (long i = threadIdx.x; i < (long)nh * a.Nq; i += 256) s += a.x2[((long)b * a.H + h0) * a.Nq + i];
    red[threadIdx.x] = s;
    __syncthreads();
    for (int w = 128; w > 0; w >>= 1) {
        if ((int)threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x == 0) dlam[blockIdx.x] = (float)-red[0];
}

// ---- host --------------------------------------------------------------------------------------------------------------------------------------
int check(const hs_diff_attn_desc* d, bool backward) {
    if (!d || d->struct_size != sizeof(hs_diff_attn_desc)) return HS_ERR_ARG;
    if (d->dtype != HS_PREC_BF16 && d->dtype != HS_PREC_F16) return HS_ERR_ARG;
    if (!(d->scale > 0.f) || !(d->scale < 1e6f) || d->lam_stride < 0) return HS_ERR_ARG;
    if (d->B < 1 || d->Nq < 1 || d->Nk < 1 || d->H < 1 || d->Hkv < 1 || d->H % d->Hkv) return HS_ERR_SHAPE;
    if (d->d != 32 && d->d != 64 && d->d != 128) return HS_ERR_SHAPE;
    if (d->Nq > (1 << 28) || d->Nk > (1 << 28) || d->H > (1 << 16) || (int64_t)d->B * d->H * ((int64_t)d->Nq + d->Nk) > ((int64_t)1 << 36)) return HS_ERR_SHAPE;
    if ((int64_t)d->B * d->H * (((int64_t)(d->Nq > d->Nk ? d->Nq : d->Nk) + 127) / 128) > (1 << 30)) return HS_ERR_SHAPE;
    for (int64_t s : {d->q_b, d->q_n, d->q_h, d->k_b, d->k_n, d->k_h, d->v_b, d->v_n, d->v_h})
        if (s < 0 || (s & 7)) return HS_ERR_SHAPE;
    if (backward)
        for (int64_t s : {d->go_b, d->go_n, d->go_h})
            if (s < 0 || (s & 7)) return HS_ERR_SHAPE;
    return HS_OK;
}
bool misaligned(const void* p, unsigned n = 16) { return !p || (uintptr_t)p % n; }

struct Split { int tiles, nsplit, chunk; };
// Whether the split forward runs, and how it cuts the keys
Split split_of(const hs_diff_attn_desc* d) {
    const int64_t rows = (int64_t)(d->H / d->Hkv) * d->Nq, tiles = (rows + 31) / 32;
    if (rows > 32) return {0, 0, 0};
    const int64_t blocks = (int64_t)d->B * d->Hkv * tiles;
    int64_t want = (1024 + blocks - 1) / blocks;
    int64_t chunk = ((d->Nk + want - 1) / want + 127) / 128 * 128;
    if (chunk < 256) chunk = 256;
    return {(int)tiles, (int)((d->Nk + chunk - 1) / chunk), (int)chunk};
}
size_t split_bytes(const hs_diff_attn_desc* d, const Split& s) {
    return s.nsplit > 1 ? (size_t)d->B * d->Hkv * s.tiles * s.nsplit * 2 * 32 * (2 * d->d + 2) * 4 : 0;
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
template <int D, bool F16> void forward(const Args& a, const Split& sp, hipStream_t s) {
    if (sp.nsplit) {
        constexpr int NW = 4;
        launch(diff_split_kernel<D, F16, NW>, (int64_t)a.B * a.Hkv * sp.tiles * sp.nsplit, NW * 64, (size_t)NW * 256 * D, s, a);
        if (sp.nsplit > 1) launch(diff_join_kernel<D, F16>, ((int64_t)a.B * a.H * a.Nq + 3) / 4, 256, 0, s, a);
        return;
    }
    constexpr int NW = D == 128 ? 4 : 8;
    launch(diff_fwd_kernel<D, F16, NW>, (int64_t)a.B * a.H * ((a.Nq + NW * 32 - 1) / (NW * 32)), NW * 64, (size_t)2 * (D == 128 ? 32 : 64) * D * 8, s, a);
}
template <int D, bool F16> void backward(const Args& a, hipStream_t s) {
    constexpr int LANES = D / 4, NW = D == 128 ? 4 : 8;
    launch(diff_rows_kernel<D, F16>, ((int64_t)a.B * a.Nq * a.H * LANES + 255) / 256, 256, 0, s, a);
    launch(diff_dq_kernel<D, F16, NW>, (int64_t)a.B * a.H * ((a.Nq + NW * 32 - 1) / (NW * 32)), NW * 64, (size_t)2 * 64 * D * 8, s, a);
    const int64_t blocks = (int64_t)a.B * a.Hkv * ((a.Nk + 127) / 128);
    if constexpr (D == 128) {
        launch(diff_dkv_kernel<D, F16, 4, 1>, blocks, 256, (size_t)2 * 64 * D * 8, s, a);
        launch(diff_dkv_kernel<D, F16, 4, 2>, blocks, 256, (size_t)2 * 64 * D * 8, s, a);
    } else {
        launch(diff_dkv_kernel<D, F16, 4, 3>, blocks, 256, (size_t)2 * 64 * D * 8, s, a);
    }
}
#define HS_BY_TYPE(call)                                                               \
    do {                                                                               \
        const bool f16 = d->dtype == HS_PREC_F16;                                      \
        if (d->d == 32) { if (f16) call(32, true); else call(32, false); }             \
        else if (d->d == 64) { if (f16) call(64, true); else call(64, false); }        \
        else { if (f16) call(128, true); else call(128, false); }                      \
    } while (0)

}  // namespace

extern "C" size_t hs_diff_attn_fwd_ws_bytes(const hs_diff_attn_desc* d) { return check(d, false) == HS_OK ? split_bytes(d, split_of(d)) : 0; }
extern "C" size_t hs_diff_attn_bwd_ws_bytes(const hs_diff_attn_desc* d) { return check(d, false) == HS_OK ? (size_t)d->B * d->H * d->Nq * 12 : 0; }

extern "C" int hs_diff_attn_fwd(const hs_diff_attn_desc* d, const void* q, const void* k, const void* v, const float* lam, const int32_t* q_start,
                                const int32_t* kv_len, void* o, void* maps, float* lse, void* ws, size_t ws_bytes, void* stream) {
    const int rc = check(d, false);
    if (rc != HS_OK) return rc;
    if (!q || !k || !v || !o || !lam || !maps != !lse) return HS_ERR_ARG;
    if (misaligned(q) || misaligned(k) || misaligned(v) || misaligned(o) || (maps && misaligned(maps))) return HS_ERR_SHAPE;
    const Split sp = split_of(d);
    const size_t need = split_bytes(d, sp);
    if (need && (misaligned(ws) || ws_bytes < need)) return HS_ERR_SHAPE;
    Args a = args_of(d);
    a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.lam = lam; a.q_start = q_start; a.kv_len = kv_len;
    a.o = (bf16_t*)o; a.maps = (bf16_t*)maps; a.lse = lse; a.part = (float*)ws;
    a.tiles = sp.tiles; a.nsplit = sp.nsplit; a.chunk = sp.chunk;
    hipStream_t s = (hipStream_t)stream;
#define CALL(D, F) forward<D, F>(a, sp, s)
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
    if (ws_bytes < hs_diff_attn_bwd_ws_bytes(d)) return HS_ERR_SHAPE;
    Args a = args_of(d);
    a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.v = (const bf16_t*)v; a.go = (const bf16_t*)d_o; a.lam = lam;
    a.q_start = q_start; a.kv_len = kv_len; a.maps = (bf16_t*)maps; a.lse = (float*)lse;
    a.D = (float*)ws; a.x2 = a.D + (size_t)d->B * d->H * 2 * d->Nq;
    a.dq = (bf16_t*)dq; a.dk = (bf16_t*)dk; a.dv = (bf16_t*)dv;
    hipStream_t s = (hipStream_t)stream;
#define CALL(D, F) backward<D, F>(a, s)
    HS_BY_TYPE(CALL);
#undef CALL
    HS_CHECK_LAUNCH();
    hipLaunchKernelGGL(diff_dlam_kernel, dim3(a.lam_stride ? a.H : 1), dim3(256), 0, s, a, dlam);
    HS_CHECK_LAUNCH();
    return HS_OK;
}
