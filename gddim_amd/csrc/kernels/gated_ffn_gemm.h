// The matrix products of the gated feed-forward block (one translation unit per element type includes this).
//
//   forward    h = act(x Wg^T) (.) (x Wu^T)      both projections share the tiles of x; activation and product in the epilogue
//              y = h Wd^T
//   backward   dh = dy Wd, and in its epilogue    dgate = dh (.) up (.) act'(gate),   dup = dh (.) act(gate)
//              dx = dgate Wg + dup Wu              one sum over 2 F
//              dWg = dgate^T x, dWu = dup^T x, dWd = dy^T h     one launch
//
// C[m][n] = sum_k A[m][k] B[n][k].  Each operand lies in memory with k adjacent (KC: x, weights as torch.nn.Linear keeps them) or with its other index
// adjacent (the weights in dh and dx, everything in the weights' gradients); no operand is transposed in memory.
//
// Tiles.  A step of the k loop takes 64 bytes of k (32 16-bit or 16 float32 values) of BM rows of A and BN of B.  A fragment is 16 bytes a lane: row
// (lane % 16) and k = 8 (lane / 16) .. + 7 of a 16-row x 32-k block (16-bit types; the transposing LDS read gathers it where k is not adjacent), one
// v_mfma_f32_16x16x32; in float32 four values, four v_mfma_f32_16x16x4.  A sum does not care which k a lane holds as long as both operands agree, so
// both layouts and all types share one loop.  The MFMA's first operand is B: a lane then ends with four ADJACENT n of one row m.
// Memory goes to LDS directly, 16 bytes a lane (buffer_load ... lds: no registers, out-of-range pieces arrive as zeros); where rows are not whole
// 16-byte pieces, through registers.  KC rows take whole 128-byte lines, two steps a stage, 8 pieces of 16, piece c of row r at c ^ swizzle(r): with
// 64-byte rows the requests to L2 doubled and became the bound (y of 16384 x 1024 x 4096: 153 us instead of 129).  Other operands keep their k rows, pieces
// moved by k.  No bank conflicts either way (counted).
// Step k multiplies fragments that were read during step k - 1, while those of step k + 1 are read.  Stages lie in a ring: two of two steps, or four of one
// step where no operand is KC; a stage is requested into the place of one that all waves have read, two / three steps (2048 / 3072 MFMA cycles of a
// 256 x 256 tile) before it is read.
//
// All sums are float32 in the matrix core's accumulators.  Rounded to the tensors' type are only operands of a next product, as the 16-bit matrix core
// wants them -- h, dgate, dup -- and the results.  gate and up, which a training step keeps, stay float32: rounded to bf16 they put the gradients at
// 1.8 times the error of one final rounding (relative 3.1e-3 instead of 2.4e-3; 1.7e-3 is the final rounding alone).
#pragma once
#include "../common.h"
#include "../token_ops.h"

namespace gd {
namespace ffn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename T> struct quad { typedef T type __attribute__((ext_vector_type(4))); };

// ---- activation and its derivative, float32 ----
// Exponentials and quotients are the hardware's (v_exp_f32, v_rcp_f32, one step of float32 each): an absolute error of a few 2^-24 in a sigmoid or a
// tanh is the same in its product with z, relative to |z|; with the library's forms the epilogue took as long as the products.
__device__ __forceinline__ float fast_exp(float z) { return __builtin_amdgcn_exp2f(z * 1.44269504088896341f); }
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + fast_exp(-z)); }
__device__ __forceinline__ float fast_tanh(float z) { return 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + fast_exp(2.f * z)); }

template <int ACT> __device__ __forceinline__ float act_value(float z) {
    if constexpr (ACT == GD_ACT_SILU) return z * sigmoid(z);
    else if constexpr (ACT == GD_ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    else return 0.5f * z * (1.f + fast_tanh(0.79788456080286536f * (z + 0.044715f * z * z * z)));
}

template <int ACT> __device__ __forceinline__ void act_grad(float z, float &a, float &da) {
    if constexpr (ACT == GD_ACT_SILU) {
        const float s = sigmoid(z);
        a = z * s;
        da = s + a * (1.f - s);
    } else if constexpr (ACT == GD_ACT_GELU) {
        const float c = 0.5f * (1.f + erff(z * 0.70710678118654752f));
        a = z * c;
        da = c + z * 0.39894228040143268f * fast_exp(-0.5f * z * z);
    } else {
        const float t = fast_tanh(0.79788456080286536f * (z + 0.044715f * z * z * z));
        a = 0.5f * z * (1.f + t);
        da = 0.5f * (1.f + t) + 0.5f * z * (1.f - t * t) * 0.79788456080286536f * (1.f + 0.134145f * z * z);
    }
}

// ---- epilogues on four adjacent columns of one row ----
template <typename T> __device__ __forceinline__ void store4(void *p, long long o, f32x4 v, int n_left, bool whole) {
    T *d = static_cast<T *>(p) + o;
    if (whole) *reinterpret_cast<typename quad<T>::type *>(d) = __builtin_convertvector(v, typename quad<T>::type);
    else
        for (int i = 0; i < 4 && i < n_left; ++i) d[i] = (T)v[i];
}

template <typename T> __device__ __forceinline__ f32x4 load4(const void *p, long long o, int n_left, bool whole) {
    const T *d = static_cast<const T *>(p) + o;
    if (whole) return __builtin_convertvector(*reinterpret_cast<const typename quad<T>::type *>(d), f32x4);
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < 4 && i < n_left; ++i) v[i] = (float)d[i];
    return v;
}

// row m, columns n .. n + 3; c1: up (EPI_GATED), g / u: gate and up as kept (EPI_GATED_BWD)
template <typename T, int EPI, int ACT>
__device__ __forceinline__ void epilogue_act(const GemmProblem &q, int m, int n, f32x4 c0, f32x4 c1, f32x4 g, f32x4 u) {
    const int left = q.N - n;
    if (m >= q.M || left <= 0) return;
    const bool whole = q.quads && left >= 4;
    const long long o = (long long)m * q.N + n;
    if constexpr (EPI == EPI_STORE) store4<T>(q.out[0], o, c0, left, whole);
    else if constexpr (EPI == EPI_GATED) {
        f32x4 h;
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = act_value<ACT>(c0[e]) * c1[e];
        store4<T>(q.out[0], o, h, left, whole);
        if (q.out[1]) {
            store4<float>(q.out[1], o, c0, left, whole);
            store4<float>(q.out[2], o, c1, left, whole);
        }
    } else {
        f32x4 dg, du;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float a, da;
            act_grad<ACT>(g[e], a, da);
            dg[e] = c0[e] * u[e] * da;
            du[e] = c0[e] * a;
        }
        store4<T>(q.out[0], o, dg, left, whole);
        store4<T>(q.out[1], o, du, left, whole);
    }
}

template <typename T, int EPI>
__device__ __forceinline__ void epilogue(const GemmProblem &q, int act, int m, int n, f32x4 c0, f32x4 c1, f32x4 g, f32x4 u) {
    if (EPI == EPI_STORE || act == GD_ACT_SILU) epilogue_act<T, EPI, GD_ACT_SILU>(q, m, n, c0, c1, g, u);
    else if (act == GD_ACT_GELU) epilogue_act<T, EPI, GD_ACT_GELU>(q, m, n, c0, c1, g, u);
    else epilogue_act<T, EPI, GD_ACT_GELU_TANH>(q, m, n, c0, c1, g, u);
}

// what EPI_GATED_BWD reads
__device__ __forceinline__ void load_kept(const GemmProblem &q, int m, int n, f32x4 &g, f32x4 &u) {
    const int left = q.N - n;
    g = u = f32x4{0.f, 0.f, 0.f, 0.f};
    if (m >= q.M || left <= 0) return;
    const bool whole = q.quads && left >= 4;
    const long long o = (long long)m * q.N + n;
    g = load4<float>(q.in[0], o, left, whole);
    u = load4<float>(q.in[1], o, left, whole);
}

// ---- one 16-byte fragment each: acc += B-fragment x A-fragment ----
template <typename T> __device__ __forceinline__ f32x4 mma(i32x4 b, i32x4 a, f32x4 c);
template <> __device__ __forceinline__ f32x4 mma<__bf16>(i32x4 b, i32x4 a, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mma<_Float16>(i32x4 b, i32x4 a, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mma<float>(i32x4 b, i32x4 a, f32x4 c) {
    const f32x4 bf = __builtin_bit_cast(f32x4, b), af = __builtin_bit_cast(f32x4, a);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(bf[i], af[i], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ int kc_swizzle(int row) { return (row >> 1) & 7; }

// a raw buffer of `bytes` bytes: reads past its end give zeros
__device__ __forceinline__ i32x4 buffer_of(const char *p, int bytes) {
    const unsigned long long v = (unsigned long long)p;
    i32x4 r = {(int)(unsigned)v, (int)((unsigned)(v >> 32) & 0xffffu), bytes, 0x00020000};
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __builtin_amdgcn_readfirstlane(r[i]);
    return r;
}

// 16 bytes a lane from buffer + off straight to LDS at lds + 16 lane.  Written out rather than taken from the builtin, after which the compiler
// waits for every such request (vmcnt(0)) before each transposing LDS read, though the ring keeps their places apart: wait_loads + lds_barrier below say when
// a stage has arrived.  The instruction has no register result.
__device__ __forceinline__ void load_to_lds(i32x4 buffer, unsigned off, char *lds) {
    const int at = __builtin_amdgcn_readfirstlane((int)(unsigned long long)(__attribute__((address_space(3))) char *)lds);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(at), "v"(off), "s"(buffer) : "memory", "m0");
}

constexpr unsigned OUT_OF_RANGE = 0x80000000u;  // a buffer offset past every num_records used here: the piece arrives as zeros

// One operand: R rows (of m or n) x STEPS * 64 bytes of k per stage
template <typename T, int R, bool KC, int STEPS, int THREADS, bool GATED_B>
struct Operand {
    static_assert(!KC || STEPS == 2, "rows of whole 128-byte lines");
    static constexpr int ES = sizeof(T), KSTAGE = STEPS * 64 / ES, V = 16 / ES;  // k per stage, elements of a piece
    static constexpr int WAVES = THREADS / 64;
    static constexpr int PIECES = R * 4 * STEPS / THREADS;                // 16-byte pieces a thread stages
    static constexpr int CPR = KC ? 8 : R * ES / 16;                      // pieces of an LDS row
    static constexpr int BYTES = R * 64 * STEPS;

    const char *base[2];   // element (first row, k = 0) of each source
    long long end[2];      // bytes from there to the end of the matrix
    long long ld;          // bytes
    int k_len;             // k of one source
    int rows_left;         // rows (KC) / columns (else) from the tile's first
    int row[PIECES], piece[PIECES];  // of the matrix tile: KC row / k row; source piece

    __device__ __forceinline__ void init(int wave, int lane) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int slot = (i * WAVES + wave) * 64 + lane;  // 16-byte slot of the stage
            row[i] = slot / CPR;
            piece[i] = (slot % CPR) ^ swizzle(row[i]);
        }
    }
    __device__ static __forceinline__ int swizzle(int r) {
        if constexpr (KC) return kc_swizzle(r);
        else if constexpr (ES == 2) return 2 * (r & 3) + 8 * ((r >> 3) & 1);
        else return 4 * ((r >> 2) & 3);
    }
    // gated B tiles: rows of gate and up alternate in blocks of 32, so that a wave's 64 columns hold both of its 32
    __device__ static __forceinline__ int source_of(int r) { return GATED_B ? (r >> 5) & 1 : 0; }
    __device__ static __forceinline__ int row_in_source(int r) { return GATED_B ? ((r >> 6) << 5) + (r & 31) : r; }

    // stage st (src: which source of a two-part sum) straight into LDS
    __device__ __forceinline__ void stage_direct(char *lds, int src, int st, int wave) const {
        const long long adv = KC ? (long long)st * 128 : (long long)st * KSTAGE * ld;
        i32x4 rs[GATED_B ? 2 : 1];
#pragma unroll
        for (int g = 0; g < (GATED_B ? 2 : 1); ++g) {
            const int s = GATED_B ? g : src;
            long long left = end[s] - adv;
            left = left < 0 ? 0 : left > 0x7fffffffLL ? 0x7fffffffLL : left;
            rs[g] = buffer_of(base[s] + adv, (int)left);
        }
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            unsigned off;
            bool in;
            if constexpr (KC) {
                off = (unsigned)row_in_source(row[i]) * (unsigned)ld + piece[i] * 16;
                in = st * KSTAGE + piece[i] * V < k_len;
            } else {
                off = (unsigned)row[i] * (unsigned)ld + piece[i] * 16;
                in = st * KSTAGE + row[i] < k_len;
            }
            off = in ? off : OUT_OF_RANGE;
            const int g = GATED_B ? source_of((i * WAVES + wave) * 64 / CPR) : 0;
            load_to_lds(rs[g], off, lds + (i * WAVES + wave) * 1024);
        }
    }
    // ... through registers, for rows that are not whole aligned pieces
    __device__ __forceinline__ void load_regs(i32x4 *r, int src, int st) const {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int k0 = st * KSTAGE + (KC ? piece[i] * V : row[i]);
            const int s = GATED_B ? source_of(row[i]) : src;
            const int rr = KC ? row_in_source(row[i]) : piece[i] * V;  // first row / column
            const char *p = KC ? base[s] + (long long)rr * ld + (long long)k0 * ES : base[s] + (long long)k0 * ld + (long long)rr * ES;
            const bool line = KC ? rr < rows_left : k0 < k_len;
            const int left = line ? (KC ? k_len - k0 : rows_left - rr) : 0;
            r[i] = i32x4{0, 0, 0, 0};
            if (left >= V) __builtin_memcpy(&r[i], p, 16);
            else if (left > 0) {
                T t[V];
#pragma unroll
                for (int j = 0; j < V; ++j) t[j] = j < left ? reinterpret_cast<const T *>(p)[j] : (T)0.f;
                __builtin_memcpy(&r[i], t, 16);
            }
        }
    }
    __device__ __forceinline__ void store_regs(char *lds, const i32x4 *r, int wave, int lane) const {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) *reinterpret_cast<i32x4 *>(lds + ((i * WAVES + wave) * 64 + lane) * 16) = r[i];
    }

    // fragment: rows r0 + lane % 16, k of the stage's step `sub`
    __device__ static __forceinline__ i32x4 fragment(const char *lds, int r0, int sub, int lane) {
        const int i = lane & 15, g = lane >> 4;
        if constexpr (KC) {
            const int r = r0 + i;
            return *reinterpret_cast<const i32x4 *>(lds + r * 128 + (((sub * 4 + g) ^ kc_swizzle(r)) << 4));
        } else if constexpr (ES == 2) {
            typedef __attribute__((address_space(3))) i16x4 *lds_ptr;
            const int k = sub * 32 + g * 8 + (i >> 2);
            const char *p = lds + k * (R * 2) + (((r0 / 8 + ((i & 3) >> 1)) ^ swizzle(k)) << 4) + (i & 1) * 8;
            const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p);
            const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 4 * R * 2));
            return __builtin_bit_cast(i32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            f32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = sub * 16 + g * 4 + j, c = r0 + i;
                v[j] = *reinterpret_cast<const float *>(lds + k * (R * 4) + (((c >> 2) ^ swizzle(k)) << 4) + (c & 3) * 4);
            }
            return __builtin_bit_cast(i32x4, v);
        }
    }
};

// s_waitcnt vmcnt(n), the other counters left alone
template <int N> __device__ __forceinline__ void wait_loads() {
    static_assert(N < 64, "");
    __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | ((N >> 4) << 14));
}
// what this wave wrote to and read from LDS is done, and so it is for everyone; requests to global memory stay on their way
__device__ __forceinline__ void lds_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// workgroup -> (problem, tile, split): workgroups go round-robin over the 8 XCDs, each with an L2 of its own; consecutive tiles of one XCD share
// operand rows, eight m tiles to a group
struct Place {
    int problem, mt, nt, split;
};
__device__ __forceinline__ Place place(const GemmLaunch &p) {
    const int total = gridDim.x, id = blockIdx.x;
    const int q = total >> 3, r = total & 7, xcd = id & 7;
    int t = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (id >> 3);
    Place w;
    w.problem = 0;
    while (w.problem + 1 < p.problems && t >= p.q[w.problem].blocks) t -= p.q[w.problem++].blocks;
    const GemmProblem &g = p.q[w.problem];
    const int tiles = g.tiles_m * g.tiles_n;
    w.split = t / tiles;
    t -= w.split * tiles;
    const int group = 8 * g.tiles_n;
    const int first = t / group * 8, size = min(8, g.tiles_m - first);
    t %= group;
    w.mt = first + t % size;
    w.nt = t / size;
    return w;
}

template <typename T, int BM, int BN, int WM, int WN, bool AKC, bool BKC, int EPI, bool DIRECT>
__global__ __launch_bounds__(WM *WN * 64, 1) void gemm_kernel(const GemmLaunch p) {
    constexpr int THREADS = WM * WN * 64;
    constexpr bool GATED = EPI == EPI_GATED;
    constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
    static_assert(TN == 64 && TM % 64 == 0, "a wave's 64 columns (32 of gate and 32 of up) and groups of 64 rows go through 16 KB of LDS");
    constexpr int STEPS = AKC || BKC || !DIRECT ? 2 : 1, RING = 4 / STEPS;
    typedef Operand<T, BM, AKC, STEPS, THREADS, false> OpA;
    typedef Operand<T, BN, BKC, STEPS, THREADS, GATED> OpB;
    constexpr int STAGE = OpA::BYTES + OpB::BYTES, LOADS = OpA::PIECES + OpB::PIECES;
    static_assert(WM * WN * 16384 <= RING * STAGE, "");
    constexpr int KSTAGE = OpA::KSTAGE;
    __shared__ __attribute__((aligned(16))) char lds[RING * STAGE];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const Place w = place(p);
    const GemmProblem &q = p.q[w.problem];
    const int m0 = w.mt * BM, n0 = w.nt * (GATED ? BN / 2 : BN);

    OpA a;
    OpB b;
    a.init(wave, lane);
    b.init(wave, lane);
    a.ld = q.lda; b.ld = q.ldb;
    a.k_len = b.k_len = q.K;
    a.rows_left = q.M - m0; b.rows_left = q.N - n0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const long long oa = AKC ? (long long)m0 * q.lda : (long long)m0 * sizeof(T);
        const long long ob = BKC ? (long long)n0 * q.ldb : (long long)n0 * sizeof(T);
        a.base[s] = static_cast<const char *>(q.a[s]) + oa;
        b.base[s] = static_cast<const char *>(q.b[s]) + ob;
        a.end[s] = q.a_bytes - oa;
        b.end[s] = q.b_bytes - ob;
    }
    const int per_part = (q.K + KSTAGE - 1) / KSTAGE;  // stages of one part of the sum
    const int st0 = w.split * q.stages_per_split;
    const int st1 = min(st0 + q.stages_per_split, per_part * q.parts);

    f32x4 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    i32x4 ra[DIRECT ? 1 : OpA::PIECES], rb[DIRECT ? 1 : OpB::PIECES];
    auto place_of = [&](int st) __attribute__((always_inline)) { return lds + ((st - st0) & (RING - 1)) * STAGE; };
    auto fetch = [&](int st) __attribute__((always_inline)) {
        const int src = st >= per_part, k = src ? st - per_part : st;
        if constexpr (DIRECT) {
            a.stage_direct(place_of(st), src, k, wave);
            b.stage_direct(place_of(st) + OpA::BYTES, src, k, wave);
        } else {
            a.load_regs(ra, src, k);
            b.load_regs(rb, src, k);
        }
    };
    auto commit = [&](int st) __attribute__((always_inline)) {
        a.store_regs(place_of(st), ra, wave, lane);
        b.store_regs(place_of(st) + OpA::BYTES, rb, wave, lane);
    };
    i32x4 fa[2][FM], fb[2][FN];
    auto read = [&](int st, int sub, int set) __attribute__((always_inline)) {
        const char *at = place_of(st);
#pragma unroll
        for (int i = 0; i < FN; ++i) fb[set][i] = OpB::fragment(at + OpA::BYTES, wn * TN + i * 16, sub, lane);
#pragma unroll
        for (int j = 0; j < FM; ++j) fa[set][j] = OpA::fragment(at, wm * TM + j * 16, sub, lane);
    };
    auto multiply = [&](int set) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FM; ++j) acc[i][j] = mma<T>(fb[set][i], fa[set][j], acc[i][j]);
    };
    // step `sub` of stage st, its fragments in (or on their way to) set.  At the stage's last step all its fragments have been read: behind the barrier its place
    // is free and the next stage complete.  full: stages up to st + RING exist (no conditions in the long part of the loop)
    auto step = [&](int st, int sub, int set, bool full) __attribute__((always_inline)) {
        if (sub + 1 < STEPS) read(st, sub + 1, set ^ 1);
        else if (full || st + 1 < st1) {
            if constexpr (DIRECT) {
                if (full || st + RING - 1 < st1) wait_loads<(RING - 2) * LOADS>();  // stages up to st + RING - 1 have been requested
                else wait_loads<0>();
            } else commit(st + 1);
            lds_barrier();
            if constexpr (DIRECT) {
                if (full || st + RING < st1) fetch(st + RING);
            } else {
                if (full || st + 2 < st1) fetch(st + 2);
            }
            read(st + 1, 0, set ^ 1);
        }
        multiply(set);
        __builtin_amdgcn_sched_barrier(0);  // the products stay between the reads and the next barrier: they cover the reads' way
    };

    if (st0 < st1) {
        if constexpr (DIRECT) {
#pragma unroll
            for (int k = 0; k < RING; ++k)
                if (st0 + k < st1) fetch(st0 + k);
            if (st0 + RING <= st1) wait_loads<(RING - 1) * LOADS>();
            else wait_loads<0>();
        } else {
            fetch(st0);
            commit(st0);
            if (st0 + 1 < st1) fetch(st0 + 1);
        }
        lds_barrier();
        read(st0, 0, 0);
        int st = st0;
        if constexpr (STEPS == 2) {
            for (; st + RING < st1; ++st) {
                step(st, 0, 0, true);
                step(st, 1, 1, true);
            }
            for (; st < st1; ++st) {
                step(st, 0, 0, false);
                step(st, 1, 1, false);
            }
        } else {
            for (; st + 1 + RING < st1; st += 2) {
                step(st, 0, 0, true);
                step(st + 1, 0, 1, true);
            }
            for (; st < st1; st += 2) {
                step(st, 0, 0, false);
                if (st + 1 < st1) step(st + 1, 0, 1, false);
            }
        }
    }

    constexpr int NI = GATED ? FN / 2 : FN;
    const int mw = m0 + wm * TM, nw = n0 + wn * (GATED ? TN / 2 : TN);  // the wave's first row and column
    if (q.splits == 1) {
        // The accumulators go through LDS, 64 rows of the wave at a time (16 KB a wave, 16-byte pieces of row r at piece ^ r), and come back row by row:
        // global memory is read and written in whole lines, and the loop over them stays a loop (unrolled over the accumulators, three activations
        // kept the accumulators in scratch memory: dh of 16384 x 4096 x 1024 with its epilogue took 977 us, now 329).
        constexpr int LPR = GATED ? 8 : 16, RPI = 64 / LPR, ITER = 64 / RPI, BATCH = 4;
        char *mine = lds + wave * 16384;
        __syncthreads();  // every wave has read the last stage
#pragma unroll
        for (int jc = 0; jc < FM; jc += 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < FN; ++i) {
                    const int r = j * 16 + (lane & 15);
                    *reinterpret_cast<f32x4 *>(mine + r * 256 + (((i * 4 + (lane >> 4)) ^ (r & 15)) << 4)) = acc[i][jc + j];
                }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const int piece = lane & (LPR - 1), n = nw + piece * 4;
#pragma unroll 1
            for (int it = 0; it < ITER; it += BATCH) {
                f32x4 g[BATCH], u[BATCH];
#pragma unroll
                for (int k = 0; k < BATCH; ++k) {
                    g[k] = u[k] = f32x4{0.f, 0.f, 0.f, 0.f};
                    if constexpr (EPI == EPI_GATED_BWD) load_kept(q, mw + jc * 16 + (it + k) * RPI + lane / LPR, n, g[k], u[k]);
                }
#pragma unroll
                for (int k = 0; k < BATCH; ++k) {
                    const int r = (it + k) * RPI + lane / LPR;
                    const f32x4 c0 = *reinterpret_cast<const f32x4 *>(mine + r * 256 + ((piece ^ (r & 15)) << 4));
                    f32x4 c1 = {0.f, 0.f, 0.f, 0.f};
                    if constexpr (GATED) c1 = *reinterpret_cast<const f32x4 *>(mine + r * 256 + (((piece + 8) ^ (r & 15)) << 4));
                    epilogue<T, EPI>(q, p.act, mw + jc * 16 + r, n, c0, c1, g[k], u[k]);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    } else {
        // partial sums, rows padded to whole quads: [split][plane][M][N4]
        const long long n4 = (q.N + 3) & ~3, plane = (long long)q.M * n4;
        float *part = q.partial + (long long)w.split * (GATED ? 2 : 1) * plane;
        const int nr = nw + (lane >> 4) * 4;
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int m = mw + (lane & 15) + j * 16;
            if (m >= q.M) continue;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                if (nr + i * 16 >= q.N) continue;
                float *d = part + (long long)m * n4 + nr + i * 16;
                *reinterpret_cast<f32x4 *>(d) = acc[i][j];
                if constexpr (GATED) *reinterpret_cast<f32x4 *>(d + plane) = acc[(i + NI) % FN][j];
            }
        }
    }
}

// the splits' partial sums in order, then the epilogue: one quad of columns per thread
template <typename T, int EPI>
__global__ __launch_bounds__(256) void join_kernel(const GemmLaunch p) {
    constexpr bool GATED = EPI == EPI_GATED;
    long long t = (long long)blockIdx.x * 256 + threadIdx.x;
    int k = 0;
    while (k + 1 < p.problems && t >= p.q[k].join_threads) t -= p.q[k++].join_threads;
    const GemmProblem &q = p.q[k];
    if (q.splits == 1 || t >= q.join_threads) return;
    const int quads = (q.N + 3) >> 2;
    const int m = (int)(t / quads), n = (int)(t - (long long)m * quads) * 4;
    if (m >= q.M) return;
    const long long n4 = (long long)quads * 4, plane = (long long)q.M * n4;
    const float *d = q.partial + (long long)m * n4 + n;
    f32x4 c0 = {0.f, 0.f, 0.f, 0.f}, c1 = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < q.splits; ++s) {
        c0 += *reinterpret_cast<const f32x4 *>(d + (long long)s * (GATED ? 2 : 1) * plane);
        if constexpr (GATED) c1 += *reinterpret_cast<const f32x4 *>(d + (long long)s * 2 * plane + plane);
    }
    f32x4 g = {0.f, 0.f, 0.f, 0.f}, u = g;
    if constexpr (EPI == EPI_GATED_BWD) load_kept(q, m, n, g, u);
    epilogue<T, EPI>(q, p.act, m, n, c0, c1, g, u);
}

template <typename T, bool AKC, bool BKC, int EPI>
int launch_gemm(const GemmLaunch &p, int blocks, hipStream_t s) {
    if (blocks > 0) {
        if (p.tile == TILE_256) {
            if constexpr (sizeof(T) == 2) gemm_kernel<T, 256, 256, 2, 4, AKC, BKC, EPI, true><<<blocks, 512, 0, s>>>(p);
        } else if (p.direct) gemm_kernel<T, 128, 128, 2, 2, AKC, BKC, EPI, true><<<blocks, 256, 0, s>>>(p);
        else gemm_kernel<T, 128, 128, 2, 2, AKC, BKC, EPI, false><<<blocks, 256, 0, s>>>(p);
        GD_HIP(hipGetLastError());
    }
    if (p.join_blocks > 0) {
        join_kernel<T, EPI><<<p.join_blocks, 256, 0, s>>>(p);
        GD_HIP(hipGetLastError());
    }
    return 0;
}

template <typename T>
int launch_type(const GemmLaunch &p, GemmKind kind, int blocks, hipStream_t s) {
    switch (kind) {
        case GEMM_GATE_UP: return launch_gemm<T, true, true, EPI_GATED>(p, blocks, s);
        case GEMM_DOWN: return launch_gemm<T, true, true, EPI_STORE>(p, blocks, s);
        case GEMM_DHIDDEN: return launch_gemm<T, true, false, EPI_GATED_BWD>(p, blocks, s);
        case GEMM_DX: return launch_gemm<T, true, false, EPI_STORE>(p, blocks, s);
        case GEMM_DW: return launch_gemm<T, false, false, EPI_STORE>(p, blocks, s);
    }
    return 1;
}

}  // namespace ffn
}  // namespace gd
