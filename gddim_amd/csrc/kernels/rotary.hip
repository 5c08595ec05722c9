// Rotary positions with several axes, and RMS norms of queries and keys for each head with that rotation in the same pass.
//
//   rotation      pair p of a head (p < R/2) belongs to axis a(p) and turns by phi = pos[token][a(p)] * freq[p]:
//                     (a, b) -> (a cos phi - b sin phi, a sin phi + b cos phi);  channels >= R pass through
//   norm          y = rotation(w (.) x * rho),  rho = (mean_D x^2 + eps)^-1/2
//   its gradient  g = rotation^-1(dy);  dx = rho (g w - xh mean_D(g w xh)),  xh = x rho;  dw = sum over tokens and heads of g xh
//
// All three are bound by HBM: each element is read once and written once (the gradient: two reads, one write), everything between stays in
// registers.  What would cost more than the bytes is the angle: far positions times a frequency need 64 bits before the whole turns are
// taken off.  One wave therefore takes a token -- or, with few tokens, a share of a token's heads -- computes the R/2 cosines and sines ONCE
// (lane p pair p) into a table of its own in LDS, and walks the token's query and key heads with them.  A token has few heads (20 heads of 128
// channels are three steps of a wave), so what a token begins with is read while the one before it is worked on: its positions, and behind the last heads of
// the one its first; the sums of a head are lane permutes and its root the hardware's.
//
// Layout: a lane holds W pairs = two vectors of W channels.  (i, i + R/2) pairs: vector 0 from the first half, vector 1 from the second;
// (2i, 2i + 1) pairs: 2W adjacent channels.  No pair spans two lanes, and a lane keeps its pairs from head to head: the weight-gradient sums stay in
// registers (norm weights come from LDS, queries and keys apart).  lp lanes hold a head (with the norm a power of two: its sums are log2 lp permutes), 64 / lp
// heads are in flight per wave.  Channels that pass through lie in lanes as pairs do, and every pair behind the last section is kept from the rotation by a
// choice: a product with cos 0 = 1 and sin 0 = 0 would hand a neighbour's infinity on as NaN.
//
// W is 16 bytes of a type where pairs, strides and addresses allow it (the gradient in 16-bit types: 8), 8 bytes else, one pair where nothing is aligned.
//
// Measured, against the bytes at the 5.1 TB/s of a large copy: rotation of 46800 x 16 x 128 bf16 (383 MB) 80 us, 4.8 TB/s; norm and rotation of 65536 tokens x
// (4 + 4) x 64 float32 (268 MB) 57 us, 4.7 TB/s, and its gradient (403 MB) 87 us, 4.6 TB/s; of 16382 x (16 + 4) x 128 bf16 (168 MB) 43 us, 3.9 TB/s, and its
// gradient (252 MB) 76 us, 3.3 TB/s, + 5 us for the weights' sums.  The 16-bit gradient has 16 waves a CU (119 registers), each with loads of 8 bytes.
#include <type_traits>

#include "../common.h"
#include "../token_ops.h"

namespace gd {

namespace {

template <typename T, int W> struct vec_of { typedef T type __attribute__((ext_vector_type(W))); };
template <typename T> struct vec_of<T, 1> { typedef T type; };
template <typename T, int W> using vec = typename vec_of<T, W>::type;

template <typename T, int W> __device__ __forceinline__ void to_f32(const vec<T, W> &v, float *f) {
    if constexpr (W == 1) f[0] = (float)v;
    else {
#pragma unroll
        for (int i = 0; i < W; ++i) f[i] = (float)v[i];
    }
}

template <typename T, int W> __device__ __forceinline__ vec<T, W> from_f32(const float *f) {
    if constexpr (W == 1) return (T)f[0];
    else {
        vec<float, W> t;
#pragma unroll
        for (int i = 0; i < W; ++i) t[i] = f[i];
        return __builtin_convertvector(t, vec<T, W>);
    }
}

// sine and cosine of phi = pos * freq.  phi in quarter turns and the nearest whole number of them in 64 bits; what is left, |r| <= 1/2, fits 32
// bits.  Taylor sums on [-pi/4, pi/4]: first dropped terms x^11/11! = 1.8e-9 and x^12/12! = 1.1e-10, under half a step of a float near 1.
__device__ __forceinline__ float2 cos_sin(double pos, double freq) {
    const double t = pos * (freq * 0.63661977236758134308);  // 2 / pi
    const double k = rint(t);
    const float x = (float)((t - k) * 1.57079632679489661923);
    const int quarter = (int)((long long)k & 3);
    const float x2 = x * x;
    const float s = x + x * x2 * (-1.f / 6 + x2 * (1.f / 120 + x2 * (-1.f / 5040 + x2 * (1.f / 362880))));
    const float c = 1.f + x2 * (-0.5f + x2 * (1.f / 24 + x2 * (-1.f / 720 + x2 * (1.f / 40320 + x2 * (-1.f / 3628800)))));
    const float cc = (quarter & 1) ? s : c, ss = (quarter & 1) ? c : s;
    return make_float2((quarter == 1 || quarter == 2) ? -cc : cc, (quarter >= 2) ? -ss : ss);
}

__device__ __forceinline__ double load_pos(const RotaryParams &p, int b, int n, int a) {
    const long long o = b * p.pos_sb + n * p.pos_sn + a * p.pos_sa;
    if (p.pos_type == GD_POS_I32) return (double)static_cast<const int *>(p.pos)[o];
    if (p.pos_type == GD_POS_I64) return (double)static_cast<const long long *>(p.pos)[o];
    return (double)static_cast<const float *>(p.pos)[o];
}

// sum over the 2^lp_log2 lanes of a head: within 16 lanes by lane permutes in the adder's own operand, beyond by shuffles
template <int CTRL> __device__ __forceinline__ float permuted(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float head_sum(float v, int lp_log2) {
    if (lp_log2 > 0) v += permuted<0xb1>(v);   // lanes 1 0 3 2 of four
    if (lp_log2 > 1) v += permuted<0x4e>(v);   // 2 3 0 1
    if (lp_log2 > 2) v += permuted<0x141>(v);  // 7 .. 0 of eight: the other four
    if (lp_log2 > 3) v += permuted<0x140>(v);  // 15 .. 0 of sixteen: the other eight
    if (lp_log2 > 4) v += __shfl_xor(v, 16);
    if (lp_log2 > 5) v += __shfl_xor(v, 32);
    return v;
}

// v^-1/2 of the hardware (one step of float32), also where v is subnormal
__device__ __forceinline__ float inverse_root(float v) {
    const bool tiny = v < 1e-30f;
    return __builtin_amdgcn_rsqf(tiny ? v * 0x1p100f : v) * (tiny ? 0x1p50f : 1.f);
}

// NC: chunks of W pairs per lane (1 unless one head needs more than 64 lanes)
template <typename T, int W, int NC, bool HALVES, int MODE>
__global__ __launch_bounds__(MODE == ROT_NORM_BWD ? ROT_BWD_THREADS : 256) void rotary_kernel(const RotaryParams p, const int lp_log2, const int lp) {
    constexpr bool NORM = MODE != ROT_PLAIN, BWD = MODE == ROT_NORM_BWD;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6;
    const int pairs = (p.D + 1) / 2, R2 = p.R / 2;
    const int chunks = (pairs + W - 1) / W;  // W > 1: whole (the launcher's rule)
    float2 *table = reinterpret_cast<float2 *>(smem) + wave * (p.group * chunks * W);
    const int wpad = (p.D + 3) & ~3;
    float *weights = reinterpret_cast<float *>(smem + (size_t)waves * p.group * chunks * W * sizeof(float2));  // [2][wpad], float32
    const int row_step = 64 / lp;
    const int sub = lane / lp, in_head = lane - sub * lp;  // (sub == row_step: lanes left over where lp is no power of two)

    if constexpr (NORM) {
        for (int i = threadIdx.x; i < 2 * p.D; i += blockDim.x) {
            const int s = i >= p.D, e = s ? i - p.D : i;
            weights[s * wpad + e] = !p.w[s] ? 1.f : p.w_f32 ? static_cast<const float *>(p.w[s])[e] : (float)static_cast<const T *>(p.w[s])[e];
        }
        __syncthreads();
    }

    // this lane's channels: e0[c] .. + W - 1 and e1[c] .. + W - 1
    int e0[NC], e1[NC], ch[NC];
    bool on0[NC], on1[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        ch[c] = in_head + 64 * c;
        const int pr = ch[c] * W;
        if (!HALVES) { e0[c] = 2 * pr; e1[c] = 2 * pr + W; }
        else if (pr < R2) { e0[c] = pr; e1[c] = R2 + pr; }
        else { e0[c] = p.R + (pr - R2); e1[c] = p.R + (p.D - p.R + 1) / 2 + (pr - R2); }
        on0[c] = ch[c] < chunks && sub < row_step;
        on1[c] = on0[c] && e1[c] < p.D;  // an odd head has one channel without a partner (W == 1)
    }
    float dw[2][NC][2 * W];
    if constexpr (BWD)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < 2 * W; ++i) dw[s][c][i] = 0.f;
    const float inv_d = 1.f / (float)p.D;
    const int rows = p.heads[0] + p.heads[1];

    // An item: `group` tokens from (b, n) on, or a share of one token's heads; rows [i0, i1) of it, row i being head i % heads of token i / heads
    struct Item {
        int b, n, i0, i1;
    };
    const unsigned tokens = (unsigned)p.batch * (unsigned)p.tokens;
    auto locate = [&](unsigned id) __attribute__((always_inline)) {
        Item t;
        const unsigned q = id / (unsigned)p.items_per_token, token = q * p.group;
        t.b = (int)(token / (unsigned)p.tokens);
        t.n = (int)(token - (unsigned)t.b * p.tokens);
        t.i0 = (int)(id - q * p.items_per_token) * p.rows_per_item;
        t.i1 = p.group > 1 ? (int)min((unsigned)p.group, tokens - token) * rows : min(rows, t.i0 + p.rows_per_item);
        return t;
    };
    // token k of an item
    auto step_token = [&](const Item &t, int k, int &b, int &n) __attribute__((always_inline)) {
        b = t.b;
        n = t.n + k;
        while (n >= p.tokens) { n -= p.tokens; ++b; }
    };
    auto axis_of = [&](int pr) __attribute__((always_inline)) {
        int a = 0;
#pragma unroll
        for (int i = 0; i < ROT_MAX_AXES - 1; ++i) a += (i + 1 < p.n_axes && pr >= p.axis_end[i]);
        return a;
    };
    // The table holds P pairs of every token of the item.  A lane's first one keeps its frequency, and its position is read an item ahead
    const int P = chunks * W, entries = p.group * P;
    const int k0 = lane / P, pr0 = lane - k0 * P;
    const bool turns0 = lane < entries && pr0 < R2;
    const int axis0 = axis_of(pr0);
    const double freq0 = turns0 ? p.freq[pr0] : 0.0;
    auto pos_of = [&](const Item &t, int k, int axis) __attribute__((always_inline)) {
        int b, n;
        step_token(t, k, b, n);
        return b < p.batch ? load_pos(p, b, n, axis) : 0.0;  // (the last item may hold fewer tokens)
    };

    vec<T, W> v0[NC], v1[NC], g0[NC], g1[NC];
    auto at = [&](const HeadsView *hv, int b, int n, int r) __attribute__((always_inline)) {
        const int seg = r >= p.heads[0];
        const HeadsView &h = hv[seg];
        return static_cast<T *>(h.p) + (b * h.sb + n * h.sn + (r - (seg ? p.heads[0] : 0)) * h.sh);
    };
    auto load = [&](int b, int n, int r) __attribute__((always_inline)) {
        const T *src = at(p.x, b, n, r);
        const T *gsrc = BWD ? at(p.dy, b, n, r) : nullptr;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            v0[c] = vec<T, W>{}; v1[c] = vec<T, W>{};
            if (on0[c]) v0[c] = *reinterpret_cast<const vec<T, W> *>(src + e0[c]);
            if (on1[c]) v1[c] = *reinterpret_cast<const vec<T, W> *>(src + e1[c]);
            if constexpr (BWD) {
                g0[c] = vec<T, W>{}; g1[c] = vec<T, W>{};
                if (on0[c]) g0[c] = *reinterpret_cast<const vec<T, W> *>(gsrc + e0[c]);
                if (on1[c]) g1[c] = *reinterpret_cast<const vec<T, W> *>(gsrc + e1[c]);
            }
        }
    };
    float cs[NC][W], sn[NC][W];
    auto read_table = [&](const float2 *from) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const float2 t = from[on0[c] ? ch[c] * W + i : 0];
                cs[c][i] = t.x; sn[c][i] = t.y;
            }
    };
    float a[NC][2 * W], g[NC][2 * W];
    auto convert = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            to_f32<T, W>(v0[c], a[c]); to_f32<T, W>(v1[c], a[c] + W);
            if constexpr (BWD) { to_f32<T, W>(g0[c], g[c]); to_f32<T, W>(g1[c], g[c] + W); }
        }
    };
    // head r of token (b, n), in a and g; every lane of the wave takes part in the sums
    auto work = [&](int b, int n, int r, bool row_on) __attribute__((always_inline)) {
        const int seg = r >= p.heads[0];
        // index of a pair's two channels among the lane's 2W
        auto turn_pairs = [&](float *y, int c, auto all) __attribute__((always_inline)) {
            constexpr bool whole = decltype(all)::value;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const int ia = HALVES ? i : 2 * i, ib = HALVES ? W + i : 2 * i + 1;
                const float u = y[ia], v = y[ib];
                const bool turns = whole || ch[c] * W + i < R2;
                y[ia] = turns ? u * cs[c][i] - v * sn[c][i] : u;
                y[ib] = turns ? u * sn[c][i] + v * cs[c][i] : v;
            }
        };
        // Norms in 16-bit types take heads that turn whole apart, by one branch of the wave: with the choice in them too, the gradient of 16 + 4 heads of 128
        // channels took 81 us instead of 79.  The plain rotation (86 us with the branch, 82 without) and float32 (131 registers, 121) choose pair by pair.
        auto turn = [&](float *y, int c) __attribute__((always_inline)) {
            if (NORM && sizeof(T) == 2 && p.R == p.D) turn_pairs(y, c, std::true_type{});
            else turn_pairs(y, c, std::false_type{});
        };
        if constexpr (NORM) {
            float ss = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < 2 * W; ++i) ss += a[c][i] * a[c][i];
            float w[NC][2 * W];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const float *ws = weights + (seg ? wpad : 0);
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    w[c][i] = ws[on0[c] ? e0[c] + i : 0];
                    w[c][W + i] = ws[on1[c] ? e1[c] + i : 0];
                }
            }
            if constexpr (BWD) {
                float gx = 0.f;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    turn(g[c], c);
#pragma unroll
                    for (int i = 0; i < 2 * W; ++i) gx += g[c][i] * w[c][i] * a[c][i];
                }
                ss = head_sum(ss, lp_log2);
                gx = head_sum(gx, lp_log2);
                const float rho = inverse_root(ss * inv_d + p.eps);
                const float k = gx * inv_d * rho * rho;  // mean(g w xh) rho: xh mean(g w xh) = x k
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int i = 0; i < 2 * W; ++i) {
                        const float gi = row_on ? g[c][i] * (a[c][i] * rho) : 0.f;
                        dw[0][c][i] += seg ? 0.f : gi;
                        dw[1][c][i] += seg ? gi : 0.f;
                        a[c][i] = rho * (g[c][i] * w[c][i] - a[c][i] * k);
                    }
            } else {
                const float rho = inverse_root(head_sum(ss, lp_log2) * inv_d + p.eps);
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int i = 0; i < 2 * W; ++i) a[c][i] = a[c][i] * rho * w[c][i];
            }
        }
        if (row_on) {
            T *dst = at(p.out, b, n, r);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                if constexpr (!BWD) turn(a[c], c);
                if (on0[c]) *reinterpret_cast<vec<T, W> *>(dst + e0[c]) = from_f32<T, W>(a[c]);
                if (on1[c]) *reinterpret_cast<vec<T, W> *>(dst + e1[c]) = from_f32<T, W>(a[c] + W);
            }
        }
    };

    // the rows that are on their way: token k of their item, (b, n), head r
    int lk = 0, lb = 0, ln = 0, lr = 0;
    bool lon = false;
    auto fetch = [&](const Item &t, int base) __attribute__((always_inline)) {
        const int i = base + sub;
        lon = i < t.i1 && sub < row_step;
        lk = p.group > 1 ? i / rows : 0;
        lr = i - lk * rows;
        step_token(t, lon ? lk : 0, lb, ln);
        if (lon) load(lb, ln, lr);
    };

    unsigned id = blockIdx.x * waves + wave;
    const unsigned stride = gridDim.x * waves;
    Item cur{0, 0, 0, 0};
    double pos0 = 0.0;
    if (id < p.items) {
        cur = locate(id);
        if (turns0) pos0 = pos_of(cur, k0, axis0);
        fetch(cur, cur.i0);
    }
    while (id < p.items) {
        if (lane < entries) {
            float2 c = turns0 ? cos_sin(pos0, freq0) : make_float2(1.f, 0.f);
            c.y *= p.sign;
            table[lane] = c;
        }
        for (int e = lane + 64; e < entries; e += 64) {
            const int k = e / P, pr = e - k * P;
            float2 c = make_float2(1.f, 0.f);
            if (pr < R2) c = cos_sin(pos_of(cur, k, axis_of(pr)), p.freq[pr]);
            c.y *= p.sign;
            table[e] = c;
        }
        // the next item's positions and, behind this one's last rows, its first are on their way while this one is worked on
        const unsigned next_id = id + stride;
        Item next{0, 0, 0, 0};
        if (next_id < p.items) {
            next = locate(next_id);
            if (turns0) pos0 = pos_of(next, k0, axis0);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        for (int base = cur.i0; base < cur.i1; base += row_step) {
            const int b = lb, n = ln, r = lr;
            const bool on = lon;
            if (p.group > 1 || base == cur.i0) read_table(table + (on ? lk : 0) * P);
            convert();
            if (base + row_step < cur.i1) fetch(cur, base + row_step);
            else if (next_id < p.items) fetch(next, next.i0);
            work(b, n, r, on);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();  // the table is read before the next item overwrites it
        id = next_id;
        cur = next;
    }

    if constexpr (BWD) {
        // weight gradients: the wave's heads by shuffles, the workgroup's waves through LDS in wave order, one row of partials per
        // workgroup (summed in order by rotary_dw_kernel: the same bits every time)
        float *red = reinterpret_cast<float *>(smem);  // [waves][2][D]
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < 2 * W; ++i) {
                    float t = dw[s][c][i];
                    for (int m = lp; m < 64; m <<= 1) t += __shfl_xor(t, m);
                    const int e = i < W ? e0[c] + i : e1[c] + i - W;
                    if (sub == 0 && (i < W ? on0[c] : on1[c])) red[(wave * 2 + s) * p.D + e] = t;
                }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * p.D; i += blockDim.x) {
            float t = 0.f;
            for (int k = 0; k < waves; ++k) t += red[k * 2 * p.D + i];
            p.dw_part[(size_t)blockIdx.x * 2 * p.D + i] = t;
        }
    }
}

// dw[i] = sum over workgroups of their partial rows: 16 columns x 64 row groups per workgroup, added in a fixed order
template <typename T>
__global__ __launch_bounds__(1024) void rotary_dw_kernel(const float *part, int blocks, int D, void *dw0, void *dw1, int w_f32) {
    __shared__ float red[64][17];
    const int col = blockIdx.x * 16 + (threadIdx.x & 15), grp = threadIdx.x >> 4;
    float t = 0.f;
    if (col < 2 * D) {
        static_assert(ROT_BWD_BLOCKS % 64 == 0, "");
        float v[ROT_BWD_BLOCKS / 64];  // all on their way at once
#pragma unroll
        for (int k = 0; k < ROT_BWD_BLOCKS / 64; ++k) v[k] = grp + 64 * k < blocks ? part[(size_t)(grp + 64 * k) * 2 * D + col] : 0.f;
#pragma unroll
        for (int k = 0; k < ROT_BWD_BLOCKS / 64; ++k) t += v[k];
    }
    red[grp][threadIdx.x & 15] = t;
    __syncthreads();
    if (grp == 0 && col < 2 * D) {
        double sum = 0.0;
        for (int k = 0; k < 64; ++k) sum += (double)red[k][threadIdx.x];
        void *dst = col < D ? dw0 : dw1;
        const int e = col < D ? col : col - D;
        if (!dst) return;
        if (w_f32) static_cast<float *>(dst)[e] = (float)sum;
        else static_cast<T *>(dst)[e] = (T)(float)sum;
    }
}

template <typename T, int W, int NC, bool HALVES>
int launch_mode(const RotaryParams &p, RotaryMode mode, int lp_log2, int lp, int blocks, void *dw0, void *dw1, hipStream_t s) {
    const int chunks = ((p.D + 1) / 2 + W - 1) / W;
    const int waves = mode == ROT_NORM_BWD ? ROT_BWD_THREADS / 64 : 4;
    size_t lds = (size_t)waves * p.group * chunks * W * sizeof(float2) + (mode == ROT_PLAIN ? 0 : 2 * ((p.D + 3) & ~3) * sizeof(float));
    switch (mode) {
        case ROT_PLAIN: rotary_kernel<T, W, NC, HALVES, ROT_PLAIN><<<blocks, 256, lds, s>>>(p, lp_log2, lp); break;
        case ROT_NORM: rotary_kernel<T, W, NC, HALVES, ROT_NORM><<<blocks, 256, lds, s>>>(p, lp_log2, lp); break;
        case ROT_NORM_BWD:
            if (lds < (size_t)waves * 2 * p.D * sizeof(float)) lds = (size_t)waves * 2 * p.D * sizeof(float);
            if constexpr (W * sizeof(T) <= 8 || sizeof(T) == 4) rotary_kernel<T, W, NC, HALVES, ROT_NORM_BWD><<<blocks, ROT_BWD_THREADS, lds, s>>>(p, lp_log2, lp);
            GD_HIP(hipGetLastError());
            rotary_dw_kernel<T><<<(2 * p.D + 15) / 16, 1024, 0, s>>>(p.dw_part, blocks, p.D, dw0, dw1, p.w_f32);
            break;
    }
    GD_HIP(hipGetLastError());
    return 0;
}

template <typename T, int W, int NC>
int launch_pairs(const RotaryParams &p, RotaryMode mode, int lp_log2, int lp, int blocks, void *dw0, void *dw1, hipStream_t s) {
    return p.halves ? launch_mode<T, W, NC, true>(p, mode, lp_log2, lp, blocks, dw0, dw1, s)
                    : launch_mode<T, W, NC, false>(p, mode, lp_log2, lp, blocks, dw0, dw1, s);
}

// vectors of W channels: every address a multiple of their size, the halves' pairs and pass-through channels whole vectors
bool vec_ok(const RotaryParams &p, int W, int elem, bool bwd) {
    const size_t bytes = (size_t)W * elem;
    if (p.D % (2 * W) || (p.halves && p.R % (2 * W))) return false;  // (2i, 2i + 1) pairs may end inside a lane's: the rest pass through
    auto ok = [&](const HeadsView &h) {
        return (size_t)h.p % bytes == 0 && h.sb % W == 0 && h.sn % W == 0 && h.sh % W == 0;
    };
    for (int s = 0; s < 2; ++s)
        if (p.heads[s] && !(ok(p.x[s]) && ok(p.out[s]) && (!bwd || ok(p.dy[s])))) return false;
    return true;
}

template <typename T>
int launch_type(RotaryParams &p, RotaryMode mode, void *dw0, void *dw1, hipStream_t s) {
    constexpr int WV = 16 / sizeof(T);
    const bool bwd = mode == ROT_NORM_BWD;
    const bool narrow = sizeof(T) == 2 && bwd;  // fewer registers: 71 us against 83 for 16 + 4 heads of 128 channels at 16382 tokens
    const int W = !narrow && vec_ok(p, WV, sizeof(T), bwd) ? WV : vec_ok(p, WV / 2, sizeof(T), bwd) ? WV / 2 : 1;
    const int chunks = ((p.D + 1) / 2 + W - 1) / W;
    int lp_log2 = 0;
    while (lp_log2 < 6 && (1 << lp_log2) < chunks) ++lp_log2;
    const int lp = mode == ROT_PLAIN && chunks < 64 ? chunks : 1 << lp_log2;  // lanes of a head: without sums over them, no more than it has chunks
    const int rows = p.heads[0] + p.heads[1], row_step = 64 / lp;
    const long long tokens = (long long)p.batch * p.tokens;
    if (tokens == 0) {
        if (bwd) rotary_dw_kernel<T><<<(2 * p.D + 15) / 16, 1024, 0, s>>>(p.dw_part, 0, p.D, dw0, dw1, p.w_f32);
        GD_HIP(hipGetLastError());
        return 0;
    }
    // a wave takes whole tokens once they fill the chip (16 waves per CU), else a share of a token's heads, at least one step of them
    const int max_blocks = bwd ? ROT_BWD_BLOCKS : device_cus() * 16;
    const long long want = (long long)device_cus() * 16;
    long long shares = tokens >= want ? 1 : (want + tokens - 1) / tokens;
    const int steps = (rows + row_step - 1) / row_step;
    if (shares > steps) shares = steps;
    p.rows_per_item = (int)((steps + shares - 1) / shares) * row_step;
    p.items_per_token = (rows + p.rows_per_item - 1) / p.rows_per_item;
    p.items = (unsigned)(tokens * p.items_per_token);  // < 2^31: shares are taken only where tokens are few
    // A step or a few a token are mostly the way from its position to its angles: an item of several tokens then, until it is four steps of the wave (and
    // its table 256 pairs), as long as there are items enough (6 x 13278 tokens of one 64-channel head in fp16: 18 us
    // instead of 50; 13 x 10525 of three of 16 in float32 16 instead of 69)
    const int P = chunks * W;
    p.group = 1;
    if (shares == 1 && rows <= 4 * row_step) {
        long long group = (4LL * row_step + rows - 1) / rows;
        if (group > 256 / P) group = 256 / P;
        if (group > tokens / want) group = tokens / want;
        if (group > 1) {
            p.group = (int)group;
            p.items = (unsigned)((tokens + group - 1) / group);
            p.items_per_token = 1;
        }
    }
    const unsigned per_block = bwd ? ROT_BWD_THREADS / 64 : 4;
    unsigned blocks = (p.items + per_block - 1) / per_block;
    if (blocks > (unsigned)max_blocks) blocks = max_blocks;
    // (a head of up to 512 channels: at most 64 chunks of 16 bytes or of 8 in a 16-bit type, 128 of 8 bytes in float32, 256 of one pair)
    if (W == WV) return launch_pairs<T, WV, 1>(p, mode, lp_log2, lp, (int)blocks, dw0, dw1, s);
    if (W > 1 && chunks <= 64) return launch_pairs<T, WV / 2, 1>(p, mode, lp_log2, lp, (int)blocks, dw0, dw1, s);
    if constexpr (sizeof(T) == 4)
        if (W > 1) return launch_pairs<T, WV / 2, 2>(p, mode, lp_log2, lp, (int)blocks, dw0, dw1, s);
    if (chunks <= 64) return launch_pairs<T, 1, 1>(p, mode, lp_log2, lp, (int)blocks, dw0, dw1, s);
    if (chunks <= 128) return launch_pairs<T, 1, 2>(p, mode, lp_log2, lp, (int)blocks, dw0, dw1, s);
    return launch_pairs<T, 1, 4>(p, mode, lp_log2, lp, (int)blocks, dw0, dw1, s);
}

}  // namespace

int launch_rotary(RotaryParams p, int dtype, RotaryMode mode, void *dw0, void *dw1, hipStream_t s) {
    switch (dtype) {
        case GD_F32: return launch_type<float>(p, mode, dw0, dw1, s);
        case GD_BF16: return launch_type<__bf16>(p, mode, dw0, dw1, s);
        case GD_F16: return launch_type<_Float16>(p, mode, dw0, dw1, s);
    }
    GD_CHECK(false, "unknown element type %d", dtype);
}

}  // namespace gd
