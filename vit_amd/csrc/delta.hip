// Gated delta rule in its chunked (matrix-pipe) form, forward and backward, and for single tokens.
//
// The recurrence per (batch, head), state S [dv, dk] (dk = dv = hd), decay a_t, write strength b_t:
//     S_t = a_t S_{t-1} (I - b_t k_t k_t^T) + b_t v_t k_t^T,        o_t = S_t q_t.
// With M = S^T the update is rank 1, M_t = a_t M_{t-1} + k_t u_t^T, u_t = b_t (v_t - a_t M_{t-1}^T k_t).  For a chunk of
// C = 64 tokens that starts at state M, with g_ij = a_{j+1} ... a_i (decay from token j to token i), g_i = a_1 ... a_i,
// rows of K, Q, V, U = the chunk's tokens:
//     (I + A) U = diag(b) (V - diag(g) K M),   A_ij = b_i g_ij k_i.k_j  (i > j),      T = (I + A)^-1
//     O   = diag(g) Q M + P U,                 P_ij = g_ij q_i.k_j      (i >= j)
//     M_C = g_C M + K^T diag(g_C.) U.
// Everything but the two products with M and the last line is independent between chunks.  Three launches:
//     delta_prep_kernel   per chunk: decays, K K^T, Q K^T, T, P                       (parallel over B H L/64)
//     delta_scan_kernel   per (head, 16 columns of M): chunk after chunk               (parallel over B H hd/16 waves)
// and for the gradient, with G = dL/dM at the chunk's end, X = dO M^T, Y = R M^T, Z = U G^T:
//     dU = P^T dO + diag(g_C.) K G,   R = T^T dU,   dV = diag(b) R,   G <- g_C G + Q^T diag(g) dO - K^T diag(b g) R
//     dQ = diag(g) X + (dP o g) K,    dK = diag(g_C.) Z - diag(b g) Y + (dP o g)^T Q + (E + E^T) K
//     dP = dO U^T,  dA = -R U^T,  E_ij = b_i g_ij dA_ij
//     db_i = sum_j dA_ij g_ij k_i.k_j + R_i.v_i - g_i k_i.Y_i
//     da_t = sum_{i >= t} g_it w_t[i],  w_{t+1}[i] = a_t w_t[i] + d(g_it),  w_1[i] = d(g_i)
// (the last line needs no division by a decay, so decays of zero are ordinary numbers; the decays themselves are running
// products, never differences of logarithms).  delta_scan_kernel runs once more for U and the chunks' states, then
// delta_rscan_kernel backwards, then delta_grad_kernel per chunk.
//
// All products run on the f32 matrix instruction (16x16x4): its operand for contraction index 4g+r of lane group g is
// register r of an accumulator tile, so results (V - K M, U, M, G) feed the next product from where they lie, and a
// left operand is one 16-byte read of a row.
#include "common.h"

namespace {

constexpr int DC = 64;                    // tokens per chunk
constexpr int TRI = 10;                   // 16x16 blocks of a lower triangle of 64x64
constexpr int FRAG = 256;                 // floats of one 16x16 operand block: lane l holds row l%16, columns 4(l/16)..+3
constexpr int SQ = DC + 4;                // row stride of 64x64 matrices in LDS

VA_DEVINL f32x4_t mfma_f32(float a, float b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
// index of block (it, jt), it >= jt, of a lower triangle
__host__ __device__ constexpr int tri(int it, int jt) { return it * (it + 1) / 2 + jt; }

VA_DEVINL f32x4_t widen4(f32x4_t v) { return v; }
VA_DEVINL f32x4_t widen4(u32x2_t p) {
    return (f32x4_t){__uint_as_float(p[0] << 16), __uint_as_float(p[0] & 0xffff0000u), __uint_as_float(p[1] << 16),
                     __uint_as_float(p[1] & 0xffff0000u)};
}
template <typename T> struct elem;
template <> struct elem<float> {
    typedef f32x4_t raw4;
    static VA_DEVINL float get(const float* p) { return *p; }
    static VA_DEVINL void put(float* p, float x) { *p = x; }
};
template <> struct elem<bf16_t> {
    typedef u32x2_t raw4;
    static VA_DEVINL float get(const bf16_t* p) { return bf16_to_f32(*p); }
    static VA_DEVINL void put(bf16_t* p, float x) { *p = f32_to_bf16(x); }      // the output's own type: one rounding
};
template <typename T> VA_DEVINL f32x4_t load4(const T* p) { return widen4(*(const typename elem<T>::raw4*)p); }

// where a token's row of one head lies: rows of `ld` elements, heads side by side
struct Rows {
    int64_t ld;
    VA_DEVINL int64_t at(int64_t b, int64_t L, int64_t t, int64_t h, int64_t hd) const { return (b * L + t) * ld + h * hd; }
};

// Decays of a chunk.  a[] in LDS (1 behind the sequence's end).  Lane i of one wave walks the tokens back from i:
// gt[j][i] = a_{j+1} ... a_i for j <= i, 0 above.
VA_DEVINL void chunk_decays(const float* a, float (*gt)[SQ], int lane) {
    float p = 0.f;
    for (int j = DC - 1; j >= 0; --j) {
        p = j == lane ? 1.0f : j < lane ? p * a[j + 1] : 0.f;      // j < lane: j + 1 is inside the chunk
        gt[j][lane] = p;
    }
}
// lane i: a_0 ... a_i
VA_DEVINL float chunk_prefix(const float* a, int lane) {
    float p = 1.f, mine = 1.f;
    for (int j = 0; j < DC; ++j) {
        p *= a[j];
        mine = j == lane ? p : mine;
    }
    return mine;
}

template <int HD, typename T, int THREADS>
VA_DEVINL void rows_to_lds(const T* __restrict__ src, int64_t first, int64_t ld, int rows_left, float (*dst)[HD + 4], int tid) {
    constexpr int N = DC * HD / 4 / THREADS;
#pragma unroll
    for (int p = 0; p < N; ++p) {
        const int idx = p * THREADS + tid, row = idx / (HD / 4), c = (idx % (HD / 4)) * 4;
        f32x4_t v = {0.f, 0.f, 0.f, 0.f};
        if (row < rows_left) v = load4(src + first + (int64_t)row * ld + c);
        *(f32x4_t*)&dst[row][c] = v;
    }
}

// ---------------------------------------------------------------------------------------------------------------
// One workgroup of four waves per chunk.  Tiles are formed transposed, D[j][i] = k_j.x_i, so that a lane holds row i and
// four consecutive j: the operand order in which T and P are kept.  GRAD: T, T^T and P^T for the gradient's scans,
// otherwise T and P.
template <int HD, typename T, bool GRAD>
__global__ __launch_bounds__(256) void delta_prep_kernel(const T* __restrict__ Q, const T* __restrict__ K, Rows rq, Rows rk,
                                                         const float* __restrict__ ALPHA, const float* __restrict__ BETA,
                                                         float* __restrict__ TF, float* __restrict__ TT, float* __restrict__ PF,
                                                         float* __restrict__ GAM, int L, int H, int NC) {
    extern __shared__ __align__(16) char lds[];
    float(*ks)[HD + 4] = (float(*)[HD + 4])lds;
    float(*qs)[HD + 4] = ks + DC;
    float(*gt)[SQ] = (float(*)[SQ])(qs + DC);
    float(*am)[SQ] = gt + DC;                     // A, then T
    float(*dg)[20] = (float(*)[20])(am + DC);     // inverses of the four diagonal blocks of I + A
    float* sa = (float*)(dg + DC);
    float* sb = sa + DC;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, g4 = (lane >> 4) * 4;
    const int64_t ci = blockIdx.x;
    const int64_t bh = ci / NC;
    const int c = (int)(ci % NC), t0 = c * DC, left = L - t0 < DC ? L - t0 : DC;
    const int64_t b = bh / H, h = bh % H;
    rows_to_lds<HD, T, 256>(K, rk.at(b, L, t0, h, HD), rk.ld, left, ks, tid);
    rows_to_lds<HD, T, 256>(Q, rq.at(b, L, t0, h, HD), rq.ld, left, qs, tid);
    if (tid < DC) {
        const int64_t at = (b * L + t0 + tid) * H + h;
        sa[tid] = tid < left ? ALPHA[at] : 1.0f;
        sb[tid] = tid < left ? BETA[at] : 0.0f;
    }
    __syncthreads();
    if (wave == 0) chunk_decays(sa, gt, lane);
    if (wave == 1) GAM[ci * 2 * DC + lane] = chunk_prefix(sa, lane);
    f32x4_t acc[5];                               // 20 tiles (K K^T and Q K^T), five to a wave
#pragma unroll
    for (int s = 0; s < 5; ++s) {
        const int x = wave + 4 * s, tile = x % TRI;
        const int it = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3, jt = tile - tri(it, 0);
        const bool qk = x >= TRI;
        const float* rj = ks[16 * jt + m] + g4;
        const float* ri = (qk ? qs : ks)[16 * it + m] + g4;
        // P^T for the gradient: lane holds row j and four consecutive i
        const float* ra = qk && GRAD ? ri : rj;
        const float* rb = qk && GRAD ? rj : ri;
        f32x4_t d = {0.f, 0.f, 0.f, 0.f}, e = d;
#pragma unroll
        for (int u = 0; u < HD / 16; ++u) {
            const f32x4_t x4 = *(const f32x4_t*)(ra + 16 * u), y4 = *(const f32x4_t*)(rb + 16 * u);
            d = mfma_f32(x4[0], y4[0], d);
            e = mfma_f32(x4[1], y4[1], e);
            d = mfma_f32(x4[2], y4[2], d);
            e = mfma_f32(x4[3], y4[3], e);
        }
        acc[s] = d + e;
    }
    __syncthreads();                              // the decays are there
    if (wave == 2) GAM[ci * 2 * DC + DC + lane] = gt[lane][DC - 1];
#pragma unroll
    for (int s = 0; s < 5; ++s) {
        const int x = wave + 4 * s, tile = x % TRI;
        const int it = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3, jt = tile - tri(it, 0);
        f32x4_t v = acc[s];
        if (x < TRI) {
            const int i = 16 * it + m;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = 16 * jt + g4 + r;
                v[r] = i > j ? v[r] * sb[i] * gt[j][i] : 0.f;
            }
            *(f32x4_t*)&am[i][16 * jt + g4] = v;
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = GRAD ? 16 * it + g4 + r : 16 * it + m, j = GRAD ? 16 * jt + m : 16 * jt + g4 + r;
                v[r] *= gt[j][i];                 // 0 above the diagonal
            }
            *(f32x4_t*)(PF + (ci * TRI + tile) * FRAG + lane * 4) = v;
        }
    }
    __syncthreads();
    // inverse of a diagonal block by forward substitution, lane = column
    {
        const float(*ab)[SQ] = am + 16 * wave;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float s = i == m ? 1.f : 0.f;
#pragma unroll
            for (int j = 0; j < i; ++j) s = fmaf(-ab[i][16 * wave + j], x[j], s);
            x[i] = s;
        }
        if (lane < 16) {
#pragma unroll
            for (int i = 0; i < 16; ++i) dg[16 * wave + i][m] = x[i];
        }
    }
    __syncthreads();
    // the blocks below, by block columns: X_ij = -D_i sum_{j <= k < i} A_ik X_kj; a block column per wave, in registers
    f32x4_t xb[4];
    {
        const int jt = wave;
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            if (it < jt) continue;
            if (it == jt) {
#pragma unroll
                for (int r = 0; r < 4; ++r) xb[it][r] = dg[16 * it + g4 + r][m];
                continue;
            }
            f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kt = 0; kt < it; ++kt) {
                if (kt < jt) continue;
                const f32x4_t a4 = *(const f32x4_t*)&am[16 * it + m][16 * kt + g4];
#pragma unroll
                for (int r = 0; r < 4; ++r) s = mfma_f32(a4[r], xb[kt][r], s);
            }
            const f32x4_t d4 = *(const f32x4_t*)&dg[16 * it + m][g4];
            f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int r = 0; r < 4; ++r) o = mfma_f32(-d4[r], s[r], o);
            xb[it] = o;
        }
    }
    __syncthreads();
#pragma unroll
    for (int it = 0; it < 4; ++it) {
        if (it < wave) continue;
        if (GRAD) *(f32x4_t*)(TT + (ci * TRI + tri(it, wave)) * FRAG + lane * 4) = xb[it];
#pragma unroll
        for (int r = 0; r < 4; ++r) am[16 * it + g4 + r][16 * wave + m] = xb[it][r];
    }
    __syncthreads();
    for (int x = wave; x < TRI; x += 4) {
        const int it = x < 1 ? 0 : x < 3 ? 1 : x < 6 ? 2 : 3, jt = x - tri(it, 0);
        *(f32x4_t*)(TF + (ci * TRI + x) * FRAG + lane * 4) = *(const f32x4_t*)&am[16 * it + m][16 * jt + g4];
    }
}

// acc[it] += X (64 rows, HD columns, in LDS) * B, B = accumulator tiles
template <int HD>
VA_DEVINL void rows_times_tiles(const float (*x)[HD + 4], const f32x4_t* bt, f32x4_t* acc, int m, int g4) {
#pragma unroll
    for (int u = 0; u < HD / 16; ++u) {
        f32x4_t a[4];
#pragma unroll
        for (int it = 0; it < 4; ++it) a[it] = *(const f32x4_t*)&x[16 * it + m][16 * u + g4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int it = 0; it < 4; ++it) acc[it] = mfma_f32(a[it][r], bt[u][r], acc[it]);
    }
}
// acc[u] += X^T (HD rows, 64 columns) * B
template <int HD>
VA_DEVINL void columns_times_tiles(const float (*x)[HD + 4], const f32x4_t* bt, f32x4_t* acc, int m, int g4) {
#pragma unroll
    for (int jt = 0; jt < 4; ++jt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int u = 0; u < HD / 16; ++u) acc[u] = mfma_f32(x[16 * jt + g4 + r][16 * u + m], bt[jt][r], acc[u]);
}

// ---------------------------------------------------------------------------------------------------------------
// The sequential part.  A wave owns 16 columns (values of the head) of the state for the whole sequence: M in HD/16
// accumulator tiles; W waves share a chunk's K and Q through LDS.  The next chunk's rows are requested before the
// current one computes.  OUT: writes o.  SAVE: writes U and every chunk's starting state (rows of S) for the gradient.
template <int HD, typename T, int W, bool OUT, bool SAVE>
__global__ __launch_bounds__(64 * W) void delta_scan_kernel(const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V,
                                                            Rows rq, Rows rk, Rows rv, const float* __restrict__ BETA,
                                                            const float* __restrict__ TF, const float* __restrict__ PF,
                                                            const float* __restrict__ GAM, const float* __restrict__ STATE_IN,
                                                            T* __restrict__ O, float* __restrict__ STATE_OUT,
                                                            float* __restrict__ US, float* __restrict__ MS, int L, int H, int NC) {
    extern __shared__ __align__(16) char lds[];
    float(*ks)[HD + 4] = (float(*)[HD + 4])lds;
    float(*qs)[HD + 4] = ks + DC;
    float* sb = (float*)(ks + (OUT ? 2 : 1) * DC);
    float* sg = sb + DC;
    float* se = sg + DC;
    constexpr int GROUPS = HD / 16 / W, N = DC * HD / 4 / (64 * W);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, g4 = (lane >> 4) * 4;
    const int wid = xcd_remap(blockIdx.x, gridDim.x);
    const int64_t bh = wid / GROUPS, b = bh / H, h = bh % H;
    const int v = ((wid % GROUPS) * W + wave) * 16 + m;
    const int64_t qrow = rq.at(b, L, 0, h, HD), krow = rk.at(b, L, 0, h, HD), vrow = rv.at(b, L, 0, h, HD);
    typedef typename elem<T>::raw4 raw4;
    raw4 kn[N], qn[N];
    float bn = 0.f, gn = 0.f, en = 0.f;
    auto request = [&](int c) {
        const int left = L - c * DC;
#pragma unroll
        for (int p = 0; p < N; ++p) {
            const int idx = p * 64 * W + tid, row = idx / (HD / 4), col = (idx % (HD / 4)) * 4;
            const int64_t t = (int64_t)c * DC + row;
            kn[p] = raw4{};
            if (row < left) kn[p] = *(const raw4*)(K + krow + t * rk.ld + col);
            if (OUT) {
                qn[p] = raw4{};
                if (row < left) qn[p] = *(const raw4*)(Q + qrow + t * rq.ld + col);
            }
        }
        if (tid < DC) {
            bn = tid < left ? BETA[(b * L + (int64_t)c * DC + tid) * H + h] : 0.f;
            gn = GAM[(bh * NC + c) * 2 * DC + tid];
            en = GAM[(bh * NC + c) * 2 * DC + DC + tid];
        }
    };
    f32x4_t M[HD / 16];
#pragma unroll
    for (int u = 0; u < HD / 16; ++u) {
        M[u] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
        if (STATE_IN != nullptr) M[u] = *(const f32x4_t*)(STATE_IN + (bh * HD + v) * HD + 16 * u + g4);
    }
    request(0);
    for (int c = 0; c < NC; ++c) {
        const int t0 = c * DC, left = L - t0;
        const int64_t ci = bh * NC + c;
        __syncthreads();                          // everybody is done with the chunk before
#pragma unroll
        for (int p = 0; p < N; ++p) {
            const int idx = p * 64 * W + tid, row = idx / (HD / 4), col = (idx % (HD / 4)) * 4;
            *(f32x4_t*)&ks[row][col] = widen4(kn[p]);
            if (OUT) *(f32x4_t*)&qs[row][col] = widen4(qn[p]);
        }
        if (tid < DC) sb[tid] = bn, sg[tid] = gn, se[tid] = en;
        __syncthreads();
        // this chunk's v column (C order) and T, requested ahead of their use
        f32x4_t vv[4], tf[TRI];
#pragma unroll
        for (int it = 0; it < 4; ++it)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * it + g4 + r;
                vv[it][r] = i < left ? elem<T>::get(V + vrow + (int64_t)(t0 + i) * rv.ld + v) : 0.f;
            }
#pragma unroll
        for (int x = 0; x < TRI; ++x) tf[x] = *(const f32x4_t*)(TF + (ci * TRI + x) * FRAG + lane * 4);
        if (c + 1 < NC) request(c + 1);
        if (SAVE) {
#pragma unroll
            for (int u = 0; u < HD / 16; ++u) *(f32x4_t*)(MS + (ci * HD + v) * HD + 16 * u + g4) = M[u];
        }
        f32x4_t rhs[4], U[4];
#pragma unroll
        for (int it = 0; it < 4; ++it) rhs[it] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
        rows_times_tiles<HD>(ks, M, rhs, m, g4);
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            const f32x4_t b4 = *(const f32x4_t*)(sb + 16 * it + g4), gg = *(const f32x4_t*)(sg + 16 * it + g4);
#pragma unroll
            for (int r = 0; r < 4; ++r) rhs[it][r] = b4[r] * (vv[it][r] - gg[r] * rhs[it][r]);
            U[it] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int jt = 0; jt < 4; ++jt)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int it = jt; it < 4; ++it) U[it] = mfma_f32(tf[tri(it, jt)][r], rhs[jt][r], U[it]);
        if (SAVE) {
#pragma unroll
            for (int it = 0; it < 4; ++it)
#pragma unroll
                for (int r = 0; r < 4; ++r) US[(ci * DC + 16 * it + g4 + r) * HD + v] = U[it][r];
        }
        if (OUT) {
            f32x4_t pf[TRI], o[4];
#pragma unroll
            for (int x = 0; x < TRI; ++x) pf[x] = *(const f32x4_t*)(PF + (ci * TRI + x) * FRAG + lane * 4);
#pragma unroll
            for (int it = 0; it < 4; ++it) o[it] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
            rows_times_tiles<HD>(qs, M, o, m, g4);
#pragma unroll
            for (int it = 0; it < 4; ++it) o[it] *= *(const f32x4_t*)(sg + 16 * it + g4);
#pragma unroll
            for (int jt = 0; jt < 4; ++jt)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int it = jt; it < 4; ++it) o[it] = mfma_f32(pf[tri(it, jt)][r], U[jt][r], o[it]);
#pragma unroll
            for (int it = 0; it < 4; ++it)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * it + g4 + r;
                    if (i < left) elem<T>::put(O + ((b * L + t0 + i) * H + h) * HD + v, o[it][r]);
                }
        }
        const float gc = sg[DC - 1];
#pragma unroll
        for (int u = 0; u < HD / 16; ++u) M[u] *= gc;
#pragma unroll
        for (int it = 0; it < 4; ++it) U[it] *= *(const f32x4_t*)(se + 16 * it + g4);
        columns_times_tiles<HD>(ks, U, M, m, g4);
    }
    if (STATE_OUT != nullptr) {
#pragma unroll
        for (int u = 0; u < HD / 16; ++u) *(f32x4_t*)(STATE_OUT + (bh * HD + v) * HD + 16 * u + g4) = M[u];
    }
}

// ---------------------------------------------------------------------------------------------------------------
// The same walk backwards for G = dL/dM: writes every chunk's G (at its end, rows of dS), R and dv.
template <int HD, typename T, int W>
__global__ __launch_bounds__(64 * W) void delta_rscan_kernel(const T* __restrict__ Q, const T* __restrict__ K, Rows rq, Rows rk,
                                                             const T* __restrict__ DO, const float* __restrict__ BETA,
                                                             const float* __restrict__ TT, const float* __restrict__ PT,
                                                             const float* __restrict__ GAM, const float* __restrict__ DSTATE,
                                                             T* __restrict__ DV, float* __restrict__ DSTATE_IN,
                                                             float* __restrict__ RS, float* __restrict__ GS, int L, int H, int NC) {
    extern __shared__ __align__(16) char lds[];
    float(*ks)[HD + 4] = (float(*)[HD + 4])lds;
    float(*qs)[HD + 4] = ks + DC;
    float* sb = (float*)(qs + DC);
    float* sg = sb + DC;
    float* se = sg + DC;
    constexpr int GROUPS = HD / 16 / W, N = DC * HD / 4 / (64 * W);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, g4 = (lane >> 4) * 4;
    const int wid = xcd_remap(blockIdx.x, gridDim.x);
    const int64_t bh = wid / GROUPS, b = bh / H, h = bh % H;
    const int v = ((wid % GROUPS) * W + wave) * 16 + m;
    const int64_t qrow = rq.at(b, L, 0, h, HD), krow = rk.at(b, L, 0, h, HD);
    typedef typename elem<T>::raw4 raw4;
    raw4 kn[N], qn[N];
    float bn = 0.f, gn = 0.f, en = 0.f;
    auto request = [&](int c) {
        const int left = L - c * DC;
#pragma unroll
        for (int p = 0; p < N; ++p) {
            const int idx = p * 64 * W + tid, row = idx / (HD / 4), col = (idx % (HD / 4)) * 4;
            const int64_t t = (int64_t)c * DC + row;
            kn[p] = raw4{};
            qn[p] = raw4{};
            if (row < left) {
                kn[p] = *(const raw4*)(K + krow + t * rk.ld + col);
                qn[p] = *(const raw4*)(Q + qrow + t * rq.ld + col);
            }
        }
        if (tid < DC) {
            bn = tid < left ? BETA[(b * L + (int64_t)c * DC + tid) * H + h] : 0.f;
            gn = GAM[(bh * NC + c) * 2 * DC + tid];
            en = GAM[(bh * NC + c) * 2 * DC + DC + tid];
        }
    };
    f32x4_t G[HD / 16];
#pragma unroll
    for (int u = 0; u < HD / 16; ++u) {
        G[u] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
        if (DSTATE != nullptr) G[u] = *(const f32x4_t*)(DSTATE + (bh * HD + v) * HD + 16 * u + g4);
    }
    request(NC - 1);
    for (int c = NC - 1; c >= 0; --c) {
        const int t0 = c * DC, left = L - t0;
        const int64_t ci = bh * NC + c;
        __syncthreads();
#pragma unroll
        for (int p = 0; p < N; ++p) {
            const int idx = p * 64 * W + tid, row = idx / (HD / 4), col = (idx % (HD / 4)) * 4;
            *(f32x4_t*)&ks[row][col] = widen4(kn[p]);
            *(f32x4_t*)&qs[row][col] = widen4(qn[p]);
        }
        if (tid < DC) sb[tid] = bn, sg[tid] = gn, se[tid] = en;
        __syncthreads();
        f32x4_t dov[4], pt[TRI], tt[TRI];
#pragma unroll
        for (int it = 0; it < 4; ++it)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * it + g4 + r;
                dov[it][r] = i < left ? elem<T>::get(DO + ((b * L + t0 + i) * H + h) * HD + v) : 0.f;
            }
#pragma unroll
        for (int x = 0; x < TRI; ++x) {
            pt[x] = *(const f32x4_t*)(PT + (ci * TRI + x) * FRAG + lane * 4);
            tt[x] = *(const f32x4_t*)(TT + (ci * TRI + x) * FRAG + lane * 4);
        }
        if (c > 0) request(c - 1);
#pragma unroll
        for (int u = 0; u < HD / 16; ++u) *(f32x4_t*)(GS + (ci * HD + v) * HD + 16 * u + g4) = G[u];
        f32x4_t du[4], R[4];
#pragma unroll
        for (int it = 0; it < 4; ++it) du[it] = R[it] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
        rows_times_tiles<HD>(ks, G, du, m, g4);
#pragma unroll
        for (int it = 0; it < 4; ++it) du[it] *= *(const f32x4_t*)(se + 16 * it + g4);
#pragma unroll
        for (int it = 0; it < 4; ++it)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int jt = 0; jt <= it; ++jt) du[jt] = mfma_f32(pt[tri(it, jt)][r], dov[it][r], du[jt]);
#pragma unroll
        for (int it = 0; it < 4; ++it)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int jt = 0; jt <= it; ++jt) R[jt] = mfma_f32(tt[tri(it, jt)][r], du[it][r], R[jt]);
        const float gc = sg[DC - 1];
#pragma unroll
        for (int u = 0; u < HD / 16; ++u) G[u] *= gc;
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            const f32x4_t b4 = *(const f32x4_t*)(sb + 16 * it + g4), gg = *(const f32x4_t*)(sg + 16 * it + g4);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 16 * it + g4 + r;
                RS[(ci * DC + i) * HD + v] = R[it][r];
                const float dv = b4[r] * R[it][r];
                if (i < left) elem<T>::put(DV + ((b * L + t0 + i) * H + h) * HD + v, dv);
                dov[it][r] *= gg[r];
                R[it][r] = -gg[r] * dv;
            }
        }
        columns_times_tiles<HD>(qs, dov, G, m, g4);
        columns_times_tiles<HD>(ks, R, G, m, g4);
    }
    if (DSTATE_IN != nullptr) {
#pragma unroll
        for (int u = 0; u < HD / 16; ++u) *(f32x4_t*)(DSTATE_IN + (bh * HD + v) * HD + 16 * u + g4) = G[u];
    }
}

// ---------------------------------------------------------------------------------------------------------------
// What is left of the gradient, chunk by chunk in parallel.  Wave w owns all 64 rows of columns [w HD/4, (w+1) HD/4) of
// dQ and dK, so a chunk's M and G are read once; the 64x64 matrices are formed tile by tile and shared through LDS.
template <int HD, typename T>
__global__ __launch_bounds__(256) void delta_grad_kernel(const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V,
                                                         Rows rq, Rows rk, Rows rv, const T* __restrict__ DO,
                                                         const float* __restrict__ ALPHA, const float* __restrict__ BETA,
                                                         const float* __restrict__ US, const float* __restrict__ RS,
                                                         const float* __restrict__ MS, const float* __restrict__ GS,
                                                         T* __restrict__ DQ, T* __restrict__ DK, float* __restrict__ DALPHA,
                                                         float* __restrict__ DBETA, int L, int H, int NC) {
    extern __shared__ __align__(16) char lds[];
    float(*ks)[HD + 4] = (float(*)[HD + 4])lds;
    float(*qs)[HD + 4] = ks + DC;
    float(*gt)[SQ] = (float(*)[SQ])(qs + DC);      // decays, [j][i]
    float(*dg)[SQ] = gt + DC;                      // gradients of the decays, [j][i]
    float(*dm)[SQ] = dg + DC;                      // dP o g, [i][j]; later the terms of da
    float(*es)[SQ] = dm + DC;                      // E + E^T
    float* sa = (float*)(es + DC);
    float* sb = sa + DC;
    float* sg = sb + DC;
    float(*sdb)[DC] = (float(*)[DC])(sg + DC);     // [jt][i]
    float(*red)[3][DC] = (float(*)[3][DC])(sdb + 4);   // [wave][q.X, k.Y, k.Z][i]
    float* srv = (float*)(red + 4);
    float* fro = srv + DC;
    constexpr int NN = HD / 64;                    // column tiles of a wave
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, m = lane & 15, g4 = (lane >> 4) * 4;
    const int64_t ci = blockIdx.x;
    const int64_t bh = ci / NC;
    const int c = (int)(ci % NC), t0 = c * DC, left = L - t0 < DC ? L - t0 : DC;
    const int64_t b = bh / H, h = bh % H;
    rows_to_lds<HD, T, 256>(K, rk.at(b, L, t0, h, HD), rk.ld, left, ks, tid);
    rows_to_lds<HD, T, 256>(Q, rq.at(b, L, t0, h, HD), rq.ld, left, qs, tid);
    if (tid < DC) {
        const int64_t at = (b * L + t0 + tid) * H + h;
        sa[tid] = tid < left ? ALPHA[at] : 1.0f;
        sb[tid] = tid < left ? BETA[at] : 0.0f;
    }
    (&sdb[0][0])[tid] = 0.f;
    __syncthreads();
    if (wave == 0) chunk_decays(sa, gt, lane);
    if (wave == 1) sg[lane] = chunk_prefix(sa, lane);
    __syncthreads();
    const float* ub = US + ci * DC * HD;
    const float* rb = RS + ci * DC * HD;
    const T* dob = DO + ((b * L + t0) * H + h) * HD;
    const int64_t dold = (int64_t)H * HD;
    auto do4 = [&](int row, int col) -> f32x4_t {
        return row < left ? load4(dob + (int64_t)row * dold + col) : (f32x4_t){0.f, 0.f, 0.f, 0.f};
    };
    // the 64x64 matrices: lane holds column i, rows j = 4g..4g+3 of a tile
    for (int tile = wave; tile < TRI; tile += 4) {
        const int it = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3, jt = tile - tri(it, 0);
        const int i = 16 * it + m, jr = 16 * jt + m;
        f32x4_t qk = {0.f, 0.f, 0.f, 0.f}, kk = qk, dp = qk, ru = qk;
#pragma unroll 4
        for (int u = 0; u < HD / 16; ++u) {
            const int col = 16 * u + g4;
            const f32x4_t kj = *(const f32x4_t*)&ks[jr][col], qi = *(const f32x4_t*)&qs[i][col],
                          ki = *(const f32x4_t*)&ks[i][col], uj = *(const f32x4_t*)(ub + jr * HD + col),
                          ri = *(const f32x4_t*)(rb + i * HD + col), oi = do4(i, col);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                qk = mfma_f32(kj[r], qi[r], qk);
                kk = mfma_f32(kj[r], ki[r], kk);
                dp = mfma_f32(uj[r], oi[r], dp);
                ru = mfma_f32(uj[r], ri[r], ru);
            }
        }
        const float bi = sb[i];
        f32x4_t d;
        float db = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int j = 16 * jt + g4 + r;
            const float gij = gt[j][i];            // 0 above the diagonal
            d[r] = dp[r] * gij;
            const float ag = i > j ? -ru[r] * gij : 0.f;      // dA_ij g_ij
            db = fmaf(ag, kk[r], db);
            dg[j][i] = i > j ? fmaf(dp[r], qk[r], -ru[r] * bi * kk[r]) : 0.f;
            if (i >= j) {
                es[i][j] = bi * ag;
                es[j][i] = bi * ag;
            }
        }
        *(f32x4_t*)&dm[i][16 * jt + g4] = d;
        db += __shfl_xor(db, 16);
        db += __shfl_xor(db, 32);
        if (lane < 16) sdb[jt][i] = db;
    }
    // X, Y, Z and <G, M>
    f32x4_t X[4][NN], Y[4][NN], Z[4][NN];
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
        for (int n = 0; n < NN; ++n) X[it][n] = Y[it][n] = Z[it][n] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    const float* mb = MS + ci * HD * HD + wave * (HD / 4) + m;
    const float* gb = GS + ci * HD * HD + wave * (HD / 4) + m;
    float gm = 0.f, rdotv = 0.f;
    const int64_t vrow = rv.at(b, L, t0, h, HD);
#pragma unroll 1
    for (int u = 0; u < HD / 16; ++u) {
        const int col = 16 * u + g4;
        f32x4_t ao[4], ar[4], au[4];
        float bm[NN][4], bg[NN][4];
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            const int row = 16 * it + m;
            ao[it] = do4(row, col);
            ar[it] = *(const f32x4_t*)(rb + row * HD + col);
            au[it] = *(const f32x4_t*)(ub + row * HD + col);
        }
#pragma unroll
        for (int n = 0; n < NN; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                bm[n][r] = mb[(col + r) * HD + 16 * n];
                bg[n][r] = gb[(col + r) * HD + 16 * n];
            }
        {
            const int row = 16 * wave + m;
            f32x4_t vv = {0.f, 0.f, 0.f, 0.f};
            if (row < left) vv = load4(V + vrow + (int64_t)row * rv.ld + col);
            const f32x4_t rr = *(const f32x4_t*)(rb + row * HD + col);
#pragma unroll
            for (int r = 0; r < 4; ++r) rdotv = fmaf(rr[r], vv[r], rdotv);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int n = 0; n < NN; ++n) {
                gm = fmaf(bm[n][r], bg[n][r], gm);
#pragma unroll
                for (int it = 0; it < 4; ++it) {
                    X[it][n] = mfma_f32(ao[it][r], bm[n][r], X[it][n]);
                    Y[it][n] = mfma_f32(ar[it][r], bm[n][r], Y[it][n]);
                    Z[it][n] = mfma_f32(au[it][r], bg[n][r], Z[it][n]);
                }
            }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) gm += __shfl_xor(gm, off);
    if (lane == 0) fro[wave] = gm;
    rdotv += __shfl_xor(rdotv, 16);
    rdotv += __shfl_xor(rdotv, 32);
    if (lane < 16) srv[16 * wave + m] = rdotv;
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = 16 * it + g4 + r;
            float x = 0.f, y = 0.f, z = 0.f;
#pragma unroll
            for (int n = 0; n < NN; ++n) {
                const int col = wave * (HD / 4) + 16 * n + m;
                const float kv = ks[i][col];
                x = fmaf(qs[i][col], X[it][n][r], x);
                y = fmaf(kv, Y[it][n][r], y);
                z = fmaf(kv, Z[it][n][r], z);
            }
#pragma unroll
            for (int off = 1; off < 16; off <<= 1) {
                x += __shfl_xor(x, off);
                y += __shfl_xor(y, off);
                z += __shfl_xor(z, off);
            }
            if (m == 0) red[wave][0][i] = x, red[wave][1][i] = y, red[wave][2][i] = z;
            const float gi = sg[i], ge = gt[i][DC - 1], bgi = sb[i] * gi;
#pragma unroll
            for (int n = 0; n < NN; ++n) {
                Z[it][n][r] = ge * Z[it][n][r] - bgi * Y[it][n][r];
                X[it][n][r] *= gi;
            }
        }
    __syncthreads();                               // dm, es, dg and the row sums are complete
#pragma unroll 1
    for (int jt = 0; jt < 4; ++jt) {
        f32x4_t ad[4], ae[4];
        float at[4][4], bk[NN][4], bq[NN][4];
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            if (it >= jt) ad[it] = *(const f32x4_t*)&dm[16 * it + m][16 * jt + g4];
            ae[it] = *(const f32x4_t*)&es[16 * it + m][16 * jt + g4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (it <= jt) at[it][r] = dm[16 * jt + g4 + r][16 * it + m];
        }
#pragma unroll
        for (int n = 0; n < NN; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int col = wave * (HD / 4) + 16 * n + m;
                bk[n][r] = ks[16 * jt + g4 + r][col];
                bq[n][r] = qs[16 * jt + g4 + r][col];
            }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int n = 0; n < NN; ++n)
#pragma unroll
                for (int it = 0; it < 4; ++it) {
                    if (it >= jt) X[it][n] = mfma_f32(ad[it][r], bk[n][r], X[it][n]);
                    if (it <= jt) Z[it][n] = mfma_f32(at[it][r], bq[n][r], Z[it][n]);
                    Z[it][n] = mfma_f32(ae[it][r], bk[n][r], Z[it][n]);
                }
    }
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = 16 * it + g4 + r;
            if (i < left) {
                const int64_t at = ((b * L + t0 + i) * H + h) * HD + wave * (HD / 4) + m;
#pragma unroll
                for (int n = 0; n < NN; ++n) {
                    elem<T>::put(DQ + at + 16 * n, X[it][n][r]);
                    elem<T>::put(DK + at + 16 * n, Z[it][n][r]);
                }
            }
        }
    __syncthreads();                               // dm is free
    if (wave == 0) {
        const float ky = red[0][1][lane] + red[1][1][lane] + red[2][1][lane] + red[3][1][lane];
        const float qx = red[0][0][lane] + red[1][0][lane] + red[2][0][lane] + red[3][0][lane];
        float w = qx - sb[lane] * ky;              // d(g_i)
        if (lane == DC - 1) w += fro[0] + fro[1] + fro[2] + fro[3];
        for (int t = 0; t < DC; ++t) {
            dm[t][lane] = t <= lane ? gt[t][lane] * w : 0.f;
            float d = t < lane ? dg[t][lane] : 0.f;
            // the decays from every token to the chunk's end carry k_t.Z_t too
            if (lane == DC - 1 && t < DC - 1) d += red[0][2][t] + red[1][2][t] + red[2][2][t] + red[3][2][t];
            w = fmaf(sa[t], w, d);
        }
        float da = 0.f;
        for (int i = 0; i < DC; ++i) da += dm[lane][i];
        if (lane < left) {
            const int64_t at = (b * L + t0 + lane) * H + h;
            DALPHA[at] = da;
            DBETA[at] = sdb[0][lane] + sdb[1][lane] + sdb[2][lane] + sdb[3][lane] + srv[lane] - sg[lane] * ky;
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------
// One token: S <- a S + u k^T, u = b (v - a S k), o = S q = a (S_old q) + u (k.q).  The state is read and written once and
// its rows are independent: HD/4 lanes hold a row (16 bytes each), the row's two dot products are summed across them.
template <int HD, typename T>
__global__ __launch_bounds__(256) void delta_step_kernel(const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V,
                                                         int64_t ldq, int64_t ldk, int64_t ldv, const float* __restrict__ ALPHA,
                                                         const float* __restrict__ BETA, float* __restrict__ STATE,
                                                         T* __restrict__ O, int H, int rows_per_wg) {
    constexpr int LPR = HD / 4, RPP = 256 / LPR;   // lanes of a row, rows of a pass
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const int per = HD / rows_per_wg;
    const int64_t bh = blockIdx.x / per, b = bh / H, h = bh % H;
    const int row0 = (int)(blockIdx.x % per) * rows_per_wg;
    const f32x4_t k4 = load4(K + b * ldk + h * HD + 4 * lane), q4 = load4(Q + b * ldq + h * HD + 4 * lane);
    const float a = ALPHA[bh], bt = BETA[bh];
    float kq = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) kq = fmaf(k4[e], q4[e], kq);
#pragma unroll
    for (int off = 1; off < LPR; off <<= 1) kq += __shfl_xor(kq, off);
    for (int row = row0 + sub; row < row0 + rows_per_wg; row += RPP) {
        f32x4_t* p = (f32x4_t*)(STATE + (bh * HD + row) * HD + 4 * lane);
        const float v = elem<T>::get(V + b * ldv + h * HD + row);
        f32x4_t s = *p;
        float sk = 0.f, sq = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) sk = fmaf(s[e], k4[e], sk), sq = fmaf(s[e], q4[e], sq);
#pragma unroll
        for (int off = 1; off < LPR; off <<= 1) {
            sk += __shfl_xor(sk, off);
            sq += __shfl_xor(sq, off);
        }
        const float u = bt * (v - a * sk);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = fmaf(u, k4[e], a * s[e]);
        *p = s;
        if (lane == 0) elem<T>::put(O + bh * HD + row, fmaf(u, kq, a * sq));
    }
}

// ---- host side ------------------------------------------------------------------------------------------------
struct DeltaArgs {
    const void *q, *k, *v;
    int64_t ldq, ldk, ldv;
    const float *alpha, *beta;
    int64_t B, L, H, hd;
    bool bf16;
    int64_t chunks() const { return (L + DC - 1) / DC; }
};

int delta_check(const char* who, const DeltaArgs& d) {
    VA_CHECK_ARG(d.q && d.k && d.v && d.alpha && d.beta, "%s: null operand", who);
    VA_CHECK_ARG(d.B > 0 && d.L > 0 && d.H > 0, "%s: empty problem", who);
    VA_CHECK_ARG(d.hd == 64 || d.hd == 128, "%s: head dim %lld not supported (64 or 128)", who, (long long)d.hd);
    const int64_t bytes = d.bf16 ? 8 : 16;         // four elements are read at a time
    VA_CHECK_ARG(d.ldq >= d.H * d.hd && d.ldk >= d.H * d.hd && d.ldv >= d.H * d.hd && (d.ldq | d.ldk | d.ldv) % 4 == 0,
                 "%s: a row stride must be at least H * hd and a multiple of 4", who);
    VA_CHECK_ARG(((uintptr_t)d.q | (uintptr_t)d.k | (uintptr_t)d.v) % bytes == 0, "%s: misaligned operand", who);
    VA_CHECK_ARG(d.L < (1ll << 30) && d.H < (1ll << 20) && d.B < (1ll << 30) && d.B * d.H < (1ll << 24) &&
                     d.B * d.H * d.chunks() < (1ll << 31) && d.ldq < (1ll << 30) && d.ldk < (1ll << 30) && d.ldv < (1ll << 30),
                 "%s: problem too large", who);
    return VA_OK;
}

int reserve_lds(const char* who, const void* fn, int bytes) {
    if (hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) {
        (void)hipGetLastError();
        va_set_error("%s: cannot reserve %d bytes of LDS", who, bytes);
        return VA_ERR_LAUNCH;
    }
    return VA_OK;
}
#define VA_TRY(x)                    \
    do {                             \
        const int rc__ = (x);        \
        if (rc__ != VA_OK) return rc__; \
    } while (0)

template <int HD, typename T, bool GRAD>
int launch_prep(const DeltaArgs& d, float* tf, float* tt, float* pf, float* gam, hipStream_t stream) {
    constexpr int lds = (2 * DC * (HD + 4) + 2 * DC * SQ + DC * 20 + 2 * DC) * 4;
    const auto fn = delta_prep_kernel<HD, T, GRAD>;
    VA_TRY(reserve_lds("va_gated_delta", (const void*)fn, lds));
    hipLaunchKernelGGL(fn, dim3((unsigned)(d.B * d.H * d.chunks())), dim3(256), lds, stream, (const T*)d.q, (const T*)d.k,
                       Rows{d.ldq}, Rows{d.ldk}, d.alpha, d.beta, tf, tt, pf, gam, (int)d.L, (int)d.H, (int)d.chunks());
    VA_CHECK_LAUNCH("va_gated_delta (decays)");
    return VA_OK;
}

template <int HD, typename T, int W, bool OUT, bool SAVE>
int launch_scan(const DeltaArgs& d, const float* tf, const float* pf, const float* gam, const float* state_in, void* out,
                float* state_out, float* us, float* ms, hipStream_t stream) {
    constexpr int lds = ((OUT ? 2 : 1) * DC * (HD + 4) + 3 * DC) * 4;
    const auto fn = delta_scan_kernel<HD, T, W, OUT, SAVE>;
    VA_TRY(reserve_lds("va_gated_delta", (const void*)fn, lds));
    hipLaunchKernelGGL(fn, dim3((unsigned)(d.B * d.H * (HD / 16 / W))), dim3(64 * W), lds, stream, (const T*)d.q, (const T*)d.k,
                       (const T*)d.v, Rows{d.ldq}, Rows{d.ldk}, Rows{d.ldv}, d.beta, tf, pf, gam, state_in, (T*)out, state_out, us,
                       ms, (int)d.L, (int)d.H, (int)d.chunks());
    VA_CHECK_LAUNCH("va_gated_delta (scan)");
    return VA_OK;
}

template <int HD, typename T, int W>
int launch_rscan(const DeltaArgs& d, const void* d_out, const float* tt, const float* pt, const float* gam, const float* d_state,
                 void* dv, float* d_state_in, float* rs, float* gs, hipStream_t stream) {
    constexpr int lds = (2 * DC * (HD + 4) + 3 * DC) * 4;
    const auto fn = delta_rscan_kernel<HD, T, W>;
    VA_TRY(reserve_lds("va_gated_delta_bwd", (const void*)fn, lds));
    hipLaunchKernelGGL(fn, dim3((unsigned)(d.B * d.H * (HD / 16 / W))), dim3(64 * W), lds, stream, (const T*)d.q, (const T*)d.k,
                       Rows{d.ldq}, Rows{d.ldk}, (const T*)d_out, d.beta, tt, pt, gam, d_state, (T*)dv, d_state_in, rs, gs,
                       (int)d.L, (int)d.H, (int)d.chunks());
    VA_CHECK_LAUNCH("va_gated_delta_bwd (scan)");
    return VA_OK;
}

// Waves per workgroup of the scans: a wave's work does not depend on it, only how many waves share one copy of a chunk's
// rows.  Few heads are spread over as many CUs as there are pairs of waves, many heads keep all columns together.
int scan_waves(int64_t heads, int hd) { return heads * (hd / 16) >= 8 * 256 ? hd / 16 : 2; }

constexpr int64_t FWD_CHUNK_FLOATS = 2 * TRI * FRAG + 2 * DC;

template <int HD, typename T>
int delta_fwd(const DeltaArgs& d, const float* state_in, void* out, float* state_out, float* ws, hipStream_t stream) {
    const int64_t n = d.B * d.H * d.chunks();
    float *tf = ws, *pf = tf + n * TRI * FRAG, *gam = pf + n * TRI * FRAG;
    VA_TRY((launch_prep<HD, T, false>(d, tf, nullptr, pf, gam, stream)));
    if (scan_waves(d.B * d.H, HD) == 2)
        return launch_scan<HD, T, 2, true, false>(d, tf, pf, gam, state_in, out, state_out, nullptr, nullptr, stream);
    return launch_scan<HD, T, HD / 16, true, false>(d, tf, pf, gam, state_in, out, state_out, nullptr, nullptr, stream);
}

template <int HD, typename T>
int delta_bwd(const DeltaArgs& d, const void* d_out, const float* d_state, const float* state_in, void* dq, void* dk, void* dv,
              float* dalpha, float* dbeta, float* d_state_in, float* ws, hipStream_t stream) {
    const int64_t n = d.B * d.H * d.chunks();
    float *tf = ws, *tt = tf + n * TRI * FRAG, *pt = tt + n * TRI * FRAG, *gam = pt + n * TRI * FRAG;
    float *us = gam + n * 2 * DC, *rs = us + n * DC * HD, *ms = rs + n * DC * HD, *gs = ms + n * HD * HD;
    VA_TRY((launch_prep<HD, T, true>(d, tf, tt, pt, gam, stream)));
    if (scan_waves(d.B * d.H, HD) == 2) {
        VA_TRY((launch_scan<HD, T, 2, false, true>(d, tf, nullptr, gam, state_in, nullptr, nullptr, us, ms, stream)));
        VA_TRY((launch_rscan<HD, T, 2>(d, d_out, tt, pt, gam, d_state, dv, d_state_in, rs, gs, stream)));
    } else {
        VA_TRY((launch_scan<HD, T, HD / 16, false, true>(d, tf, nullptr, gam, state_in, nullptr, nullptr, us, ms, stream)));
        VA_TRY((launch_rscan<HD, T, HD / 16>(d, d_out, tt, pt, gam, d_state, dv, d_state_in, rs, gs, stream)));
    }
    constexpr int lds = (2 * DC * (HD + 4) + 4 * DC * SQ + 3 * DC + 4 * DC + 12 * DC + DC + 4) * 4;
    const auto fn = delta_grad_kernel<HD, T>;
    VA_TRY(reserve_lds("va_gated_delta_bwd", (const void*)fn, lds));
    hipLaunchKernelGGL(fn, dim3((unsigned)n), dim3(256), lds, stream, (const T*)d.q, (const T*)d.k, (const T*)d.v, Rows{d.ldq},
                       Rows{d.ldk}, Rows{d.ldv}, (const T*)d_out, d.alpha, d.beta, us, rs, ms, gs, (T*)dq, (T*)dk, dalpha, dbeta,
                       (int)d.L, (int)d.H, (int)d.chunks());
    VA_CHECK_LAUNCH("va_gated_delta_bwd (gradients)");
    return VA_OK;
}

}  // namespace

extern "C" int64_t va_gated_delta_fwd_workspace_floats(int64_t B, int64_t L, int64_t H, int64_t hd) {
    if (B <= 0 || L <= 0 || H <= 0 || (hd != 64 && hd != 128)) return 0;
    return B * H * ((L + DC - 1) / DC) * FWD_CHUNK_FLOATS;
}

extern "C" int64_t va_gated_delta_bwd_workspace_floats(int64_t B, int64_t L, int64_t H, int64_t hd) {
    if (B <= 0 || L <= 0 || H <= 0 || (hd != 64 && hd != 128)) return 0;
    return B * H * ((L + DC - 1) / DC) * (3 * TRI * FRAG + 2 * DC + 2 * DC * hd + 2 * hd * hd);
}

extern "C" int va_gated_delta_fwd(const void* q, const void* k, const void* v, int64_t ldq, int64_t ldk, int64_t ldv, int is_bf16,
                                  const float* alpha, const float* beta, const float* state_in, void* out, float* state_out,
                                  float* workspace, int64_t B, int64_t L, int64_t H, int64_t hd, hipStream_t stream) {
    const DeltaArgs d = {q, k, v, ldq, ldk, ldv, alpha, beta, B, L, H, hd, is_bf16 != 0};
    VA_TRY(delta_check("va_gated_delta_fwd", d));
    VA_CHECK_ARG(out && state_out && workspace, "va_gated_delta_fwd: null operand");
    VA_CHECK_ARG(((uintptr_t)state_in | (uintptr_t)state_out | (uintptr_t)workspace) % 16 == 0,
                 "va_gated_delta_fwd: misaligned state or workspace");
    if (hd == 128)
        return d.bf16 ? delta_fwd<128, bf16_t>(d, state_in, out, state_out, workspace, stream)
                      : delta_fwd<128, float>(d, state_in, out, state_out, workspace, stream);
    return d.bf16 ? delta_fwd<64, bf16_t>(d, state_in, out, state_out, workspace, stream)
                  : delta_fwd<64, float>(d, state_in, out, state_out, workspace, stream);
}

extern "C" int va_gated_delta_bwd(const void* d_out, const float* d_state, const void* q, const void* k, const void* v, int64_t ldq,
                                  int64_t ldk, int64_t ldv, int is_bf16, const float* alpha, const float* beta,
                                  const float* state_in, void* dq, void* dk, void* dv, float* dalpha, float* dbeta,
                                  float* d_state_in, float* workspace, int64_t B, int64_t L, int64_t H, int64_t hd,
                                  hipStream_t stream) {
    const DeltaArgs d = {q, k, v, ldq, ldk, ldv, alpha, beta, B, L, H, hd, is_bf16 != 0};
    VA_TRY(delta_check("va_gated_delta_bwd", d));
    VA_CHECK_ARG(d_out && dq && dk && dv && dalpha && dbeta && workspace, "va_gated_delta_bwd: null operand");
    VA_CHECK_ARG(((uintptr_t)state_in | (uintptr_t)d_state | (uintptr_t)d_state_in | (uintptr_t)workspace | (uintptr_t)d_out) % 16 == 0,
                 "va_gated_delta_bwd: misaligned state, gradient or workspace");
    if (hd == 128)
        return d.bf16 ? delta_bwd<128, bf16_t>(d, d_out, d_state, state_in, dq, dk, dv, dalpha, dbeta, d_state_in, workspace, stream)
                      : delta_bwd<128, float>(d, d_out, d_state, state_in, dq, dk, dv, dalpha, dbeta, d_state_in, workspace, stream);
    return d.bf16 ? delta_bwd<64, bf16_t>(d, d_out, d_state, state_in, dq, dk, dv, dalpha, dbeta, d_state_in, workspace, stream)
                  : delta_bwd<64, float>(d, d_out, d_state, state_in, dq, dk, dv, dalpha, dbeta, d_state_in, workspace, stream);
}

extern "C" int va_gated_delta_step(const void* q, const void* k, const void* v, int64_t ldq, int64_t ldk, int64_t ldv, int is_bf16,
                                   const float* alpha, const float* beta, float* state, void* out, int64_t B, int64_t H, int64_t hd,
                                   hipStream_t stream) {
    const DeltaArgs d = {q, k, v, ldq, ldk, ldv, alpha, beta, B, 1, H, hd, is_bf16 != 0};
    VA_TRY(delta_check("va_gated_delta_step", d));
    VA_CHECK_ARG(state && out, "va_gated_delta_step: null operand");
    VA_CHECK_ARG((uintptr_t)state % 16 == 0, "va_gated_delta_step: misaligned state");
    // rows per workgroup: one pass of rows while that leaves fewer than four workgroups to a CU, the whole state otherwise
    const int pass = 1024 / (int)hd;
    const int rows = B * H * (hd / pass) <= 4 * 256 ? pass : (int)hd;
    const unsigned grid = (unsigned)(B * H * (hd / rows));
    if (hd == 128) {
        if (d.bf16)
            hipLaunchKernelGGL((delta_step_kernel<128, bf16_t>), dim3(grid), dim3(256), 0, stream, (const bf16_t*)q, (const bf16_t*)k,
                               (const bf16_t*)v, ldq, ldk, ldv, alpha, beta, state, (bf16_t*)out, (int)H, rows);
        else
            hipLaunchKernelGGL((delta_step_kernel<128, float>), dim3(grid), dim3(256), 0, stream, (const float*)q, (const float*)k,
                               (const float*)v, ldq, ldk, ldv, alpha, beta, state, (float*)out, (int)H, rows);
    } else {
        if (d.bf16)
            hipLaunchKernelGGL((delta_step_kernel<64, bf16_t>), dim3(grid), dim3(256), 0, stream, (const bf16_t*)q, (const bf16_t*)k,
                               (const bf16_t*)v, ldq, ldk, ldv, alpha, beta, state, (bf16_t*)out, (int)H, rows);
        else
            hipLaunchKernelGGL((delta_step_kernel<64, float>), dim3(grid), dim3(256), 0, stream, (const float*)q, (const float*)k,
                               (const float*)v, ldq, ldk, ldv, alpha, beta, state, (float*)out, (int)H, rows);
    }
    VA_CHECK_LAUNCH("va_gated_delta_step");
    return VA_OK;
}
