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
// products, never differences of logarithms).  delta_rscan_kernel walks backwards, then delta_grad_kernel takes the chunks in
// parallel, both from the forward's T^T, P^T, U and chunk states (kept by it, or formed again by its two kernels).
// Heads with a result that is not finite go through delta_grad_by_token_kernel behind them.
//
// Numbers on the matrix pipe.  The bf16 instruction (16x16x32) does sixteen times the products of the f32 one (16x16x4) per
// cycle, so the scans split every f32 operand into three bf16 numbers, x = x0 + x1 + x2 with |x1| <= 2^-8 |x| and
// |x2| <= 2^-16 |x| (nothing is left of 24 bits), and add the six products x_a y_b with a + b <= 2 into one f32 accumulator;
// what is left out, x1 y2 + x2 y1 + x2 y2, is at most 2^-23 + 2^-32 of |x y|, an f32 product's step.  bf16 inputs are one such
// number: three products.  Where a result is rounded to bf16 in the end, two numbers per operand are kept: 2^-16 of each operand
// and of each product is lost, a 256th of that rounding's half step.  The 64x64 systems (prep) and the
// last gradients (grad) run on the f32 instruction.
// Both instructions take a right operand from an accumulator as it lies: register r of lane group g holds row 4g+r of a tile,
// and any order of the contraction index will do if the left operand follows it: for the f32 one index 4g+r at step r, for
// the bf16 one elements 0..3 from the first and 4..7 from the second of two tiles.  V - K M, U, M and G feed the next product
// from their registers.
#include "common.h"

namespace {

constexpr int DC = 64;                    // tokens per chunk
constexpr int TRI = 10;                   // 16x16 blocks of a lower triangle of 64x64
constexpr int SQ = DC + 4;                // row stride of 64x64 matrices in LDS
constexpr int BLK = 6;                    // 16x32 operand blocks that cover a triangle of 64x64
constexpr int BFRAG = 512;                // bf16 numbers of one: lane l holds row l%16, columns 4(l/16)+{0..3, 16..19}

template <int V> struct int_c { static constexpr int value = V; };

VA_DEVINL f32x4_t mfma_f32(float a, float b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
// index of block (it, jt), it >= jt, of a lower triangle
__host__ __device__ constexpr int tri(int it, int jt) { return it * (it + 1) / 2 + jt; }

VA_DEVINL f32x4_t widen4(f32x4_t v) { return v; }
VA_DEVINL f32x4_t widen4(u32x2_t p) {
    return (f32x4_t){__uint_as_float(p[0] << 16), __uint_as_float(p[0] & 0xffff0000u), __uint_as_float(p[1] << 16),
                     __uint_as_float(p[1] & 0xffff0000u)};
}
// A chunk's rows of one head through a buffer descriptor that ends behind the chunk's last token: offsets of 32 bits, rows
// behind the sequence read as zeros and are not written, without a branch.
template <typename T> struct ChunkOf;
struct ChunkBase {
    __amdgpu_buffer_rsrc_t r;
    int row;                                      // bytes between rows
};
VA_DEVINL ChunkBase chunk_base(const void* first, int64_t row_bytes, int rows) {
    ChunkBase c;
    c.row = (int)row_bytes;
    c.r = __builtin_amdgcn_make_buffer_rsrc((void*)first, (short)0, (int)(row_bytes * rows), 0x00020000);
    return c;
}
template <> struct ChunkOf<float> {
    typedef f32x4_t raw4;
    ChunkBase c;
    VA_DEVINL raw4 raw(int row, int col) const { return __builtin_bit_cast(raw4, __builtin_amdgcn_raw_buffer_load_b128(c.r, row * c.row + col * 4, 0, 0)); }
    VA_DEVINL float get(int row, int col) const { return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(c.r, row * c.row + col * 4, 0, 0)); }
    VA_DEVINL void put(int row, int col, float x) const { __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x), c.r, row * c.row + col * 4, 0, 0); }
};
template <> struct ChunkOf<bf16_t> {
    typedef u32x2_t raw4;
    ChunkBase c;
    VA_DEVINL raw4 raw(int row, int col) const { return __builtin_bit_cast(raw4, __builtin_amdgcn_raw_buffer_load_b64(c.r, row * c.row + col * 2, 0, 0)); }
    VA_DEVINL float get(int row, int col) const { return bf16_to_f32(__builtin_amdgcn_raw_buffer_load_b16(c.r, row * c.row + col * 2, 0, 0)); }
    // results of the tensors' own type: one rounding
    VA_DEVINL void put(int row, int col, float x) const { __builtin_amdgcn_raw_buffer_store_b16(f32_to_bf16(x), c.r, row * c.row + col * 2, 0, 0); }
};
template <typename T> VA_DEVINL ChunkOf<T> chunk_of(const T* first, int64_t ld, int rows) {
    return ChunkOf<T>{chunk_base(first, ld * (int64_t)sizeof(T), rows)};
}

// where a token's row of one head lies: rows of `ld` elements, heads side by side
struct Rows {
    int64_t ld;
    VA_DEVINL int64_t at(int64_t b, int64_t L, int64_t t, int64_t h, int64_t hd) const { return (b * L + t) * ld + h * hd; }
};
// Chunk of a workgroup in the kernels that take all chunks at once: the heads of a token are neighbours in memory, so
// neighbouring workgroups take them (one head's rows alone keep to few memory channels).
VA_DEVINL void chunk_place(int64_t id, int H, int NC, int64_t& b, int& h, int& c) {
    h = (int)(id % H);
    c = (int)(id / H % NC);
    b = id / H / NC;
}

// how many bf16 numbers stand for an input element, for an intermediate, and for an operand of an output
template <typename T> struct parts;
template <> struct parts<float> { static constexpr int IN = 3, MID = 3, OUT = 3; };
template <> struct parts<bf16_t> { static constexpr int IN = 1, MID = 3, OUT = 2; };

// eight f32 values (two accumulator tiles of a lane) -> N operands of eight bf16 numbers each
template <int N>
VA_DEVINL void split(f32x4_t a, f32x4_t b, bf16x8_t (&out)[N]) {
    float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
#pragma unroll
    for (int n = 0; n < N; ++n) {
        u32x4_t w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[e] = pack_bf16x2(x[2 * e], x[2 * e + 1]);
            x[2 * e] -= __uint_as_float(w[e] << 16);
            x[2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
        }
        out[n] = __builtin_bit_cast(bf16x8_t, w);
    }
}
// acc[c][first + x] += a[x] * b[c] from their parts, every pair whose product is above 2^-24 of the whole; independent
// accumulators follow each other
template <int X, int NA, int NB, int CG, int N>
VA_DEVINL void mfma_parts(const bf16x8_t (&a)[X][NA], const bf16x8_t (&b)[CG][NB], f32x4_t (&acc)[CG][N], int first) {
    constexpr int KEEP = NA > NB ? NA : NB;
#pragma unroll
    for (int i = NA - 1; i >= 0; --i)
#pragma unroll
        for (int j = NB - 1; j >= 0; --j)
            if (i + j < KEEP) {
#pragma unroll
                for (int x = 0; x < X; ++x)
#pragma unroll
                    for (int c = 0; c < CG; ++c) acc[c][first + x] = mfma16(a[x][i], b[c][j], acc[c][first + x]);
            }
}
// operand blocks: (row tile it, columns 32u..) of a lower triangle, and of an upper one
__host__ __device__ constexpr int low_block(int it, int u) { return it < 2 ? it : 2 * it - 2 + u; }
__host__ __device__ constexpr int up_block(int jt, int u) { return jt < 2 ? 2 * jt + u : 2 + jt; }
template <int N>
VA_DEVINL void load_block(const char* base, int block, int lane, bf16x8_t (&out)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) out[n] = *(const bf16x8_t*)(base + (block * N + n) * BFRAG * 2 + lane * 16);
}
// acc[c][first..] += (row tiles first..first + X - 1, column block u) of an operand in LDS times b
template <int X, bool UP, int NA, int NB, int CG>
VA_DEVINL void blocks_times(const char* base, int first, int u, const bf16x8_t (&b)[CG][NB], f32x4_t (&acc)[CG][4], int lane) {
    bf16x8_t a[X][NA];
#pragma unroll
    for (int x = 0; x < X; ++x) load_block(base, UP ? up_block(first + x, u) : low_block(first + x, u), lane, a[x]);
    mfma_parts(a, b, acc, first);
}
template <int N>
VA_DEVINL void store_block(bf16_t* base, int block, int lane, const bf16x8_t (&v)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n) *(bf16x8_t*)(base + (block * N + n) * BFRAG + lane * 8) = v[n];
}

// Decays of a chunk, `mine` = lane's own a (1 behind the sequence's end): lane i of one wave walks the tokens back from i,
// gt[j][i] = a_{j+1} ... a_i for j <= i, 0 above.
VA_DEVINL void chunk_decays(float mine, float (*gt)[SQ], int lane) {
    float p = 0.f;
#pragma unroll
    for (int j = DC - 1; j >= 0; --j) {
        if (j + 1 < DC) p *= __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine), j + 1));
        p = j == lane ? 1.0f : j < lane ? p : 0.f;
        gt[j][lane] = p;
    }
}
// lane i: a_0 ... a_i
VA_DEVINL float chunk_prefix(float mine, int lane) {
    float p = mine;
#pragma unroll
    for (int off = 1; off < DC; off <<= 1) {
        const float q = __shfl_up(p, off);
        p = lane >= off ? p * q : p;
    }
    return p;
}

template <int HD, typename T, int THREADS>
VA_DEVINL void rows_to_lds(const ChunkOf<T>& src, float (*dst)[HD + 4], int tid) {
    constexpr int N = DC * HD / 4 / THREADS;
#pragma unroll
    for (int p = 0; p < N; ++p) {
        const int idx = p * THREADS + tid, row = idx / (HD / 4), c = (idx % (HD / 4)) * 4;
        *(f32x4_t*)&dst[row][c] = widen4(src.raw(row, c));
    }
}

// ---------------------------------------------------------------------------------------------------------------
// A chunk's rows in LDS as bf16 parts, plane n of a matrix at [n][row], rows of HD * 2 bytes in 16-byte pieces.  Columns
// 32u + 16h + 4g + r of a row are element 4h + r of piece 4u + g, so one 16-byte read is a left operand's eight elements; the
// pieces of row t stand at (piece ^ turn(t)), which spreads the sixteen rows of such a read, and the four rows times four
// pieces of a transposed one, over all banks.
template <int HD> VA_DEVINL int turn(int row) {
    return HD == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}
template <int HD> VA_DEVINL int piece_at(int row, int piece) { return row * HD * 2 + ((piece ^ turn<HD>(row)) << 4); }
// columns 4c .. 4c+3 of a row
template <int HD> VA_DEVINL int quad_at(int row, int c) { return piece_at<HD>(row, (c >> 3) * 4 + (c & 3)) + ((c >> 2) & 1) * 8; }

VA_DEVINL void put_rows(char* at, int plane, f32x4_t v) {        // f32: three parts
    float x[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int n = 0; n < 3; ++n) {
        const u32x2_t w = {pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3])};
        *(u32x2_t*)(at + n * plane) = w;
        x[0] -= __uint_as_float(w[0] << 16);
        x[1] -= __uint_as_float(w[0] & 0xffff0000u);
        x[2] -= __uint_as_float(w[1] << 16);
        x[3] -= __uint_as_float(w[1] & 0xffff0000u);
    }
}
VA_DEVINL void put_rows(char* at, int, u32x2_t v) { *(u32x2_t*)at = v; }

// left operand of rows 16 it.., columns 32u + 4g + {0..3, 16..19}
template <int HD, int N>
VA_DEVINL void row_frag(const char* x, int it, int u, int m, int g, bf16x8_t (&out)[N]) {
    const char* at = x + piece_at<HD>(16 * it + m, 4 * u + g);
#pragma unroll
    for (int n = 0; n < N; ++n) out[n] = *(const bf16x8_t*)(at + n * DC * HD * 2);
}

// ---------------------------------------------------------------------------------------------------------------
// One workgroup of four waves per chunk.  K K^T and Q K^T tiles are formed transposed, D[j][i] = k_j.x_i, so that a lane holds
// row i and four consecutive j; the wave with row tile w of K K^T (w + 1 tiles) takes row tile 3 - w of Q K^T, five tiles to
// each.  Writes T and P; TRAIN: T^T and P^T as well, for the gradient's scan (P^T's tiles are formed the other way round).
// Bound by memory when there are many chunks (100 KB of f32 rows and operands per chunk: 16 896 chunks of head dim 128 in
// 408 us, 4.1 TB/s), by its chain of small systems when there are few (40 chunks of bf16 rows: 9.6 us).  bf16 rows stay bf16
// in LDS and are multiplied by the bf16 instruction, whose products of them are exact (with f32 copies and the f32 instruction
// the 40 chunks took 12 us).  A and T lie over K in LDS so that three workgroups share a CU.
template <int HD, typename T, bool TRAIN>
__global__ __launch_bounds__(256) void delta_prep_kernel(const T* __restrict__ Q, const T* __restrict__ K, Rows rq, Rows rk,
                                                         const float* __restrict__ ALPHA, const float* __restrict__ BETA,
                                                         bf16_t* __restrict__ TF, bf16_t* __restrict__ PF, bf16_t* __restrict__ TT,
                                                         bf16_t* __restrict__ PT, float* __restrict__ GAM, int L, int H, int NC) {
    constexpr int NM = parts<T>::MID, NP = parts<T>::OUT;
    constexpr bool B16 = parts<T>::IN == 1;       // bf16 rows: the bf16 instruction multiplies them exactly
    constexpr int KBYTES = B16 ? DC * HD * 2 : DC * (HD + 4) * 4, ABYTES = DC * SQ * 4 + DC * 20 * 4;
    __shared__ __align__(16) char lds[(KBYTES > ABYTES ? KBYTES : ABYTES)];
    __shared__ float gt[DC][SQ];
    __shared__ float sb[DC];
    float(*ks)[HD + 4] = (float(*)[HD + 4])lds;
    float(*am)[SQ] = (float(*)[SQ])lds;           // A, then T: over K, which is not needed by then
    float(*dg)[20] = (float(*)[20])(am + DC);     // inverses of the four diagonal blocks of I + A
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 15, g4 = (lane >> 4) * 4;
    int64_t b;
    int h, c;
    chunk_place(blockIdx.x, H, NC, b, h, c);
    const int64_t ci = (b * H + h) * NC + c;
    const int t0 = c * DC, left = L - t0 < DC ? L - t0 : DC;
    const ChunkOf<T> qc = chunk_of(Q + rq.at(b, L, t0, h, HD), rq.ld, left);
    const ChunkOf<T> kc = chunk_of(K + rk.at(b, L, t0, h, HD), rk.ld, left);
    if constexpr (B16) {
#pragma unroll
        for (int p = 0; p < DC * HD / 4 / 256; ++p) {
            const int idx = p * 256 + tid, row = idx / (HD / 4), c4 = idx % (HD / 4);
            put_rows(lds + quad_at<HD>(row, c4), 0, kc.raw(row, c4 * 4));
        }
    } else {
        rows_to_lds<HD, T, 256>(kc, ks, tid);
    }
    const float mine = lane < left ? ALPHA[(b * L + t0 + lane) * H + h] : 1.0f;
    if (tid < DC) sb[tid] = tid < left ? BETA[(b * L + t0 + tid) * H + h] : 0.0f;
    if (wave == 0) chunk_decays(mine, gt, lane);
    if (wave == 1) GAM[ci * 2 * DC + lane] = chunk_prefix(mine, lane);
    __syncthreads();
    f32x4_t kk[4], qk[4], pt[4];                  // kk[jt]: rows `wave`; qk[jt]: rows 3 - wave; pt[it]: P^T's rows `wave`
#pragma unroll
    for (int x = 0; x < 4; ++x) kk[x] = qk[x] = pt[x] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    // one copy of the code per wave: which tiles it forms is then known to the compiler
    auto tiles = [&](auto wv) {
        constexpr int WV = decltype(wv)::value, QT = 3 - WV;
        if constexpr (B16) {
            const int g = g4 >> 2;
            auto q_frag = [&](int row, int u) {
                const u32x2_t lo = qc.raw(row, 32 * u + g4), hi = qc.raw(row, 32 * u + g4 + 16);
                return __builtin_bit_cast(bf16x8_t, (u32x4_t){lo[0], lo[1], hi[0], hi[1]});
            };
#pragma unroll
            for (int u = 0; u < HD / 32; ++u) {
                bf16x8_t mk[1], kx[1];
                row_frag<HD>(lds, WV, u, m, g, mk);
                const bf16x8_t mq = q_frag(16 * QT + m, u);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    if (x <= WV || x <= QT) row_frag<HD>(lds, x, u, m, g, kx);
                    if (x <= WV) kk[x] = mfma16(kx[0], mk[0], kk[x]);
                    if (x <= QT) qk[x] = mfma16(kx[0], mq, qk[x]);
                    if (TRAIN && x >= WV) pt[x] = mfma16(q_frag(16 * x + m, u), mk[0], pt[x]);
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < HD / 16; ++u) {
                const int col = 16 * u + g4;
                const f32x4_t mk = *(const f32x4_t*)&ks[16 * WV + m][col], mq = widen4(qc.raw(16 * QT + m, col));
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    f32x4_t kx = {0.f, 0.f, 0.f, 0.f}, qx = kx;
                    if (x <= WV || x <= QT) kx = *(const f32x4_t*)&ks[16 * x + m][col];
                    if (TRAIN && x >= WV) qx = widen4(qc.raw(16 * x + m, col));
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (x <= WV) kk[x] = mfma_f32(kx[r], mk[r], kk[x]);
                        if (x <= QT) qk[x] = mfma_f32(kx[r], mq[r], qk[x]);
                        if (TRAIN && x >= WV) pt[x] = mfma_f32(qx[r], mk[r], pt[x]);
                    }
                }
            }
        }
    };
    if (wave == 0) tiles(int_c<0>{});
    else if (wave == 1) tiles(int_c<1>{});
    else if (wave == 2) tiles(int_c<2>{});
    else tiles(int_c<3>{});
    __syncthreads();                              // K has been read
    if (wave == 2) GAM[ci * 2 * DC + DC + lane] = gt[lane][DC - 1];
    {
        const int i = 16 * wave + m, qt = 3 - wave;
        const float bi = sb[i];
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) {
            if (jt > wave) continue;
            f32x4_t v;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = 16 * jt + g4 + r;
                v[r] = i > j ? kk[jt][r] * bi * gt[j][i] : 0.f;
            }
            *(f32x4_t*)&am[i][16 * jt + g4] = v;
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int pi = 16 * qt + m, pj = 16 * x + g4 + r;           // P
                qk[x][r] = pi >= pj ? qk[x][r] * gt[pj][pi] : 0.f;
                const int ti = 16 * x + g4 + r;                              // P^T, row i of this wave
                if (TRAIN) pt[x][r] = ti >= i ? pt[x][r] * gt[i][ti] : 0.f;
            }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (2 * u <= qt) {
                bf16x8_t f[NP];
                split(qk[2 * u], qk[2 * u + 1], f);
                store_block(PF + ci * BLK * NP * BFRAG, low_block(qt, u), lane, f);
            }
            if (TRAIN && 2 * u + 1 >= wave) {
                bf16x8_t f[NM];
                split(pt[2 * u], pt[2 * u + 1], f);
                store_block(PT + ci * BLK * NM * BFRAG, up_block(wave, u), lane, f);
            }
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
    auto column = [&](auto wv) {
        constexpr int JT = decltype(wv)::value;
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            xb[it] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
            if (it == JT) {
#pragma unroll
                for (int r = 0; r < 4; ++r) xb[it][r] = dg[16 * it + g4 + r][m];
            }
            if (it > JT) {
                f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kt = JT; kt < it; ++kt) {
                    const f32x4_t a4 = *(const f32x4_t*)&am[16 * it + m][16 * kt + g4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) s = mfma_f32(a4[r], xb[kt][r], s);
                }
                const f32x4_t d4 = *(const f32x4_t*)&dg[16 * it + m][g4];
#pragma unroll
                for (int r = 0; r < 4; ++r) xb[it] = mfma_f32(-d4[r], s[r], xb[it]);
            }
        }
    };
    if (wave == 0) column(int_c<0>{});
    else if (wave == 1) column(int_c<1>{});
    else if (wave == 2) column(int_c<2>{});
    else column(int_c<3>{});
    __syncthreads();
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
        for (int r = 0; r < 4; ++r) am[16 * it + g4 + r][16 * wave + m] = xb[it][r];     // zeros above the diagonal too
    if (TRAIN) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (2 * u + 1 >= wave) {
                bf16x8_t f[NM];
                split(xb[2 * u], xb[2 * u + 1], f);
                store_block(TT + ci * BLK * NM * BFRAG, up_block(wave, u), lane, f);
            }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 2; ++u)
        if (2 * u <= wave) {
            const float* row = am[16 * wave + m] + 32 * u + g4;
            bf16x8_t f[NM];
            split(*(const f32x4_t*)row, *(const f32x4_t*)(row + 16), f);
            store_block(TF + ci * BLK * NM * BFRAG, low_block(wave, u), lane, f);
        }
}

// ---------------------------------------------------------------------------------------------------------------
// left operand of the transposed rows: columns 16 ct.. of x, tokens 32u + 4g + {0..3, 16..19}
template <int HD, int N>
VA_DEVINL void col_frag(const char* x, int ct, int u, int lane, bf16x8_t (&out)[N]) {
    const int q = (lane & 15) >> 2, p = lane & 3, g = lane >> 4;
    const char* lo = x + quad_at<HD>(32 * u + 4 * g + q, 4 * ct + p);
    const char* hi = x + quad_at<HD>(32 * u + 16 + 4 * g + q, 4 * ct + p);
#pragma unroll
    for (int n = 0; n < N; ++n) out[n] = join_tr(lds_read_tr16(lo + n * DC * HD * 2), lds_read_tr16(hi + n * DC * HD * 2));
}

// a workgroup's LDS writes are there; loads under way stay under way
VA_DEVINL void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// `bytes` (whole kilobytes) from memory to LDS without registers, a kilobyte per wave and step; the buffer form's LDS
// destination is one the compiler knows, so other LDS reads do not wait for it
template <int BYTES, int W>
VA_DEVINL void to_lds(const void* src, char* dst, int wave, int lane) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)src, (short)0, BYTES, 0x00020000);
#pragma unroll
    for (int x = 0; x < (BYTES / 1024 + W - 1) / W; ++x) {
        const int kb = x * W + wave;
        if (BYTES / 1024 % W == 0 || kb < BYTES / 1024)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)(dst + kb * 1024), 16, kb * 1024 + lane * 16, 0, 0, 0);
    }
}

// What the two scans share: what the next chunk needs, on its way from memory to LDS: rows of K (and Q), the two 64x64
// operands (NA and NB parts), b, g, g_C.  AHEAD: the operands wait in registers like the rows; without (two column groups
// leave no registers) they are loaded straight to LDS while the chunk's products with the state are formed.
template <int HD, typename T, int W, bool TWO, int NA, int NB, bool AHEAD>
struct ChunkRows {
    typedef typename ChunkOf<T>::raw4 raw4;
    static constexpr int N = DC * HD / 4 / (64 * W), IN = parts<T>::IN, MATRIX = IN * DC * HD * 2;
    static constexpr int A_BYTES = BLK * NA * BFRAG * 2, B_BYTES = BLK * NB * BFRAG * 2, KBS = (A_BYTES + B_BYTES) / 1024;
    static constexpr int A_AT = (TWO ? 2 : 1) * MATRIX, B_AT = A_AT + A_BYTES, F_AT = B_AT + B_BYTES, LDS = F_AT + 3 * DC * 4;
    static constexpr int NX = AHEAD ? (KBS + W - 1) / W : 1;
    const T *k, *q;                               // row 0 of this head
    int64_t ldk, ldq;
    const bf16_t *a, *b;                          // operands of this head's chunk 0
    const float *beta, *gam;
    int L, H, tid, wave;
    raw4 kn[N], qn[TWO ? N : 1];
    u32x4_t xn[NX];
    float bn, gn, en;
    VA_DEVINL void request(int c, int NC) {       // a chunk outside the sequence: nothing is read
        const bool inside = c >= 0 && c < NC;
        c = inside ? c : 0;
        const int left = inside ? (L - c * DC < DC ? L - c * DC : DC) : 0;
        const ChunkOf<T> kc = chunk_of(k + (int64_t)c * DC * ldk, ldk, left), qc = chunk_of(q + (int64_t)c * DC * ldq, ldq, left);
#pragma unroll
        for (int p = 0; p < N; ++p) {
            const int idx = p * 64 * W + tid, row = idx / (HD / 4), col = (idx % (HD / 4)) * 4;
            kn[p] = kc.raw(row, col);
            if (TWO) qn[p] = qc.raw(row, col);
        }
        if (AHEAD) {
            const ChunkBase ac = chunk_base(a + (int64_t)c * BLK * NA * BFRAG, A_BYTES, inside), bc = chunk_base(b + (int64_t)c * BLK * NB * BFRAG, B_BYTES, inside);
#pragma unroll
            for (int x = 0; x < NX; ++x) {
                const int kb = x * W + wave;      // a kilobyte of one of the two per wave and step
                if (kb < A_BYTES / 1024) xn[x] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(ac.r, kb * 1024 + (tid & 63) * 16, 0, 0));
                else if (kb < KBS) xn[x] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(bc.r, kb * 1024 - A_BYTES + (tid & 63) * 16, 0, 0));
            }
        }
        if (tid < DC) {
            bn = tid < left ? beta[((int64_t)c * DC + tid) * H] : 0.f;
            gn = gam[(int64_t)c * 2 * DC + tid];  // (chunk 0's instead)
            en = gam[(int64_t)c * 2 * DC + DC + tid];
        }
    }
    VA_DEVINL void place(char* lds, int c) {
#pragma unroll
        for (int p = 0; p < N; ++p) {
            const int idx = p * 64 * W + tid, at = quad_at<HD>(idx / (HD / 4), idx % (HD / 4));
            put_rows(lds + at, DC * HD * 2, kn[p]);
            if (TWO) put_rows(lds + MATRIX + at, DC * HD * 2, qn[p]);
        }
        if (AHEAD) {                              // the two operands lie one behind the other
#pragma unroll
            for (int x = 0; x < NX; ++x)
                if (x * W + wave < KBS) *(u32x4_t*)(lds + A_AT + (x * W + wave) * 1024 + (tid & 63) * 16) = xn[x];
        } else {
            to_lds<A_BYTES, W>(a + (int64_t)c * BLK * NA * BFRAG, lds + A_AT, wave, tid & 63);
            if (NB > 0) to_lds<B_BYTES, W>(b + (int64_t)c * BLK * NB * BFRAG, lds + B_AT, wave, tid & 63);
        }
        float* f = (float*)(lds + F_AT);
        if (tid < DC) f[tid] = bn, f[DC + tid] = gn, f[2 * DC + tid] = en;
    }
};

// acc[c][ct] += X^T B for all HD/16 column tiles of X, B (token blocks u) in parts
template <int HD, int NX, int NB, int CG>
VA_DEVINL void columns_times(const char* x_, const bf16x8_t (&b0)[CG][NB], const bf16x8_t (&b1)[CG][NB], f32x4_t (&acc)[CG][HD / 16],
                             int lane) {
#pragma unroll
    for (int ct = 0; ct < HD / 16; ct += 4) {
        bf16x8_t a[4][NX];
#pragma unroll
        for (int x = 0; x < 4; ++x) col_frag<HD>(x_, ct + x, 0, lane, a[x]);
        mfma_parts(a, b0, acc, ct);
#pragma unroll
        for (int x = 0; x < 4; ++x) col_frag<HD>(x_, ct + x, 1, lane, a[x]);
        mfma_parts(a, b1, acc, ct);
    }
}
// acc[c][it] += rows of X times B (column block u)
template <int HD, int NX, int NB, int CG>
VA_DEVINL void rows_times(const char* x, int u, const bf16x8_t (&b)[CG][NB], f32x4_t (&acc)[CG][4], int m, int g) {
    bf16x8_t a[4][NX];
#pragma unroll
    for (int it = 0; it < 4; ++it) row_frag<HD>(x, it, u, m, g, a[it]);
    mfma_parts(a, b, acc, 0);
}

// The 16 CG rows of a head's state that a wave owns, and their outputs of the tokens from `from` on, token by token: 4 / CG lanes to a row, its elements in
// registers.  The pointers stand at the head's first token; v, o and the states at the wave's first row.
template <int HD, typename T, int CG>
VA_DEVINL void rows_by_token(const T* q, const T* k, const T* v, int64_t ldq, int64_t ldk, int64_t ldv, const float* alpha,
                             const float* beta, const float* s_in, T* o, float* s_out, int from, int L, int H, int lane) {
    constexpr int ROWS = 16 * CG, N = HD * ROWS / 64 / 4;
    const int row = lane % ROWS, col = lane / ROWS * 4 * N;
    f32x4_t s[N];
#pragma unroll
    for (int n = 0; n < N; ++n) s[n] = s_in != nullptr ? *(const f32x4_t*)(s_in + row * HD + col + 4 * n) : (f32x4_t){0.f, 0.f, 0.f, 0.f};
    auto over_row = [](float x) {
#pragma unroll
        for (int off = ROWS; off < 64; off <<= 1) x += __shfl_xor(x, off);
        return x;
    };
#pragma unroll 1
    for (int t = 0; t < L; ++t) {
        const ChunkOf<T> qt = chunk_of(q + t * ldq, ldq, 1), kt = chunk_of(k + t * ldk, ldk, 1);
        const float a = alpha[(int64_t)t * H], b = beta[(int64_t)t * H];
        float dot = 0.f, sum = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const f32x4_t x = widen4(kt.raw(0, col + 4 * n));
#pragma unroll
            for (int r = 0; r < 4; ++r) dot = fmaf(s[n][r], x[r], dot);
        }
        const float add = b * (chunk_of(v + t * ldv, ldv, 1).get(0, row) - a * over_row(dot));
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const f32x4_t x = widen4(kt.raw(0, col + 4 * n)), y = widen4(qt.raw(0, col + 4 * n));
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[n][r] = fmaf(add, x[r], a * s[n][r]);
                sum = fmaf(s[n][r], y[r], sum);
            }
        }
        sum = over_row(sum);
        if (lane < ROWS && t >= from) chunk_of(o + (int64_t)t * H * HD, (int64_t)H * HD, 1).put(0, row, sum);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) *(f32x4_t*)(s_out + row * HD + col + 4 * n) = s[n];
}

// ---------------------------------------------------------------------------------------------------------------
// The sequential part.  A wave owns 16 CG columns (values of the head) of the state for the whole sequence: M in CG * HD/16
// accumulator tiles; W waves share a chunk's K, Q, T and P through LDS, the next chunk's are requested while one computes.
// OUT: writes o.  SAVE: writes U and every chunk's starting state (rows of S) for the gradient.
// Bound by its chain: per chunk and wave 360 matrix instructions (f32, head dim 128; 182 for bf16), about as many cycles of
// vector work (splits, addresses) and of LDS reads, which one wave per SIMD runs one after the other: 7.7 us a chunk for f32, 5
// for bf16; 512 heads x 2064 tokens of f32 in 0.81 ms (2.2 GB and 0.6 GB of operands).
// A product with a zero does not silence a NaN, and an infinity has no parts: a token with either would reach earlier tokens of
// its chunk.  A wave that ends with a non-finite output or state forms its rows again token by token, so that what the
// recurrence leaves finite is finite; the outputs of the chunks before stay.
template <int HD, typename T, int W, int CG, bool OUT, bool SAVE>
__global__ __launch_bounds__(64 * W) void delta_scan_kernel(const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V,
                                                            Rows rq, Rows rk, Rows rv, const float* __restrict__ ALPHA,
                                                            const float* __restrict__ BETA, const bf16_t* __restrict__ TF,
                                                            const bf16_t* __restrict__ PF, const float* __restrict__ GAM,
                                                            const float* __restrict__ STATE_IN,
                                                            T* __restrict__ O, float* __restrict__ STATE_OUT,
                                                            float* __restrict__ US, float* __restrict__ MS, int L, int H, int NC) {
    constexpr int NI = parts<T>::IN, NM = parts<T>::MID, NO = parts<T>::OUT;
    typedef ChunkRows<HD, T, W, OUT, NM, OUT ? NO : 0, CG == 1> CR;
    extern __shared__ __align__(16) char lds[];
    const char *ks = lds, *qs = lds + CR::MATRIX;
    const char *tl = lds + CR::A_AT, *pl = lds + CR::B_AT;
    const float *sb = (const float*)(lds + CR::F_AT), *sg = sb + DC, *se = sg + DC;
    constexpr int GROUPS = HD / 16 / (W * CG);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 15, g = lane >> 4, g4 = g * 4;
    const int wid = xcd_remap(blockIdx.x, gridDim.x);
    const int64_t bh = wid / GROUPS, b = bh / H, h = bh % H;
    const int v = ((wid % GROUPS) * W + wave) * 16 * CG + m;      // and v + 16 in the second group
    const T* vb = V + rv.at(b, L, 0, h, HD);
    CR cr;
    cr.k = K + rk.at(b, L, 0, h, HD), cr.q = Q + rq.at(b, L, 0, h, HD), cr.ldk = rk.ld, cr.ldq = rq.ld;
    cr.beta = BETA + b * L * H + h, cr.gam = GAM + bh * NC * 2 * DC, cr.L = L, cr.H = H, cr.tid = tid, cr.wave = wave;
    cr.a = TF + bh * NC * BLK * NM * BFRAG, cr.b = PF + bh * NC * BLK * NO * BFRAG;
    f32x4_t M[CG][HD / 16];
#pragma unroll
    for (int x = 0; x < CG; ++x)
#pragma unroll
        for (int u = 0; u < HD / 16; ++u) {
            M[x][u] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
            if (STATE_IN != nullptr) M[x][u] = *(const f32x4_t*)(STATE_IN + (bh * HD + v + 16 * x) * HD + 16 * u + g4);
        }
    int bad = NC;                                 // first chunk with a non-finite output of this lane
    cr.request(0, NC);
    for (int c = 0; c < NC; ++c) {
        const int t0 = c * DC, left = L - t0 < DC ? L - t0 : DC;
        const int64_t ci = bh * NC + c;
        __syncthreads();                          // everybody is done with the chunk before
        cr.place(lds, c);
        f32x4_t vv[CG][4];                        // this chunk's v columns, rows in accumulator order
        const ChunkOf<T> vc = chunk_of(vb + (int64_t)t0 * rv.ld, rv.ld, left);
#pragma unroll
        for (int x = 0; x < CG; ++x)
#pragma unroll
            for (int it = 0; it < 4; ++it)
#pragma unroll
                for (int r = 0; r < 4; ++r) vv[x][it][r] = vc.get(16 * it + g4 + r, v + 16 * x);
        lds_barrier();
        if (CG == 1) cr.request(c + 1, NC);
        f32x4_t rhs[CG][4], o[CG][4], U[CG][4];
#pragma unroll
        for (int x = 0; x < CG; ++x) {
            if (SAVE) {
#pragma unroll
                for (int u = 0; u < HD / 16; ++u) *(f32x4_t*)(MS + (ci * HD + v + 16 * x) * HD + 16 * u + g4) = M[x][u];
            }
#pragma unroll
            for (int it = 0; it < 4; ++it) rhs[x][it] = o[x][it] = U[x][it] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int u = 0; u < HD / 32; ++u) {
            bf16x8_t mf[CG][NM], mo[CG][NO];
#pragma unroll
            for (int x = 0; x < CG; ++x) {
                split(M[x][2 * u], M[x][2 * u + 1], mf[x]);
#pragma unroll
                for (int n = 0; n < NO; ++n) mo[x][n] = mf[x][n];
            }
            rows_times<HD, NI>(ks, u, mf, rhs, m, g);
            if (OUT) rows_times<HD, NI>(qs, u, mo, o, m, g);
        }
        bf16x8_t f0[CG][NM], f1[CG][NM];
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            const f32x4_t b4 = *(const f32x4_t*)(sb + 16 * it + g4), gg = *(const f32x4_t*)(sg + 16 * it + g4);
#pragma unroll
            for (int x = 0; x < CG; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    rhs[x][it][r] = b4[r] * (vv[x][it][r] - gg[r] * rhs[x][it][r]);
                    o[x][it][r] *= gg[r];
                }
        }
#pragma unroll
        for (int x = 0; x < CG; ++x) {
            split(rhs[x][0], rhs[x][1], f0[x]);
            split(rhs[x][2], rhs[x][3], f1[x]);
        }
        if (CG > 1) {
            wait_vm0();
            __syncthreads();                      // T and P are there
            cr.request(c + 1, NC);
        }
        blocks_times<4, false, NM>(tl, 0, 0, f0, U, lane);
        blocks_times<2, false, NM>(tl, 2, 1, f1, U, lane);
        if (SAVE) {
#pragma unroll
            for (int x = 0; x < CG; ++x)
#pragma unroll
                for (int it = 0; it < 4; ++it)
#pragma unroll
                    for (int r = 0; r < 4; ++r) US[(ci * DC + 16 * it + g4 + r) * HD + v + 16 * x] = U[x][it][r];
        }
        if (OUT) {
            bf16x8_t u0[CG][NO], u1[CG][NO];
#pragma unroll
            for (int x = 0; x < CG; ++x) {
                split(U[x][0], U[x][1], u0[x]);
                split(U[x][2], U[x][3], u1[x]);
            }
            blocks_times<4, false, NO>(pl, 0, 0, u0, o, lane);
            blocks_times<2, false, NO>(pl, 2, 1, u1, o, lane);
            const ChunkOf<T> oc = chunk_of((const T*)O + ((b * L + t0) * H + h) * HD, (int64_t)H * HD, left);
            float seen = 0.f;                     // NaN with any output that is not finite
#pragma unroll
            for (int x = 0; x < CG; ++x)
#pragma unroll
                for (int it = 0; it < 4; ++it)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        oc.put(16 * it + g4 + r, v + 16 * x, o[x][it][r]);
                        seen = fmaf(o[x][it][r], 0.f, seen);
                    }
            bad = seen != seen && c < bad ? c : bad;
        }
        const float gc = sg[DC - 1];
#pragma unroll
        for (int x = 0; x < CG; ++x) {
#pragma unroll
            for (int u = 0; u < HD / 16; ++u) M[x][u] *= gc;
#pragma unroll
            for (int it = 0; it < 4; ++it) U[x][it] *= *(const f32x4_t*)(se + 16 * it + g4);
            split(U[x][0], U[x][1], f0[x]);
            split(U[x][2], U[x][3], f1[x]);
        }
        columns_times<HD, NI>(ks, f0, f1, M, lane);
    }
    if constexpr (OUT) {
        float seen = 0.f;
#pragma unroll
        for (int x = 0; x < CG; ++x)
#pragma unroll
            for (int u = 0; u < HD / 16; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) seen = fmaf(M[x][u][r], 0.f, seen);
        if (__any(bad < NC || seen != seen)) {
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) bad = min(bad, __shfl_xor(bad, off));
            wait_vm0();                           // other lanes of the wave write over what this one has written
            const int64_t first = b * L * H + h, row = bh * HD + v - m;
            rows_by_token<HD, T, CG>(cr.q, cr.k, vb + v - m, rq.ld, rk.ld, rv.ld, ALPHA + first, cr.beta,
                                     STATE_IN != nullptr ? STATE_IN + row * HD : nullptr, O + first * HD + v - m,
                                     STATE_OUT + row * HD, bad * DC, L, H, lane);
            return;
        }
#pragma unroll
        for (int x = 0; x < CG; ++x)
#pragma unroll
            for (int u = 0; u < HD / 16; ++u) *(f32x4_t*)(STATE_OUT + (bh * HD + v + 16 * x) * HD + 16 * u + g4) = M[x][u];
    }
}

// ---------------------------------------------------------------------------------------------------------------
// The same walk backwards for G = dL/dM: writes every chunk's G (at its end, rows of dS), R and dv.  Bound as the scan: 32 heads
// x 21 chunks of f32, head dim 128, in 167 us.
template <int HD, typename T, int W, int CG>
__global__ __launch_bounds__(64 * W) void delta_rscan_kernel(const T* __restrict__ Q, const T* __restrict__ K, Rows rq, Rows rk,
                                                             const T* __restrict__ DO, const float* __restrict__ BETA,
                                                             const bf16_t* __restrict__ TT, const bf16_t* __restrict__ PT,
                                                             const float* __restrict__ GAM, const float* __restrict__ DSTATE,
                                                             T* __restrict__ DV, float* __restrict__ DSTATE_IN,
                                                             float* __restrict__ RS, float* __restrict__ GS, int L, int H, int NC) {
    constexpr int NI = parts<T>::IN, NM = parts<T>::MID;
    typedef ChunkRows<HD, T, W, true, NM, NM, CG == 1> CR;
    extern __shared__ __align__(16) char lds[];
    const char *ks = lds, *qs = lds + CR::MATRIX;
    const char *pl = lds + CR::A_AT, *tl = lds + CR::B_AT;
    const float *sb = (const float*)(lds + CR::F_AT), *sg = sb + DC, *se = sg + DC;
    constexpr int GROUPS = HD / 16 / (W * CG);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 15, g = lane >> 4, g4 = g * 4;
    const int wid = xcd_remap(blockIdx.x, gridDim.x);
    const int64_t bh = wid / GROUPS, b = bh / H, h = bh % H;
    const int v = ((wid % GROUPS) * W + wave) * 16 * CG + m;
    CR cr;
    cr.k = K + rk.at(b, L, 0, h, HD), cr.q = Q + rq.at(b, L, 0, h, HD), cr.ldk = rk.ld, cr.ldq = rq.ld;
    cr.beta = BETA + b * L * H + h, cr.gam = GAM + bh * NC * 2 * DC, cr.L = L, cr.H = H, cr.tid = tid, cr.wave = wave;
    cr.a = PT + bh * NC * BLK * NM * BFRAG, cr.b = TT + bh * NC * BLK * NM * BFRAG;
    f32x4_t G[CG][HD / 16];
#pragma unroll
    for (int x = 0; x < CG; ++x)
#pragma unroll
        for (int u = 0; u < HD / 16; ++u) {
            G[x][u] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
            if (DSTATE != nullptr) G[x][u] = *(const f32x4_t*)(DSTATE + (bh * HD + v + 16 * x) * HD + 16 * u + g4);
        }
    cr.request(NC - 1, NC);
    for (int c = NC - 1; c >= 0; --c) {
        const int t0 = c * DC, left = L - t0 < DC ? L - t0 : DC;
        const int64_t ci = bh * NC + c;
        __syncthreads();                          // everybody is done with the chunk before
        cr.place(lds, c);
        f32x4_t dov[CG][4];
        const ChunkOf<T> oc = chunk_of(DO + ((b * L + t0) * H + h) * HD, (int64_t)H * HD, left);
#pragma unroll
        for (int x = 0; x < CG; ++x)
#pragma unroll
            for (int it = 0; it < 4; ++it)
#pragma unroll
                for (int r = 0; r < 4; ++r) dov[x][it][r] = oc.get(16 * it + g4 + r, v + 16 * x);
        lds_barrier();
        if (CG == 1) cr.request(c - 1, NC);
        f32x4_t du[CG][4], R[CG][4];
#pragma unroll
        for (int x = 0; x < CG; ++x) {
#pragma unroll
            for (int u = 0; u < HD / 16; ++u) *(f32x4_t*)(GS + (ci * HD + v + 16 * x) * HD + 16 * u + g4) = G[x][u];
#pragma unroll
            for (int it = 0; it < 4; ++it) du[x][it] = R[x][it] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int u = 0; u < HD / 32; ++u) {
            bf16x8_t gf[CG][NM];
#pragma unroll
            for (int x = 0; x < CG; ++x) split(G[x][2 * u], G[x][2 * u + 1], gf[x]);
            rows_times<HD, NI>(ks, u, gf, du, m, g);
        }
        bf16x8_t o0[CG][NI], o1[CG][NI], f0[CG][NM], f1[CG][NM];
#pragma unroll
        for (int x = 0; x < CG; ++x) {
#pragma unroll
            for (int it = 0; it < 4; ++it) du[x][it] *= *(const f32x4_t*)(se + 16 * it + g4);
            split(dov[x][0], dov[x][1], o0[x]);
            split(dov[x][2], dov[x][3], o1[x]);
        }
        if (CG > 1) {
            wait_vm0();
            __syncthreads();                      // P^T and T^T are there
            cr.request(c - 1, NC);
        }
        blocks_times<2, true, NM>(pl, 0, 0, o0, du, lane);
        blocks_times<4, true, NM>(pl, 0, 1, o1, du, lane);
#pragma unroll
        for (int x = 0; x < CG; ++x) {
            split(du[x][0], du[x][1], f0[x]);
            split(du[x][2], du[x][3], f1[x]);
        }
        blocks_times<2, true, NM>(tl, 0, 0, f0, R, lane);
        blocks_times<4, true, NM>(tl, 0, 1, f1, R, lane);
        const float gc = sg[DC - 1];
        const ChunkOf<T> vc = chunk_of((const T*)DV + ((b * L + t0) * H + h) * HD, (int64_t)H * HD, left);
#pragma unroll
        for (int x = 0; x < CG; ++x) {
#pragma unroll
            for (int u = 0; u < HD / 16; ++u) G[x][u] *= gc;
#pragma unroll
            for (int it = 0; it < 4; ++it) {
                const f32x4_t b4 = *(const f32x4_t*)(sb + 16 * it + g4), gg = *(const f32x4_t*)(sg + 16 * it + g4);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * it + g4 + r;
                    RS[(ci * DC + i) * HD + v + 16 * x] = R[x][it][r];
                    const float dv = b4[r] * R[x][it][r];
                    vc.put(i, v + 16 * x, dv);
                    dov[x][it][r] *= gg[r];
                    R[x][it][r] = -gg[r] * dv;
                }
            }
            split(dov[x][0], dov[x][1], f0[x]);
            split(dov[x][2], dov[x][3], f1[x]);
        }
        columns_times<HD, NI>(qs, f0, f1, G, lane);
#pragma unroll
        for (int x = 0; x < CG; ++x) {
            split(R[x][0], R[x][1], f0[x]);
            split(R[x][2], R[x][3], f1[x]);
        }
        columns_times<HD, NI>(ks, f0, f1, G, lane);
    }
    if (DSTATE_IN != nullptr) {
#pragma unroll
        for (int x = 0; x < CG; ++x)
#pragma unroll
            for (int u = 0; u < HD / 16; ++u) *(f32x4_t*)(DSTATE_IN + (bh * HD + v + 16 * x) * HD + 16 * u + g4) = G[x][u];
    }
}

// ---------------------------------------------------------------------------------------------------------------
template <int HD> struct GradLds {                 // byte offsets
    static constexpr int K_AT = 0, Q_AT = K_AT + DC * (HD + 4) * 4, GT_AT = Q_AT + DC * (HD + 4) * 4, DG_AT = GT_AT + DC * SQ * 4;
    static constexpr int DM_AT = DG_AT + DC * SQ * 4, ES_AT = DM_AT + DC * SQ * 4, F_AT = ES_AT + DC * SQ * 4;
    static constexpr int BYTES = F_AT + (6 * DC + 4 * DC + 4 * 3 * DC + 8) * 4;
};

// What is left of the gradient, chunk by chunk in parallel, eight waves to a workgroup: a wave owns a quarter of the columns of
// half of the rows of dQ and dK (a chunk's M and G are read twice, its other operands four times; with an eighth of the columns
// and all rows it was 177 instead of 152 us at 672 chunks of f32, head dim 128; four waves 154).  The 64x64 matrices are formed tile by tile
// and shared through LDS.  Bound by the f32 matrix instruction (6000 per chunk, a third of the time) and the waits between its
// phases: 672 chunks of f32, head dim 128, in 147 us, 432 of bf16, head dim 64, in 52.
template <int HD, typename T>
__global__ __launch_bounds__(512) void delta_grad_kernel(const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V,
                                                         Rows rq, Rows rk, Rows rv, const T* __restrict__ DO,
                                                         const float* __restrict__ ALPHA, const float* __restrict__ BETA,
                                                         const float* __restrict__ US, const float* __restrict__ RS,
                                                         const float* __restrict__ MS, const float* __restrict__ GS,
                                                         T* __restrict__ DQ, T* __restrict__ DK, float* __restrict__ DALPHA,
                                                         float* __restrict__ DBETA, uint8_t* __restrict__ BAD, int L, int H, int NC) {
    constexpr int CGS = 4, NR = 2, NN = HD / 64;   // column groups; row and column tiles of a wave
    typedef GradLds<HD> S;
    extern __shared__ __align__(16) char lds[];
    float(*ks)[HD + 4] = (float(*)[HD + 4])(lds + S::K_AT);
    float(*qs)[HD + 4] = (float(*)[HD + 4])(lds + S::Q_AT);
    float(*gt)[SQ] = (float(*)[SQ])(lds + S::GT_AT);           // decays, [j][i]
    float(*dg)[SQ] = (float(*)[SQ])(lds + S::DG_AT);           // gradients of the decays, [j][i]
    float(*dm)[SQ] = (float(*)[SQ])(lds + S::DM_AT);           // dP o g, [i][j]
    float(*es)[SQ] = (float(*)[SQ])(lds + S::ES_AT);           // E + E^T
    float* sa = (float*)(lds + S::F_AT);
    float *sb = sa + DC, *sg = sb + DC, *srv = sg + DC, *sky = srv + DC, *sdg = sky + DC;   // a, b, g, R.v, k.Y, d(g_i)
    float(*sdb)[DC] = (float(*)[DC])(sdg + DC);                // [jt][i]
    float(*red)[3][DC] = (float(*)[3][DC])(sdb + 4);           // [column group][q.X, k.Y, k.Z][i]
    float* fro = (float*)(red + CGS);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 15, g4 = (lane >> 4) * 4;
    const int cg = wave % CGS, r0 = wave / CGS * NR, col = 16 * NN * cg + m;     // this wave's first column, its first row tile
    int64_t b;
    int h, c;
    chunk_place(blockIdx.x, H, NC, b, h, c);
    const int64_t ci = (b * H + h) * NC + c;
    const int t0 = c * DC, left = L - t0 < DC ? L - t0 : DC;
    const int64_t first = ((b * L + t0) * H + h) * HD, dense = (int64_t)H * HD;
    rows_to_lds<HD, T, 512>(chunk_of(K + rk.at(b, L, t0, h, HD), rk.ld, left), ks, tid);
    rows_to_lds<HD, T, 512>(chunk_of(Q + rq.at(b, L, t0, h, HD), rq.ld, left), qs, tid);
    if (tid < DC) {
        const int64_t at = (b * L + t0 + tid) * H + h;
        sa[tid] = tid < left ? ALPHA[at] : 1.0f;
        sb[tid] = tid < left ? BETA[at] : 0.0f;
    }
    if (tid < 4 * DC) (&sdb[0][0])[tid] = 0.f;
    __syncthreads();
    if (wave == 0) chunk_decays(sa[lane], gt, lane);
    if (wave == 1) sg[lane] = chunk_prefix(sa[lane], lane);
    __syncthreads();
    const float* ub = US + ci * DC * HD;
    const float* rb = RS + ci * DC * HD;
    const ChunkOf<T> doc = chunk_of(DO + first, dense, left), vc = chunk_of(V + rv.at(b, L, t0, h, HD), rv.ld, left);
    // the 64x64 matrices: lane holds column i, rows j = 4g..4g+3 of a tile
    for (int tile = wave; tile < TRI; tile += 8) {
        const int it = tile < 1 ? 0 : tile < 3 ? 1 : tile < 6 ? 2 : 3, jt = tile - tri(it, 0);
        const int i = 16 * it + m, jr = 16 * jt + m;
        f32x4_t qk = {0.f, 0.f, 0.f, 0.f}, kk = qk, dp = qk, ru = qk;
#pragma unroll
        for (int u = 0; u < HD / 16; ++u) {
            const int at = 16 * u + g4;
            const f32x4_t kj = *(const f32x4_t*)&ks[jr][at], qi = *(const f32x4_t*)&qs[i][at], ki = *(const f32x4_t*)&ks[i][at],
                          uj = *(const f32x4_t*)(ub + jr * HD + at), ri = *(const f32x4_t*)(rb + i * HD + at),
                          oi = widen4(doc.raw(i, at));
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
    // X, Y, Z, <G, M> and R.v; two operand sets in turn
    f32x4_t X[NR][NN], Y[NR][NN], Z[NR][NN];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int x = 0; x < NN; ++x) X[n][x] = Y[n][x] = Z[n][x] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    const float* mb = MS + ci * HD * HD + col;
    const float* gb = GS + ci * HD * HD + col;
    float gm = 0.f, rdotv = 0.f;
    struct Operands {
        f32x4_t o[NR], r[NR], u[NR], rr, vv;
        float m[NN][4], g[NN][4];
    };
    auto load = [&](Operands& x, int u) {
        const int at = 16 * u + g4;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const int row = 16 * (r0 + n) + m;
            x.o[n] = widen4(doc.raw(row, at));
            x.r[n] = *(const f32x4_t*)(rb + row * HD + at);
            x.u[n] = *(const f32x4_t*)(ub + row * HD + at);
        }
#pragma unroll
        for (int n = 0; n < NN; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                x.m[n][r] = mb[(at + r) * HD + 16 * n];
                x.g[n][r] = gb[(at + r) * HD + 16 * n];
            }
        if (wave < 4) {
            x.rr = *(const f32x4_t*)(rb + (16 * wave + m) * HD + at);
            x.vv = widen4(vc.raw(16 * wave + m, at));
        }
    };
    auto use = [&](const Operands& x) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (wave < 4) rdotv = fmaf(x.rr[r], x.vv[r], rdotv);
#pragma unroll
            for (int y = 0; y < NN; ++y) {
                gm = fmaf(x.m[y][r], x.g[y][r], gm);
#pragma unroll
                for (int n = 0; n < NR; ++n) {
                    X[n][y] = mfma_f32(x.o[n][r], x.m[y][r], X[n][y]);
                    Y[n][y] = mfma_f32(x.r[n][r], x.m[y][r], Y[n][y]);
                    Z[n][y] = mfma_f32(x.u[n][r], x.g[y][r], Z[n][y]);
                }
            }
        }
    };
    Operands p0, p1;
    load(p0, 0);
#pragma unroll 1
    for (int u = 0; u < HD / 16; u += 2) {
        load(p1, u + 1);
        use(p0);
        if (u + 2 < HD / 16) load(p0, u + 2);
        use(p1);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) gm += __shfl_xor(gm, off);
    if (lane == 0) fro[wave] = r0 == 0 ? gm : 0.f;             // the other row half has the same columns
    rdotv += __shfl_xor(rdotv, 16);
    rdotv += __shfl_xor(rdotv, 32);
    if (wave < 4 && lane < 16) srv[16 * wave + m] = rdotv;
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = 16 * (r0 + n) + g4 + r;
            float x = 0.f, y = 0.f, z = 0.f;
#pragma unroll
            for (int w = 0; w < NN; ++w) {
                const float kv = ks[i][col + 16 * w];
                x = fmaf(qs[i][col + 16 * w], X[n][w][r], x);
                y = fmaf(kv, Y[n][w][r], y);
                z = fmaf(kv, Z[n][w][r], z);
            }
#pragma unroll
            for (int off = 1; off < 16; off <<= 1) {
                x += __shfl_xor(x, off);
                y += __shfl_xor(y, off);
                z += __shfl_xor(z, off);
            }
            if (m == 0) red[cg][0][i] = x, red[cg][1][i] = y, red[cg][2][i] = z;
            const float gi = sg[i];
#pragma unroll
            for (int w = 0; w < NN; ++w) {
                Z[n][w][r] = gt[i][DC - 1] * Z[n][w][r] - sb[i] * gi * Y[n][w][r];
                X[n][w][r] *= gi;
            }
        }
    __syncthreads();                               // dm, es, dg and the row sums are complete
    if (wave == 0) {                               // the last row of the decays carries k_j.Z_j and <G, M> too
        float x = 0.f, y = 0.f, z = 0.f, f = 0.f;
#pragma unroll
        for (int n = 0; n < CGS; ++n) x += red[n][0][lane], y += red[n][1][lane], z += red[n][2][lane];
#pragma unroll
        for (int n = 0; n < 8; ++n) f += fro[n];
        sky[lane] = y;
        sdg[lane] = x - sb[lane] * y + (lane == DC - 1 ? f : 0.f);
        if (lane < DC - 1) dg[lane][DC - 1] += z;
    }
#pragma unroll 1
    for (int jt = 0; jt < 4; ++jt) {
        f32x4_t ad[NR], ae[NR];
        float at[NR][4], bk[NN][4], bq[NN][4];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const int it = r0 + n;
            ae[n] = *(const f32x4_t*)&es[16 * it + m][16 * jt + g4];
            // dm holds the lower tiles only; the others' operands are zeros
            const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
            ad[n] = it >= jt ? *(const f32x4_t*)&dm[16 * it + m][16 * jt + g4] : zero;
#pragma unroll
            for (int r = 0; r < 4; ++r) at[n][r] = it <= jt ? dm[16 * jt + g4 + r][16 * it + m] : 0.f;
        }
#pragma unroll
        for (int x = 0; x < NN; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                bk[x][r] = ks[16 * jt + g4 + r][col + 16 * x];
                bq[x][r] = qs[16 * jt + g4 + r][col + 16 * x];
            }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int x = 0; x < NN; ++x) {
                    X[n][x] = mfma_f32(ad[n][r], bk[x][r], X[n][x]);
                    Z[n][x] = mfma_f32(at[n][r], bq[x][r], Z[n][x]);
                    Z[n][x] = mfma_f32(ae[n][r], bk[x][r], Z[n][x]);
                }
    }
    const ChunkOf<T> dqc = chunk_of((const T*)DQ + first, dense, left), dkc = chunk_of((const T*)DK + first, dense, left);
    float seen = 0.f;                              // NaN with any result that is not finite
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int x = 0; x < NN; ++x) {
                const int i = 16 * (r0 + n) + g4 + r;
                dqc.put(i, col + 16 * x, X[n][x][r]);
                dkc.put(i, col + 16 * x, Z[n][x][r]);
                seen = fmaf(X[n][x][r], 0.f, fmaf(Z[n][x][r], 0.f, seen));
            }
    // da_t: D[t][i] = sum_{j < t} g_{t-1,j} d(g_ij) + g_{t-1} d(g_i), weighted with g_it and summed over i >= t.  The first four
    // waves take a row tile of t each.
    __syncthreads();
    if (wave < 4) {
        const int t = 16 * wave + m;
        float da[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            if (it < wave) continue;
            const int i = 16 * it + m;
            f32x4_t d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int jt = 0; jt < 4; ++jt) {
                if (jt > wave) continue;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = 16 * jt + g4 + r;
                    const float left_op = j < t ? gt[j][t - 1] : 0.f;
                    d = mfma_f32(left_op, dg[j][i], d);
                }
            }
            const float dgi = sdg[i];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int tt = 16 * wave + g4 + r;
                const float before = tt > 0 ? sg[tt - 1] : 1.f;
                if (i >= tt) da[r] = fmaf(gt[tt][i], fmaf(before, dgi, d[r]), da[r]);
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
            for (int off = 1; off < 16; off <<= 1) da[r] += __shfl_xor(da[r], off);
            const int tt = 16 * wave + g4 + r;
            if (m == 0 && tt < left) DALPHA[(b * L + t0 + tt) * H + h] = da[r];
            seen = fmaf(da[r], 0.f, seen);
        }
        const float db = sdb[0][t] + sdb[1][t] + sdb[2][t] + sdb[3][t] + srv[t] - sg[t] * sky[t];
        if (lane < 16 && t < left) DBETA[(b * L + t0 + t) * H + h] = db;
        seen = fmaf(db, 0.f, seen);
    }
    const bool bad = __any(seen != seen);
    if (lane == 0) BAD[ci * 8 + wave] = bad;
}

template <typename T> struct elem;
template <> struct elem<float> {
    static VA_DEVINL f32x4_t load4(const float* p) { return *(const f32x4_t*)p; }
    static VA_DEVINL float get(const float* p) { return *p; }
    static VA_DEVINL void put(float* p, float x) { *p = x; }
};
template <> struct elem<bf16_t> {
    static VA_DEVINL f32x4_t load4(const bf16_t* p) { return widen4(*(const u32x2_t*)p); }
    static VA_DEVINL float get(const bf16_t* p) { return bf16_to_f32(*p); }
    static VA_DEVINL void put(bf16_t* p, float x) { *p = f32_to_bf16(x); }      // the output's own type: one rounding
};

// ---------------------------------------------------------------------------------------------------------------
// The gradients of a head with a result that is not finite, token by token: there a product with a zero of the chunked form
// (a weight above the diagonal, a row behind the sequence) has turned a bad number of one token into bad gradients of others.
// A bad dv or state gradient always shows in dq, dk or a gate of its chunk too, which R and G enter.  One workgroup per head,
// HD / 16 waves of 16 rows of the state S and of G = dL/dS, four lanes to a row; with P = S_{t-1}, u = b (v - a P k), walking
// back from the last token
//     dq = S_t^T do,   G += do q^T,   dv = b G k,   da = <G, P - b (P k) k^T>,   db = (G k).(v - a P k),
//     dk = G^T u - a b P^T (G k),     G <- a (G - b (G k) k^T).
// P is formed anew from the chunk's first state for each token (GS, whose chunked contents are of no use, holds those): rare, so
// this trades time for memory (32 heads x 1290 tokens of f32, head dim 128, all bad: 37 ms).  Heads whose results are finite
// leave at once (a launch of 4-5 us behind the others).
template <int HD, typename T>
__global__ __launch_bounds__(4 * HD) void delta_grad_by_token_kernel(const T* __restrict__ Q, const T* __restrict__ K,
                                                                     const T* __restrict__ V, Rows rq, Rows rk, Rows rv,
                                                                     const T* __restrict__ DO, const float* __restrict__ ALPHA,
                                                                     const float* __restrict__ BETA, const float* __restrict__ STATE_IN,
                                                                     const float* __restrict__ DSTATE, const uint64_t* __restrict__ BAD,
                                                                     T* __restrict__ DQ, T* __restrict__ DK, T* __restrict__ DV,
                                                                     float* __restrict__ DALPHA, float* __restrict__ DBETA,
                                                                     float* __restrict__ DSTATE_IN, float* GS, int L, int H, int NC) {
    constexpr int W = HD / 16, N = HD / 16;        // waves; groups of four columns of a lane
    __shared__ float part[2][W][HD];               // column sums of a wave's rows: dq, dk
    __shared__ float gate[2][W];                   // da, db
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = 16 * wave + (lane & 15), col = (lane >> 4) * (HD / 4);
    const int64_t bh = blockIdx.x, b = bh / H, h = bh % H;
    int any = 0;
    for (int c = tid; c < NC; c += 4 * HD) any |= BAD[bh * NC + c] != 0;
    if (!__syncthreads_or(any)) return;
    const T *q = Q + rq.at(b, L, 0, h, HD), *k = K + rk.at(b, L, 0, h, HD), *v = V + rv.at(b, L, 0, h, HD);
    const int64_t first = b * L * H + h;
    const int64_t at = bh * HD * HD + row * HD + col;              // this lane's part of a state
    float* starts = GS + bh * NC * HD * HD + row * HD + col;
    f32x4_t S[N], G[N], kt[N], qt[N];
    auto over_row = [](float x) {
        x += __shfl_xor(x, 16);
        return x + __shfl_xor(x, 32);
    };
    auto over_rows = [](float x) {
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) x += __shfl_xor(x, off);
        return x;
    };
    auto row_of = [&](const T* p, int64_t ld, int t, f32x4_t (&to)[N]) {
#pragma unroll
        for (int n = 0; n < N; ++n) to[n] = elem<T>::load4(p + t * ld + col + 4 * n);
    };
    auto dot = [&](const f32x4_t (&x)[N], const f32x4_t (&y)[N]) {
        float d = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) d = fmaf(x[n][r], y[n][r], d);
        return over_row(d);
    };
    auto forward = [&](int t) {                    // S_{t-1} -> S_t
        const float a = ALPHA[first + (int64_t)t * H], bt = BETA[first + (int64_t)t * H];
        row_of(k, rk.ld, t, kt);
        const float u = bt * (elem<T>::get(v + t * rv.ld + row) - a * dot(S, kt));
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[n][r] = fmaf(u, kt[n][r], a * S[n][r]);
    };
#pragma unroll
    for (int n = 0; n < N; ++n) {
        S[n] = G[n] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
        if (STATE_IN != nullptr) S[n] = *(const f32x4_t*)(STATE_IN + at + 4 * n);
        if (DSTATE != nullptr) G[n] = *(const f32x4_t*)(DSTATE + at + 4 * n);
    }
#pragma unroll 1
    for (int c = 0; c < NC; ++c) {
#pragma unroll
        for (int n = 0; n < N; ++n) *(f32x4_t*)(starts + (int64_t)c * HD * HD + 4 * n) = S[n];
        if (c + 1 < NC)
#pragma unroll 1
            for (int t = c * DC; t < (c + 1) * DC; ++t) forward(t);
    }
#pragma unroll 1
    for (int t = L - 1; t >= 0; --t) {
        const int c = t / DC;
#pragma unroll
        for (int n = 0; n < N; ++n) S[n] = *(const f32x4_t*)(starts + (int64_t)c * HD * HD + 4 * n);
#pragma unroll 1
        for (int s = c * DC; s < t; ++s) forward(s);
        const int64_t token = first + (int64_t)t * H;
        const float a = ALPHA[token], bt = BETA[token];
        row_of(k, rk.ld, t, kt);
        row_of(q, rq.ld, t, qt);
        const float dov = elem<T>::get(DO + token * HD + row), sk = dot(S, kt), w = elem<T>::get(v + t * rv.ld + row) - a * sk, u = bt * w;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float x = over_rows(fmaf(u, kt[n][r], a * S[n][r]) * dov);
                if ((lane & 15) == 0) part[0][wave][col + 4 * n + r] = x;
                G[n][r] = fmaf(dov, qt[n][r], G[n][r]);
            }
        const float gk = dot(G, kt);
        float da = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                da = fmaf(G[n][r], fmaf(-bt * sk, kt[n][r], S[n][r]), da);
                const float x = over_rows(fmaf(G[n][r], u, -(a * bt) * gk * S[n][r]));
                if ((lane & 15) == 0) part[1][wave][col + 4 * n + r] = x;
                G[n][r] = a * fmaf(-bt * gk, kt[n][r], G[n][r]);
            }
        if (lane < 16) elem<T>::put(DV + token * HD + row, bt * gk);
        da = over_row(over_rows(da));
        const float db = over_rows(gk * w);        // the same in the four lanes of a row
        if (lane == 0) gate[0][wave] = da, gate[1][wave] = db;
        __syncthreads();
        if (tid < 2 * HD) {
            float x = 0.f;
#pragma unroll
            for (int n = 0; n < W; ++n) x += part[tid / HD][n][tid % HD];
            elem<T>::put((tid < HD ? DQ : DK) + token * HD + tid % HD, x);
        }
        if (tid < 2) {
            float x = 0.f;
#pragma unroll
            for (int n = 0; n < W; ++n) x += gate[tid][n];
            (tid == 0 ? DALPHA : DBETA)[token] = x;
        }
        __syncthreads();                           // the sums have been read
    }
    if (DSTATE_IN != nullptr) {
#pragma unroll
        for (int n = 0; n < N; ++n) *(f32x4_t*)(DSTATE_IN + at + 4 * n) = G[n];
    }
}

// ---------------------------------------------------------------------------------------------------------------
// One token: S <- a S + u k^T, u = b (v - a S k), o = S q = a (S_old q) + u (k.q).  The state is read and written once and
// its rows are independent: HD/4 lanes hold a row (16 bytes each), the row's two dot products are summed across them.  Bound by
// the state's bytes: 2048 heads of 128 in 57 us, 4.8 TB/s (44 where the last-level cache still holds the states);
// 8 heads in 3 us.
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
    const f32x4_t k4 = elem<T>::load4(K + b * ldk + h * HD + 4 * lane), q4 = elem<T>::load4(Q + b * ldq + h * HD + 4 * lane);
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
                     d.B * d.H * d.chunks() < (1ll << 31) && d.ldq < (1 << 22) && d.ldk < (1 << 22) && d.ldv < (1 << 22),
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

// A workspace in pieces of 16 bytes.
struct Pieces {
    char* at;
    template <typename E> E* take(int64_t n) {
        E* p = (E*)at;
        at += (n * (int64_t)sizeof(E) + 15) / 16 * 16;
        return p;
    }
};

// What a forward pass leaves for its gradient, and what it needs itself
template <typename T> struct Work {
    bf16_t *tf, *pf, *tt, *pt;
    float *gam, *us, *ms;
};
template <typename T> int64_t operand_numbers(const DeltaArgs& d, int parts_) { return d.B * d.H * d.chunks() * BLK * BFRAG * parts_; }
template <typename T> void take_own(const DeltaArgs& d, Pieces& p, Work<T>& w) {
    w.tf = p.template take<bf16_t>(operand_numbers<T>(d, parts<T>::MID));
    w.pf = p.template take<bf16_t>(operand_numbers<T>(d, parts<T>::OUT));
}
template <typename T> void take_kept(const DeltaArgs& d, Pieces& p, Work<T>& w) {
    const int64_t n = d.B * d.H * d.chunks();
    w.gam = p.template take<float>(n * 2 * DC);
    w.tt = p.template take<bf16_t>(operand_numbers<T>(d, parts<T>::MID));
    w.pt = p.template take<bf16_t>(operand_numbers<T>(d, parts<T>::MID));
    w.us = p.template take<float>(n * DC * d.hd);
    w.ms = p.template take<float>(n * d.hd * d.hd);
}

template <int HD, typename T, bool TRAIN>
int launch_prep(const DeltaArgs& d, const Work<T>& w, hipStream_t stream) {
    hipLaunchKernelGGL((delta_prep_kernel<HD, T, TRAIN>), dim3((unsigned)(d.B * d.H * d.chunks())), dim3(256), 0, stream,
                       (const T*)d.q, (const T*)d.k, Rows{d.ldq}, Rows{d.ldk}, d.alpha, d.beta, w.tf, w.pf, w.tt, w.pt, w.gam,
                       (int)d.L, (int)d.H, (int)d.chunks());
    VA_CHECK_LAUNCH("va_gated_delta (decays)");
    return VA_OK;
}

// The scans run four waves to a workgroup, one per SIMD.  Head dim 128 has eight groups of 16 columns: with one to a wave a
// head takes two workgroups, which is shortest while there is a CU for each; from there on two to a wave halve the LDS reads
// per product (the left operands serve both).
constexpr int SCAN_W = 4;
template <int HD> bool wide_scan(const DeltaArgs& d) { return HD == 128 && d.B * d.H > 128; }

template <int HD, typename T, int CG, bool OUT, bool SAVE>
int launch_scan(const DeltaArgs& d, const Work<T>& w, const float* state_in, void* out, float* state_out, hipStream_t stream) {
    constexpr int lds = ChunkRows<HD, T, SCAN_W, OUT, parts<T>::MID, OUT ? parts<T>::OUT : 0, CG == 1>::LDS;
    const auto fn = delta_scan_kernel<HD, T, SCAN_W, CG, OUT, SAVE>;
    VA_TRY(reserve_lds("va_gated_delta", (const void*)fn, lds));
    hipLaunchKernelGGL(fn, dim3((unsigned)(d.B * d.H * (HD / 16 / (SCAN_W * CG)))), dim3(64 * SCAN_W), lds, stream, (const T*)d.q,
                       (const T*)d.k, (const T*)d.v, Rows{d.ldq}, Rows{d.ldk}, Rows{d.ldv}, d.alpha, d.beta, w.tf, w.pf, w.gam, state_in,
                       (T*)out, state_out, w.us, w.ms, (int)d.L, (int)d.H, (int)d.chunks());
    VA_CHECK_LAUNCH("va_gated_delta (scan)");
    return VA_OK;
}
template <int HD, typename T, bool OUT, bool SAVE>
int run_scan(const DeltaArgs& d, const Work<T>& w, const float* state_in, void* out, float* state_out, hipStream_t stream) {
    if (wide_scan<HD>(d)) return launch_scan<HD, T, HD / 64, OUT, SAVE>(d, w, state_in, out, state_out, stream);
    return launch_scan<HD, T, 1, OUT, SAVE>(d, w, state_in, out, state_out, stream);
}

template <int HD, typename T, int CG>
int launch_rscan(const DeltaArgs& d, const Work<T>& w, const void* d_out, const float* d_state, void* dv, float* d_state_in, float* rs,
                 float* gs, hipStream_t stream) {
    constexpr int lds = ChunkRows<HD, T, SCAN_W, true, parts<T>::MID, parts<T>::MID, CG == 1>::LDS;
    const auto fn = delta_rscan_kernel<HD, T, SCAN_W, CG>;
    VA_TRY(reserve_lds("va_gated_delta_bwd", (const void*)fn, lds));
    hipLaunchKernelGGL(fn, dim3((unsigned)(d.B * d.H * (HD / 16 / (SCAN_W * CG)))), dim3(64 * SCAN_W), lds, stream, (const T*)d.q,
                       (const T*)d.k, Rows{d.ldq}, Rows{d.ldk}, (const T*)d_out, d.beta, w.tt, w.pt, w.gam, d_state, (T*)dv, d_state_in,
                       rs, gs, (int)d.L, (int)d.H, (int)d.chunks());
    VA_CHECK_LAUNCH("va_gated_delta_bwd (scan)");
    return VA_OK;
}

// bytes of one chunk's share of the forward's own workspace, of what it keeps, and of the gradient's own
constexpr int64_t OPERAND_BYTES = BLK * BFRAG * 2;
int64_t own_chunk_bytes() { return 6 * OPERAND_BYTES + 2 * DC * 4; }
int64_t kept_chunk_bytes(int64_t hd) { return 2 * DC * 4 + 6 * OPERAND_BYTES + DC * hd * 4 + hd * hd * 4; }
int64_t bwd_chunk_bytes(int64_t hd) { return DC * hd * 4 + hd * hd * 4 + 16; }      // 8 of the 16: a flag per wave

template <int HD, typename T>
int delta_fwd(const DeltaArgs& d, const float* state_in, void* out, float* state_out, float* ws, float* kept, hipStream_t stream) {
    Work<T> w = {};
    Pieces own = {(char*)ws};
    take_own(d, own, w);
    if (kept != nullptr) {
        Pieces k = {(char*)kept};
        take_kept(d, k, w);
        VA_TRY((launch_prep<HD, T, true>(d, w, stream)));
        return run_scan<HD, T, true, true>(d, w, state_in, out, state_out, stream);
    }
    w.gam = own.template take<float>(d.B * d.H * d.chunks() * 2 * DC);
    VA_TRY((launch_prep<HD, T, false>(d, w, stream)));
    return run_scan<HD, T, true, false>(d, w, state_in, out, state_out, stream);
}

template <int HD, typename T>
int delta_bwd(const DeltaArgs& d, const void* d_out, const float* d_state, const float* state_in, void* dq, void* dk, void* dv,
              float* dalpha, float* dbeta, float* d_state_in, float* ws, const float* kept, hipStream_t stream) {
    const int64_t n = d.B * d.H * d.chunks();
    Work<T> w = {};
    Pieces own = {(char*)ws};
    float *rs = own.take<float>(n * DC * HD), *gs = own.take<float>(n * HD * HD);
    uint8_t* bad = own.take<uint8_t>(n * 8);
    if (kept != nullptr) {
        Pieces k = {(char*)kept};
        take_kept(d, k, w);
    } else {
        take_kept(d, own, w);
        take_own(d, own, w);
        VA_TRY((launch_prep<HD, T, true>(d, w, stream)));
        VA_TRY((run_scan<HD, T, false, true>(d, w, state_in, nullptr, nullptr, stream)));
    }
    if (wide_scan<HD>(d)) VA_TRY((launch_rscan<HD, T, HD / 64>(d, w, d_out, d_state, dv, d_state_in, rs, gs, stream)));
    else VA_TRY((launch_rscan<HD, T, 1>(d, w, d_out, d_state, dv, d_state_in, rs, gs, stream)));
    constexpr int lds = GradLds<HD>::BYTES;
    const auto fn = delta_grad_kernel<HD, T>;
    VA_TRY(reserve_lds("va_gated_delta_bwd", (const void*)fn, lds));
    hipLaunchKernelGGL(fn, dim3((unsigned)n), dim3(512), lds, stream, (const T*)d.q, (const T*)d.k, (const T*)d.v, Rows{d.ldq},
                       Rows{d.ldk}, Rows{d.ldv}, (const T*)d_out, d.alpha, d.beta, w.us, rs, w.ms, gs, (T*)dq, (T*)dk, dalpha, dbeta, bad,
                       (int)d.L, (int)d.H, (int)d.chunks());
    VA_CHECK_LAUNCH("va_gated_delta_bwd (gradients)");
    hipLaunchKernelGGL((delta_grad_by_token_kernel<HD, T>), dim3((unsigned)(d.B * d.H)), dim3(4 * HD), 0, stream, (const T*)d.q,
                       (const T*)d.k, (const T*)d.v, Rows{d.ldq}, Rows{d.ldk}, Rows{d.ldv}, (const T*)d_out, d.alpha, d.beta, state_in,
                       d_state, (const uint64_t*)bad, (T*)dq, (T*)dk, (T*)dv, dalpha, dbeta, d_state_in, gs, (int)d.L, (int)d.H,
                       (int)d.chunks());
    VA_CHECK_LAUNCH("va_gated_delta_bwd (token by token)");
    return VA_OK;
}

}  // namespace

static int64_t delta_floats(int64_t B, int64_t L, int64_t H, int64_t hd, int64_t chunk_bytes) {
    if (B <= 0 || L <= 0 || H <= 0 || (hd != 64 && hd != 128)) return 0;
    return B * H * ((L + DC - 1) / DC) * chunk_bytes / 4;
}
extern "C" int64_t va_gated_delta_fwd_workspace_floats(int64_t B, int64_t L, int64_t H, int64_t hd) {
    return delta_floats(B, L, H, hd, own_chunk_bytes());
}
extern "C" int64_t va_gated_delta_kept_floats(int64_t B, int64_t L, int64_t H, int64_t hd) {
    return delta_floats(B, L, H, hd, kept_chunk_bytes(hd));
}
extern "C" int64_t va_gated_delta_bwd_workspace_floats(int64_t B, int64_t L, int64_t H, int64_t hd, int have_kept) {
    return delta_floats(B, L, H, hd, bwd_chunk_bytes(hd) + (have_kept ? 0 : own_chunk_bytes() + kept_chunk_bytes(hd)));
}

extern "C" int va_gated_delta_fwd(const void* q, const void* k, const void* v, int64_t ldq, int64_t ldk, int64_t ldv, int is_bf16,
                                  const float* alpha, const float* beta, const float* state_in, void* out, float* state_out,
                                  float* workspace, float* kept, int64_t B, int64_t L, int64_t H, int64_t hd, hipStream_t stream) {
    const DeltaArgs d = {q, k, v, ldq, ldk, ldv, alpha, beta, B, L, H, hd, is_bf16 != 0};
    VA_TRY(delta_check("va_gated_delta_fwd", d));
    VA_CHECK_ARG(out && state_out && workspace, "va_gated_delta_fwd: null operand");
    VA_CHECK_ARG(((uintptr_t)state_in | (uintptr_t)state_out | (uintptr_t)workspace | (uintptr_t)kept) % 16 == 0,
                 "va_gated_delta_fwd: misaligned state or workspace");
    if (hd == 128)
        return d.bf16 ? delta_fwd<128, bf16_t>(d, state_in, out, state_out, workspace, kept, stream)
                      : delta_fwd<128, float>(d, state_in, out, state_out, workspace, kept, stream);
    return d.bf16 ? delta_fwd<64, bf16_t>(d, state_in, out, state_out, workspace, kept, stream)
                  : delta_fwd<64, float>(d, state_in, out, state_out, workspace, kept, stream);
}

extern "C" int va_gated_delta_bwd(const void* d_out, const float* d_state, const void* q, const void* k, const void* v, int64_t ldq,
                                  int64_t ldk, int64_t ldv, int is_bf16, const float* alpha, const float* beta,
                                  const float* state_in, void* dq, void* dk, void* dv, float* dalpha, float* dbeta,
                                  float* d_state_in, float* workspace, const float* kept, int64_t B, int64_t L, int64_t H, int64_t hd,
                                  hipStream_t stream) {
    const DeltaArgs d = {q, k, v, ldq, ldk, ldv, alpha, beta, B, L, H, hd, is_bf16 != 0};
    VA_TRY(delta_check("va_gated_delta_bwd", d));
    VA_CHECK_ARG(d_out && dq && dk && dv && dalpha && dbeta && workspace, "va_gated_delta_bwd: null operand");
    VA_CHECK_ARG(((uintptr_t)state_in | (uintptr_t)d_state | (uintptr_t)d_state_in | (uintptr_t)workspace | (uintptr_t)kept) % 16 == 0 &&
                     (uintptr_t)d_out % (d.bf16 ? 8 : 16) == 0,       // four elements of d_out are read at a time
                 "va_gated_delta_bwd: misaligned state, gradient or workspace");
    if (hd == 128)
        return d.bf16 ? delta_bwd<128, bf16_t>(d, d_out, d_state, state_in, dq, dk, dv, dalpha, dbeta, d_state_in, workspace, kept, stream)
                      : delta_bwd<128, float>(d, d_out, d_state, state_in, dq, dk, dv, dalpha, dbeta, d_state_in, workspace, kept, stream);
    return d.bf16 ? delta_bwd<64, bf16_t>(d, d_out, d_state, state_in, dq, dk, dv, dalpha, dbeta, d_state_in, workspace, kept, stream)
                  : delta_bwd<64, float>(d, d_out, d_state, state_in, dq, dk, dv, dalpha, dbeta, d_state_in, workspace, kept, stream);
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
