// Key/value cache in 8 bits and the attention that reads it.
//
// Cache of a stream and head: tokens [cap][hd] as e4m3 codes, one f32 scale per block of 64 tokens; the block that is not
// full yet lies beside it in bf16 [64][hd], so what a block's codes are depends on its 64 tokens alone and not on how many
// came in one call.  A scale is the smallest power of two (2^-100 at least) that brings the block's largest finite magnitude
// to 448 or below: a code times its scale is then a bf16 number exactly, and the only rounding of a key or value is the one
// to its code, half a step: 2^-4 of the value at most, or 2^-10 of the scale for values below 2^-6 of it, where e4m3's steps no
// longer shrink (elements under 2^-10 of the scale become zero).  Infinite elements become NaN.
//
// Attention: query row r of a key/value head = (query r / G, head r % G of its G query heads); query i of a stream with
// `len` tokens of which `nb` are new stands at p = len - nb + i and sees keys j < limit: len, or with T tokens to a timestep
// min(len, (p / T + 1) T).  One pass over the keys with the running maximum and sum of the softmax, in tiles of one block:
//     S^T = K Q^T (keys are matrix rows: a lane ends up with four keys of one query),   O^T += V^T P^T
// on the bf16 matrix instruction with f32 accumulation; P (f32, unrounded in the sum) is rounded to bf16 as its operand, by
// at most 2^-8 of each weight, once.  The accumulator order of S^T is the operand order of P^T for a permutation of the keys
// that V's transposed LDS reads follow, so P never leaves its registers.
#include "common.h"

namespace {

constexpr int KB = 64;                       // tokens of a block = keys of a tile
constexpr float LOG2E = 1.44269504088896341f;
constexpr float NEG_INF = -__builtin_inff();

struct Cache {
    const uint8_t *k8, *v8;
    const float *ks, *vs;
    const bf16_t *ko, *vo;
    const int32_t* lengths;
    int64_t cap;
};

// ---- append ---------------------------------------------------------------------------------------------------
// One workgroup per block that the call touches, head and stream, keys or values.  Where the open block fills up and a
// later one is left open, one workgroup does both: it has read the open block before it writes the new one over it.  Bound by
// launches for single tokens (3 us, 5 where a block fills up), by memory for long calls (16 streams x 1290 tokens x 8 heads of
// 128: 28 us, 4.6 TB/s; 258 tokens behind them 11 us).
template <int HD>
__global__ __launch_bounds__(256) void kv8_append_kernel(const bf16_t* __restrict__ K, const bf16_t* __restrict__ V, int64_t ldk,
                                                         int64_t ldv, int64_t bsk, int64_t bsv, const int32_t* __restrict__ NEW,
                                                         int n, uint8_t* __restrict__ K8, uint8_t* __restrict__ V8,
                                                         float* __restrict__ KS, float* __restrict__ VS, bf16_t* __restrict__ KO,
                                                         bf16_t* __restrict__ VO, const int32_t* __restrict__ LENGTHS, int64_t cap,
                                                         int H) {
    constexpr int N = KB * HD / 8 / 256;     // 16-byte pieces per thread
    __shared__ uint32_t wmax[4];
    const int tid = threadIdx.x;
    const bool val = (int)blockIdx.y >= H;
    const int64_t h = val ? blockIdx.y - H : blockIdx.y, b = blockIdx.z, bh = b * H + h;
    const int64_t len = LENGTHS[b];
    int64_t nb = NEW != nullptr ? NEW[b] : n;
    nb = nb < 0 ? 0 : nb > n ? n : nb;
    const int64_t total = len + nb < cap ? len + nb : cap;
    const int64_t first = len / KB, block = first + blockIdx.x, start = block * KB;
    if (len < 0 || start >= total) return;
    const bool whole = start + KB <= total;
    if (!whole && blockIdx.x > 0) return;    // the first workgroup writes the block that stays open
    const bf16_t* src = (val ? V + b * bsv : K + b * bsk) + h * HD;
    const int64_t ld = val ? ldv : ldk;
    bf16_t* open = (val ? VO : KO) + bh * KB * HD;
    if (whole) {                             // (a block that stays open is not read)
        u32x4_t x[N];
        uint32_t big = 0;
#pragma unroll
        for (int p = 0; p < N; ++p) {
            const int idx = p * 256 + tid, row = idx / (HD / 8), c = (idx % (HD / 8)) * 8;
            const int64_t t = start + row;
            x[p] = t < len ? *(const u32x4_t*)(open + row * HD + c) : *(const u32x4_t*)(src + (t - len) * ld + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) {    // magnitudes of finite bf16 numbers order like their bits
                const uint32_t lo = x[p][e] & 0x7fffu, hi = (x[p][e] >> 16) & 0x7fffu;
                big = max(big, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
            }
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) big = max(big, (uint32_t)__shfl_xor((int)big, off));
        if ((tid & 63) == 0) wmax[tid >> 6] = big;
        __syncthreads();
        big = max(max(wmax[0], wmax[1]), max(wmax[2], wmax[3]));
        int e = (int)(big >> 7) - 127 - 8 + ((big & 0x7fu) > 96u);           // 448 = 1.75 * 2^8, 1.75 = 1 + 96 / 128
        e = big == 0 ? 0 : e < -100 ? -100 : e;
        const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
        uint8_t* dst = (val ? V8 : K8) + (bh * cap + start) * HD;
#pragma unroll
        for (int p = 0; p < N; ++p) {
            const int idx = p * 256 + tid;
            float f[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                f[2 * k] = __uint_as_float(x[p][k] << 16) * inv;
                f[2 * k + 1] = __uint_as_float(x[p][k] & 0xffff0000u) * inv;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = fabsf(f[k]) <= 448.f ? f[k] : __builtin_nanf("");
            u32x2_t out;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * k], f[4 * k + 1], 0, false);
                out[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * k + 2], f[4 * k + 3], w, true);
            }
            *(u32x2_t*)(dst + (int64_t)idx * 8) = out;
        }
        if (tid == 0) (val ? VS : KS)[bh * (cap / KB) + block] = __uint_as_float((uint32_t)(127 + e) << 23);
    }
    if (blockIdx.x > 0) return;
    __syncthreads();                         // every thread has read the open block
    const int64_t last = total / KB * KB;    // first token of the block that stays open
#pragma unroll
    for (int p = 0; p < N; ++p) {
        const int idx = p * 256 + tid, row = idx / (HD / 8), c = (idx % (HD / 8)) * 8;
        const int64_t t = last + row;
        if (t >= len && t < total) *(u32x4_t*)(open + row * HD + c) = *(const u32x4_t*)(src + (t - len) * ld + c);
    }
}

__global__ __launch_bounds__(256) void kv8_advance_kernel(int32_t* __restrict__ LENGTHS, const int32_t* __restrict__ NEW, int n,
                                                          int64_t cap, int B) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b >= B || LENGTHS[b] < 0) return;
    int64_t nb = NEW != nullptr ? NEW[b] : n;
    nb = nb < 0 ? 0 : nb > n ? n : nb;
    const int64_t total = LENGTHS[b] + nb;
    LENGTHS[b] = (int32_t)(total < cap ? total : cap);
}

// ---- attention ------------------------------------------------------------------------------------------------
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2v_t;

// 16 bytes at `at` of a span that starts at a wave-uniform address; zeros behind its end
VA_DEVINL u32x4_t span16(const void* base, int bytes, int at) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, bytes, 0x00020000);
    return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0));
}

// eight codes -> eight bf16 numbers, times the block's scale: exact
VA_DEVINL u32x4_t widen8(uint32_t lo, uint32_t hi, float scale) {
    u32x4_t r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
    return r;
}
VA_DEVINL bf16x8_t as_frag(u32x4_t v) { return __builtin_bit_cast(bf16x8_t, v); }
VA_DEVINL bool any_nonfinite(u32x4_t v) {
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) bad |= (v[e] & 0x7f80u) == 0x7f80u || (v[e] & 0x7f800000u) == 0x7f800000u;
    return bad;
}

struct AttnArgs {
    const bf16_t* q;
    int64_t ldq, bsq;
    const int32_t* new_;
    bf16_t* out;
    float *part_o, *part_ml;                 // [split][B * Hkv * rows][hd], [..][2]
    int B, n, H, G, tpt, splits, tile;       // tile: query rows of a workgroup
    float scale2;                            // softmax scale * log2(e)
};

// keys seen by query i of stream b
VA_DEVINL int key_limit(const AttnArgs& a, int i, int len, int nb) {
    const int p = len - nb + i;
    if (i >= nb || p < 0) return 0;
    if (a.tpt == 0) return len;
    const int64_t end = ((int64_t)(p / a.tpt) + 1) * a.tpt;
    return end < len ? (int)end : len;
}
VA_DEVINL void stream_lengths(const AttnArgs& a, const Cache& c, int b, int& len, int& nb) {
    len = c.lengths[b];
    len = len < 0 ? 0 : len > c.cap ? (int)c.cap : len;
    nb = a.new_ != nullptr ? a.new_[b] : a.n;
    nb = nb < 0 ? 0 : nb > a.n ? a.n : nb;
}

// Maximum over the four lane groups (lanes 16 and 32 apart): swapping rows of a register with its copy leaves one partner's
// value in each, without the LDS round trip of a shuffle.
VA_DEVINL float groups_max(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// What a part's sums count in the whole: 0 where the maximum ignored all it saw, nothing or NaN alone.  The sums are added with
// that factor too: those of nothing are zeros, and a NaN stays NaN.
VA_DEVINL float part_factor(float mx, float top, float scale2) {
#pragma clang fp contract(off)
    return mx == NEG_INF ? 0.f : __builtin_amdgcn_exp2f(mx * scale2 - top * scale2);     // bases rounded as in tile_softmax
}

// Softmax weights of one 64-key tile for 16 queries and the rescaled running state.  s[kt] = raw scores of keys 16 kt + 4 g + r;
// pf[u] = the tile's P^T operand for keys 32 u ..+31.  The running maximum is one of raw scores (the scale is positive), the
// scale goes into the exponent's multiply-add.  The sums so far stand on the rounded product of the old maximum and the scale,
// so the factor to the new base is formed from two such products: exactly 1 while the maximum stays, however many tiles follow
// (a multiply-add in its place left the product's rounding error in it, once per tile).
template <bool MASK>
VA_DEVINL float tile_softmax(f32x4_t (&s)[4], int key0, int g4, int limit, float scale2, float& mx, float& sum, bf16x8_t (&pf)[2]) {
#pragma clang fp contract(off)
    float top = NEG_INF;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (MASK) s[kt][r] = key0 + 16 * kt + g4 + r < limit ? s[kt][r] : NEG_INF;
            top = fmaxf(top, s[kt][r]);
        }
    top = groups_max(top);
    const float now = fmaxf(mx, top);
    const float base = now == NEG_INF ? 0.f : now * scale2;     // nothing seen yet: every weight is exp2(-inf) = 0
    const float fade = __builtin_amdgcn_exp2f(mx * scale2 - base);
    mx = now;
    float add = 0.f;
    uint32_t pk[4][2];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            s[kt][r] = __builtin_amdgcn_exp2f(fmaf(s[kt][r], scale2, -base));
            add += s[kt][r];
        }
        pk[kt][0] = pack_bf16x2(s[kt][0], s[kt][1]);
        pk[kt][1] = pack_bf16x2(s[kt][2], s[kt][3]);
    }
    sum = fmaf(sum, fade, add);                                 // this lane's share: its own keys
#pragma unroll
    for (int u = 0; u < 2; ++u) pf[u] = as_frag((u32x4_t){pk[2 * u][0], pk[2 * u][1], pk[2 * u + 1][0], pk[2 * u + 1][1]});
    return fade;
}

// V^T operand of columns 16 ht..+15 for keys 32 u..+31, from a tile in LDS (rows of `stride` bytes)
VA_DEVINL bf16x8_t v_frag(const char* vt, int stride, int ht, int u, int lane) {
    const int q = (lane & 15) >> 2, p = lane & 3, g = lane >> 4;
    const char* at = vt + (32 * u + 4 * g + q) * stride + (16 * ht + 4 * p) * 2;
    return join_tr(lds_read_tr16(at), lds_read_tr16(at + 16 * stride));
}
// the same with keys from `limit` on as zeros: the path of tiles in which some query must not see a non-finite value
VA_DEVINL bf16x8_t v_frag_below(const char* vt, int stride, int ht, int u, int lane, int left) {
    s16x8_t v = __builtin_bit_cast(s16x8_t, v_frag(vt, stride, ht, u, lane));
    const int g4 = (lane >> 4) * 4;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 32 * u + 16 * (e >> 2) + g4 + (e & 3) < left ? v[e] : (short)0;
    return __builtin_bit_cast(bf16x8_t, v);
}

// O^T += V^T P^T of a tile for 16 queries.  `guard`: the tile holds a non-finite value and not every query sees all of it;
// zero weights do not silence it in a product, so each query's column is formed with the keys it does not see set to zero.
template <int HD>
VA_DEVINL void tile_pv(const char* vt, int stride, const bf16x8_t (&pf)[2], f32x4_t (&o)[HD / 16], int lane, bool guard, int left) {
    if (!guard) {
#pragma unroll
        for (int ht = 0; ht < HD / 16; ++ht)
#pragma unroll
            for (int u = 0; u < 2; ++u) o[ht] = mfma16(v_frag(vt, stride, ht, u, lane), pf[u], o[ht]);
        return;
    }
#pragma unroll 1
    for (int col = 0; col < 16; ++col) {
        const int mine = __shfl(left, col);                 // keys of this tile that query `col` sees
        const bool on = (lane & 15) == col;
        bf16x8_t pc[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            u32x4_t w = __builtin_bit_cast(u32x4_t, pf[u]);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = on ? w[e] : 0u;
            pc[u] = as_frag(w);
        }
#pragma unroll
        for (int ht = 0; ht < HD / 16; ++ht) {
            f32x4_t now = o[ht];
#pragma unroll
            for (int u = 0; u < 2; ++u) now = mfma16(v_frag_below(vt, stride, ht, u, lane, mine), pc[u], now);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[ht][r] = on ? now[r] : o[ht][r];      // 0 * NaN of the other columns stays out
            __builtin_amdgcn_sched_barrier(0);              // a rare path: no registers for reads ahead
        }
    }
}

// Few rows (up to 16 per key/value head): bound by the cache's bytes.  Waves take tiles in turn, each with its own running
// state; keys go straight from memory to operands, values through a private piece of LDS for their transposition, the next
// tile's bytes are requested before the current one is used.  Streams and heads that leave CUs idle are split over the keys.
// 32 streams of up to 8256 tokens, 8 heads of 128 with four query heads each: 91 us, 4.5 TB/s (two workgroups to a CU; with
// one 105, with four 100).
template <int HD>
__global__ __launch_bounds__(256) void kv8_attn_rows_kernel(Cache c, AttnArgs a) {
    constexpr int VSTR = HD * 2 + 32;        // row stride of the values in LDS: four rows of a transposed read on distinct banks
    constexpr int NK = HD / 64;              // 16-byte pieces of a key row per lane
    constexpr int NP = HD / 16;              // 16-byte pieces of a 64-key tile per lane
    __shared__ __align__(16) char lds[4 * KB * VSTR];
    __shared__ float sml[4][2][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, g = lane >> 4, g4 = g * 4;
    const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int rows = a.n * a.G;
    int len, nb;
    stream_lengths(a, c, b, len, nb);
    const int64_t bh = (int64_t)b * a.H + h;
    const int limit = m < rows ? key_limit(a, m / a.G, len, nb) : 0;
    int most = limit, least = m < rows ? limit : 0x7fffffff;
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) most = max(most, __shfl_xor(most, off)), least = min(least, __shfl_xor(least, off));
    most = __builtin_amdgcn_readfirstlane(most);            // the four lane groups hold the same queries
    least = __builtin_amdgcn_readfirstlane(least);
    const int tiles = (most + KB - 1) / KB, full = len / KB;         // tiles below `full` are in 8 bits, the next is the open one
    const uint8_t *kb = c.k8 + bh * c.cap * HD, *vb = c.v8 + bh * c.cap * HD;
    const float *ksp = c.ks + bh * (c.cap / KB), *vsp = c.vs + bh * (c.cap / KB);
    char* vt = lds + wave * KB * VSTR;
    // queries: row m, the HD/4 elements that this lane group's key pieces hold
    bf16x8_t qf[HD / 32];
#pragma unroll
    for (int f = 0; f < HD / 32; ++f) {
        u32x4_t v = {0u, 0u, 0u, 0u};
        if (m < rows)
            v = *(const u32x4_t*)(a.q + b * a.bsq + (int64_t)(m / a.G) * a.ldq + ((int64_t)h * a.G + m % a.G) * HD + g * (HD / 4) + 8 * f);
        qf[f] = as_frag(v);
    }
    f32x4_t o[HD / 16];
#pragma unroll
    for (int ht = 0; ht < HD / 16; ++ht) o[ht] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    float mx = NEG_INF, sum = 0.f;
    u32x4_t kr[4][NK], vr[NP];
    float kscale = 1.f, vscale = 1.f;
    auto request = [&](int t) {
        const int64_t at = (int64_t)t * KB * HD;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
            for (int x = 0; x < NK; ++x) kr[kt][x] = span16(kb + at, KB * HD, (kt * 16 + m) * HD + g * (HD / 4) + x * 16);
#pragma unroll
        for (int x = 0; x < NP; ++x) vr[x] = span16(vb + at, KB * HD, (x * 64 + lane) * 16);
        kscale = ksp[t];
        vscale = vsp[t];
    };
    const int step = 4 * a.splits;
    int t = split * 4 + wave;
    if (t < tiles && t < full) request(t);
    for (; t < tiles; t += step) {
        f32x4_t s[4];
        bool bad = false;
        const bool edge = (t + 1) * KB > least;
        if (t < full) {
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                s[kt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int x = 0; x < NK; ++x) {
                    s[kt] = mfma16(as_frag(widen8(kr[kt][x][0], kr[kt][x][1], kscale)), qf[2 * x], s[kt]);
                    s[kt] = mfma16(as_frag(widen8(kr[kt][x][2], kr[kt][x][3], kscale)), qf[2 * x + 1], s[kt]);
                }
            }
#pragma unroll
            for (int x = 0; x < NP; ++x) {
                const int idx = x * 64 + lane, row = idx / (HD / 16), col = (idx % (HD / 16)) * 16;
                const u32x4_t lo = widen8(vr[x][0], vr[x][1], vscale), hi = widen8(vr[x][2], vr[x][3], vscale);
                if (edge) bad |= any_nonfinite(lo) || any_nonfinite(hi);
                *(u32x4_t*)(vt + row * VSTR + col * 2) = lo;
                *(u32x4_t*)(vt + row * VSTR + col * 2 + 16) = hi;
            }
            if (t + step < tiles && t + step < full) request(t + step);
        } else {
            const bf16_t* ko = c.ko + bh * KB * HD;
            const bf16_t* vo = c.vo + bh * KB * HD;
            const int left = len - t * KB;
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                s[kt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < HD / 32; ++f)
                    s[kt] = mfma16(as_frag(span16(ko, left * HD * 2, ((16 * kt + m) * HD + g * (HD / 4) + 8 * f) * 2)), qf[f], s[kt]);
            }
#pragma unroll
            for (int x = 0; x < 2 * NP; ++x) {
                const int idx = x * 64 + lane, row = idx / (HD / 8), col = (idx % (HD / 8)) * 8;
                const u32x4_t v = span16(vo, left * HD * 2, idx * 16);      // zeros behind the stream's end, whatever lies there
                bad |= any_nonfinite(v);
                *(u32x4_t*)(vt + row * VSTR + col * 2) = v;
            }
        }
        bf16x8_t pf[2];
        const float fade = edge ? tile_softmax<true>(s, t * KB, g4, limit, a.scale2, mx, sum, pf)
                                : tile_softmax<false>(s, t * KB, g4, limit, a.scale2, mx, sum, pf);
#pragma unroll
        for (int ht = 0; ht < HD / 16; ++ht) o[ht] *= fade;
        tile_pv<HD>(vt, VSTR, pf, o, lane, edge && __any(bad), limit - t * KB);
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    // the four waves' states, joined in LDS: rows of HD values per query
    __syncthreads();
    float* so = (float*)lds;
    constexpr int OSTR = HD + 4;
#pragma unroll
    for (int ht = 0; ht < HD / 16; ++ht) *(f32x4_t*)(so + (wave * 16 + m) * OSTR + 16 * ht + g4) = o[ht];
    if (g == 0) sml[wave][0][m] = mx, sml[wave][1][m] = sum;
    __syncthreads();
    for (int idx = threadIdx.x; idx < 16 * HD / 4; idx += 256) {
        const int row = idx / (HD / 4), col = (idx % (HD / 4)) * 4;
        if (row >= rows) continue;
        float top = NEG_INF, total = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, sml[w][0][row]);
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = part_factor(sml[w][0][row], top, a.scale2);
            total = fmaf(f, sml[w][1][row], total);
            acc += f * *(const f32x4_t*)(so + (w * 16 + row) * OSTR + col);
        }
        if (a.splits == 1) {
            acc *= total == 0.f ? 0.f : 1.f / total;        // nothing seen: zeros
            bf16_t* dst = a.out + (((int64_t)b * a.n + row / a.G) * a.H * a.G + (int64_t)h * a.G + row % a.G) * HD + col;
            *(u32x2_t*)dst = (u32x2_t){pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3])};
        } else {
            const int64_t at = ((int64_t)split * a.B * a.H + bh) * rows + row;
            *(f32x4_t*)(a.part_o + at * HD + col) = acc;
            if (col == 0) a.part_ml[2 * at] = top, a.part_ml[2 * at + 1] = total;
        }
    }
}

// Many rows: a tile's keys and values are widened to bf16 once and shared through LDS, double-buffered, with the tile after next
// already requested; W waves with 16 CT rows each.  Bound by the length of a tile's chain (widening, scores, softmax, values)
// where few waves share a SIMD, by the LDS reads of its operands where many do: 258 rows x 16 streams x 8 heads of 128 over
// up to 2064 tokens in 67 us, 390 TFLOP/s, with nine waves of 16 rows to a workgroup and CU (four waves of 32 rows and a third
// row tile of two rows: 78); 128 rows x 64 streams x 8 heads over 2064 tokens in 110 us with four waves of 32 rows, two
// workgroups to a CU (twelve of 16: 122-143).
template <int HD, int CT, int W>
__global__ __launch_bounds__(64 * W, W == 12 ? 3 : 2) void kv8_attn_tile_kernel(Cache c, AttnArgs a) {
    constexpr int KSTR = HD * 2 + 16, VSTR = HD * 2 + 32, BUF = KB * (KSTR + VSTR);
    constexpr int THREADS = 64 * W, PIECES = KB * HD / 16, N = (PIECES + THREADS - 1) / THREADS;    // 16 bytes of codes each
    extern __shared__ __align__(16) char lds[];
    __shared__ int sbad[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 15, g = lane >> 4, g4 = g * 4;
    const int rows = a.n * a.G, h = blockIdx.y, b = blockIdx.z;
    const int split = blockIdx.x % a.splits, first_row = (int)(blockIdx.x / a.splits) * a.tile, end_row = min(first_row + a.tile, rows);
    const int row0 = first_row + wave * 16 * CT;
    int len, nb;
    stream_lengths(a, c, b, len, nb);
    const int64_t bh = (int64_t)b * a.H + h;
    const uint8_t *kb = c.k8 + bh * c.cap * HD, *vb = c.v8 + bh * c.cap * HD;
    const float *ksp = c.ks + bh * (c.cap / KB), *vsp = c.vs + bh * (c.cap / KB);
    const int full = len / KB;
    // the workgroup's last visible key: limits do not fall with the row
    const int last_row = end_row - 1, last_q = min(last_row / a.G, nb - 1);
    const int most = last_q >= first_row / a.G ? key_limit(a, last_q, len, nb) : 0;
    // keys that every row of the workgroup sees
    const int all_see = last_row / a.G < nb ? key_limit(a, first_row / a.G, len, nb) : 0;
    const bool idle = row0 >= end_row;          // a wave without rows only helps to load
    const int tiles = (most + KB - 1) / KB;
    const int per = (tiles + a.splits - 1) / a.splits, t_begin = split * per, t_end = min(tiles, t_begin + per);
    bf16x8_t qf[CT][HD / 32];
    int limit[CT], least = 0x7fffffff;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        const int row = row0 + 16 * ct + m;
        limit[ct] = row < end_row ? key_limit(a, row / a.G, len, nb) : 0;
        if (row < end_row) least = min(least, limit[ct]);
#pragma unroll
        for (int f = 0; f < HD / 32; ++f) {
            u32x4_t v = {0u, 0u, 0u, 0u};
            if (row < end_row)
                v = *(const u32x4_t*)(a.q + b * a.bsq + (int64_t)(row / a.G) * a.ldq + ((int64_t)h * a.G + row % a.G) * HD + 32 * f + 8 * g);
            qf[ct][f] = as_frag(v);
        }
    }
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) least = min(least, __shfl_xor(least, off));
    least = __builtin_amdgcn_readfirstlane(least);
    f32x4_t o[CT][HD / 16];
    float mx[CT], sum[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        mx[ct] = NEG_INF, sum[ct] = 0.f;
#pragma unroll
        for (int ht = 0; ht < HD / 16; ++ht) o[ct][ht] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    }
    u32x4_t kr[N], vr[N];
    float kscale = 1.f, vscale = 1.f;
    auto request = [&](int t) {
        if (t >= t_end || t >= full) return;
        const int64_t at = (int64_t)t * KB * HD;
#pragma unroll
        for (int p = 0; p < N; ++p) {
            kr[p] = span16(kb + at, KB * HD, (p * THREADS + tid) * 16);      // zeros for threads without a piece
            vr[p] = span16(vb + at, KB * HD, (p * THREADS + tid) * 16);
        }
        kscale = ksp[t];
        vscale = vsp[t];
    };
    auto place = [&](int t) {                // requested bytes (or the open block) into the tile's buffer
        if (t >= t_end) return;
        bool bad = false;
        const bool look = (t + 1) * KB > all_see;
        // everything below is an immediate away from the thread's first piece; the compiler would keep each sum in a
        // register over the loop (and spill it) if it could see that they do not change
        int id = tid;
        asm volatile("" : "+v"(id));
        if (t < full) {
            constexpr int C = HD / 16, ROWS = THREADS / C;  // pieces of a row, rows of a pass
            char* kt_ = lds + (t & 1) * BUF + (id / C) * KSTR + (id % C) * 32;
            char* vt_ = lds + (t & 1) * BUF + KB * KSTR + (id / C) * VSTR + (id % C) * 32;
#pragma unroll
            for (int p = 0; p < N; ++p) {
                if (PIECES % THREADS != 0 && p * W + wave >= PIECES / 64) continue;
                *(u32x4_t*)(kt_ + p * ROWS * KSTR) = widen8(kr[p][0], kr[p][1], kscale);
                *(u32x4_t*)(kt_ + p * ROWS * KSTR + 16) = widen8(kr[p][2], kr[p][3], kscale);
                const u32x4_t lo = widen8(vr[p][0], vr[p][1], vscale), hi = widen8(vr[p][2], vr[p][3], vscale);
                if (look) bad |= any_nonfinite(lo) || any_nonfinite(hi);
                *(u32x4_t*)(vt_ + p * ROWS * VSTR) = lo;
                *(u32x4_t*)(vt_ + p * ROWS * VSTR + 16) = hi;
            }
        } else {
            constexpr int C = HD / 8, ROWS = THREADS / C;
            const int left = len - t * KB;
            char* kt_ = lds + (t & 1) * BUF + (id / C) * KSTR + (id % C) * 16;
            char* vt_ = lds + (t & 1) * BUF + KB * KSTR + (id / C) * VSTR + (id % C) * 16;
#pragma unroll
            for (int p = 0; p < (2 * PIECES + THREADS - 1) / THREADS; ++p) {
                if (2 * PIECES % THREADS != 0 && p * W + wave >= 2 * PIECES / 64) continue;
                const u32x4_t k = span16(c.ko + bh * KB * HD, left * HD * 2, (p * THREADS + id) * 16);
                const u32x4_t v = span16(c.vo + bh * KB * HD, left * HD * 2, (p * THREADS + id) * 16);
                bad |= any_nonfinite(v);
                *(u32x4_t*)(kt_ + p * ROWS * KSTR) = k;
                *(u32x4_t*)(vt_ + p * ROWS * VSTR) = v;
            }
        }
        if (bad) sbad[t & 1] = 1;            // every writer writes the same
    };
    if (tid < 2) sbad[tid] = 0;
    __syncthreads();
    request(t_begin);
    place(t_begin);
    request(t_begin + 1);
    for (int t = t_begin; t < t_end; ++t) {
        __syncthreads();                     // tile t is in LDS; the buffer of t + 1 is free
        const bool flagged = sbad[t & 1] != 0;
        place(t + 1);
        request(t + 2);
        if (idle) continue;
        int ln = lane;                       // as in place(): addresses are formed anew instead of kept and spilled
        asm volatile("" : "+v"(ln));
        const char *kt_ = lds + (t & 1) * BUF, *vt_ = kt_ + KB * KSTR;
        f32x4_t s[CT][4];
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            s[0][kt] = s[CT - 1][kt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < HD / 32; ++f) {
                const bf16x8_t kf = as_frag(*(const u32x4_t*)(kt_ + (ln & 15) * KSTR + (ln >> 4) * 16 + 16 * kt * KSTR + 64 * f));
                s[0][kt] = mfma16(kf, qf[0][f], s[0][kt]);
                if (CT > 1) s[CT - 1][kt] = mfma16(kf, qf[CT - 1][f], s[CT - 1][kt]);
            }
        }
        const bool edge = (t + 1) * KB > least;
        bf16x8_t pf[CT][2];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            const float fade = edge ? tile_softmax<true>(s[ct], t * KB, g4, limit[ct], a.scale2, mx[ct], sum[ct], pf[ct])
                                    : tile_softmax<false>(s[ct], t * KB, g4, limit[ct], a.scale2, mx[ct], sum[ct], pf[ct]);
#pragma unroll
            for (int ht = 0; ht < HD / 16; ++ht) o[ct][ht] *= fade;
        }
        if (edge && flagged) {
            tile_pv<HD>(vt_, VSTR, pf[0], o[0], ln, true, limit[0] - t * KB);
            if (CT > 1) tile_pv<HD>(vt_, VSTR, pf[CT - 1], o[CT - 1], ln, true, limit[CT - 1] - t * KB);
        } else {
#pragma unroll
            for (int ht = 0; ht < HD / 16; ++ht)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const bf16x8_t vf = v_frag(vt_, VSTR, ht, u, ln);
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) o[ct][ht] = mfma16(vf, pf[ct][u], o[ct][ht]);
                }
        }
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
        sum[ct] += __shfl_xor(sum[ct], 16);
        sum[ct] += __shfl_xor(sum[ct], 32);
        const int row = row0 + 16 * ct + m;
        if (row >= end_row) continue;
        if (a.splits == 1) {
            const float inv = sum[ct] == 0.f ? 0.f : 1.f / sum[ct];                     // nothing seen: zeros
            bf16_t* dst = a.out + (((int64_t)b * a.n + row / a.G) * a.H * a.G + (int64_t)h * a.G + row % a.G) * HD + g4;
#pragma unroll
            for (int ht = 0; ht < HD / 16; ++ht) {
                const f32x4_t v = o[ct][ht] * inv;
                *(u32x2_t*)(dst + 16 * ht) = (u32x2_t){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
            }
        } else {
            const int64_t at = ((int64_t)split * a.B * a.H + bh) * rows + row;
#pragma unroll
            for (int ht = 0; ht < HD / 16; ++ht) *(f32x4_t*)(a.part_o + at * HD + 16 * ht + g4) = o[ct][ht];
            if (g == 0) a.part_ml[2 * at] = mx[ct], a.part_ml[2 * at + 1] = sum[ct];
        }
    }
}

// Joins the splits: HD/4 lanes per row (1024 rows in two pieces: 5 us).
template <int HD>
__global__ __launch_bounds__(256) void kv8_attn_join_kernel(AttnArgs a) {
    const int64_t all = (int64_t)a.B * a.H * a.n * a.G;
    const int64_t idx = (int64_t)blockIdx.x * (1024 / HD) + threadIdx.x / (HD / 4);
    const int col = (threadIdx.x % (HD / 4)) * 4;
    if (idx >= all) return;
    float top = NEG_INF;
    for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_ml[2 * (s * all + idx)]);
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    float total = 0.f;
    for (int s = 0; s < a.splits; ++s) {
        const float f = part_factor(a.part_ml[2 * (s * all + idx)], top, a.scale2);
        total = fmaf(f, a.part_ml[2 * (s * all + idx) + 1], total);
        acc += f * *(const f32x4_t*)(a.part_o + (s * all + idx) * HD + col);
    }
    acc *= total == 0.f ? 0.f : 1.f / total;
    const int rows = a.n * a.G;
    const int64_t bh = idx / rows;
    const int row = (int)(idx % rows);
    bf16_t* dst = a.out + (((bh / a.H) * a.n + row / a.G) * a.H * a.G + (bh % a.H) * a.G + row % a.G) * HD + col;
    *(u32x2_t*)dst = (u32x2_t){pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3])};
}

// ---- host side ------------------------------------------------------------------------------------------------
// Query rows of a workgroup where there are many (a multiple of 16).  While that makes no more workgroups than CUs, up to twelve
// waves of 16 rows, the rows spread evenly over the workgroups (128 rows x 32 streams x 8 heads over 2064 tokens: 68 us, as
// below 76; 192 x 16 x 8: 56, 78).  From there on four waves of 32 rows, which read each key from LDS half as often and let a
// second workgroup onto the CU (128 rows x 48 streams x 8 heads: 97 us, as above 121).
int64_t kv8_even_tiles(int64_t rows) { return (rows + 191) / 192; }
bool kv8_spread(int64_t B, int64_t H, int64_t rows) { return B * H * kv8_even_tiles(rows) <= 256; }
int kv8_tile(int64_t B, int64_t H, int64_t rows) {
    const int64_t units = (rows + 15) / 16, tiles = kv8_even_tiles(rows);
    return kv8_spread(B, H, rows) ? (int)((units + tiles - 1) / tiles) * 16 : 128;
}
// Pieces that the keys are split into.  Few rows: two workgroups to a CU where there are not as many (streams, heads); many rows:
// at most one; never a piece below four tiles per wave (few rows) or per workgroup (many rows).  `max_len` only steers this.
int kv8_splits(int64_t B, int64_t H, int64_t rows, int64_t max_len) {
    const int64_t tile = rows <= 16 ? 16 : kv8_tile(B, H, rows);
    const int64_t groups = B * H * ((rows + tile - 1) / tile), tiles = (max_len + KB - 1) / KB;
    int64_t s = rows <= 16 ? (2 * 256 + groups - 1) / groups : 256 / groups;
    const int64_t most = rows <= 16 ? (tiles + 15) / 16 : (tiles + 3) / 4;
    s = s < most ? s : most;
    return (int)(s < 1 ? 1 : s > 128 ? 128 : s);
}

int kv8_check(const char* who, int64_t B, int64_t H, int64_t hd, int64_t cap, int64_t n, uintptr_t bits) {
    VA_CHECK_ARG(B > 0 && H > 0 && n > 0 && cap > 0, "%s: empty problem", who);
    VA_CHECK_ARG(hd == 64 || hd == 128, "%s: head dim %lld not supported (64 or 128)", who, (long long)hd);
    VA_CHECK_ARG(cap % KB == 0 && cap < (1ll << 30), "%s: the capacity must be a multiple of 64 below 2^30", who);
    VA_CHECK_ARG(B < 65536 && H < 32768 && n < (1ll << 24), "%s: problem too large", who);
    VA_CHECK_ARG(bits % 16 == 0, "%s: misaligned operand", who);
    return VA_OK;
}

template <int HD>
int kv8_attn(const Cache& c, const AttnArgs& a, hipStream_t stream) {
    const int rows = a.n * a.G;
    if (rows <= 16) {
        hipLaunchKernelGGL(kv8_attn_rows_kernel<HD>, dim3(a.splits, a.H, a.B), dim3(256), 0, stream, c, a);
    } else {
        constexpr int lds = 2 * KB * (HD * 4 + 48);
        const bool spread = kv8_spread(a.B, a.H, rows);
        const auto fn = spread ? kv8_attn_tile_kernel<HD, 1, 12> : kv8_attn_tile_kernel<HD, 2, 4>;
        if (hipFuncSetAttribute((const void*)fn, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) {
            (void)hipGetLastError();
            va_set_error("va_kv8_attn: cannot reserve %d bytes of LDS", lds);
            return VA_ERR_LAUNCH;
        }
        hipLaunchKernelGGL(fn, dim3((unsigned)((rows + a.tile - 1) / a.tile * a.splits), a.H, a.B), dim3(spread ? 768 : 256), lds, stream, c, a);
    }
    VA_CHECK_LAUNCH("va_kv8_attn");
    if (a.splits > 1) {
        const int64_t all = (int64_t)a.B * a.H * rows, per = 1024 / HD;
        hipLaunchKernelGGL(kv8_attn_join_kernel<HD>, dim3((unsigned)((all + per - 1) / per)), dim3(256), 0, stream, a);
        VA_CHECK_LAUNCH("va_kv8_attn (join)");
    }
    return VA_OK;
}

}  // namespace

extern "C" int va_kv8_append(const void* k, const void* v, int64_t ldk, int64_t ldv, int64_t bsk, int64_t bsv, const int32_t* new_tokens,
                             int64_t n, void* k8, void* v8, float* k_scale, float* v_scale, void* k_open, void* v_open,
                             int32_t* lengths, int64_t B, int64_t H, int64_t hd, int64_t cap, hipStream_t stream) {
    VA_CHECK_ARG(k && v && k8 && v8 && k_scale && v_scale && k_open && v_open && lengths, "va_kv8_append: null operand");
    const int rc = kv8_check("va_kv8_append", B, H, hd, cap, n, (uintptr_t)k | (uintptr_t)v | (uintptr_t)k8 | (uintptr_t)v8 |
                             (uintptr_t)k_open | (uintptr_t)v_open);
    if (rc != VA_OK) return rc;
    VA_CHECK_ARG(ldk >= H * hd && ldv >= H * hd && (ldk | ldv | bsk | bsv) % 8 == 0 && bsk >= 0 && bsv >= 0,
                 "va_kv8_append: a token stride must be at least H * hd, and the strides multiples of 8");
    const dim3 grid((unsigned)((n + KB - 2) / KB + 1), (unsigned)(2 * H), (unsigned)B);
    if (hd == 128)
        hipLaunchKernelGGL(kv8_append_kernel<128>, grid, dim3(256), 0, stream, (const bf16_t*)k, (const bf16_t*)v, ldk, ldv, bsk, bsv,
                           new_tokens, (int)n, (uint8_t*)k8, (uint8_t*)v8, k_scale, v_scale, (bf16_t*)k_open, (bf16_t*)v_open,
                           (const int32_t*)lengths, cap, (int)H);
    else
        hipLaunchKernelGGL(kv8_append_kernel<64>, grid, dim3(256), 0, stream, (const bf16_t*)k, (const bf16_t*)v, ldk, ldv, bsk, bsv,
                           new_tokens, (int)n, (uint8_t*)k8, (uint8_t*)v8, k_scale, v_scale, (bf16_t*)k_open, (bf16_t*)v_open,
                           (const int32_t*)lengths, cap, (int)H);
    VA_CHECK_LAUNCH("va_kv8_append");
    hipLaunchKernelGGL(kv8_advance_kernel, dim3((unsigned)((B + 255) / 256)), dim3(256), 0, stream, lengths, new_tokens, (int)n, cap,
                       (int)B);
    VA_CHECK_LAUNCH("va_kv8_append (lengths)");
    return VA_OK;
}

extern "C" int64_t va_kv8_attn_workspace_floats(int64_t B, int64_t n, int64_t H, int64_t group, int64_t hd, int64_t max_len) {
    if (B <= 0 || n <= 0 || H <= 0 || group <= 0 || hd <= 0) return 0;
    const int64_t s = kv8_splits(B, H, n * group, max_len);
    return s > 1 ? s * B * H * n * group * (hd + 2) : 0;
}

extern "C" int va_kv8_attn(const void* q, int64_t ldq, int64_t bsq, const int32_t* new_tokens, const void* k8, const void* v8,
                           const float* k_scale, const float* v_scale, const void* k_open, const void* v_open,
                           const int32_t* lengths, void* out, float* workspace, int64_t B, int64_t n, int64_t H, int64_t group,
                           int64_t hd, int64_t cap, int64_t max_len, int64_t tokens_per_timestep, float scale, hipStream_t stream) {
    VA_CHECK_ARG(q && k8 && v8 && k_scale && v_scale && k_open && v_open && lengths && out, "va_kv8_attn: null operand");
    const int rc = kv8_check("va_kv8_attn", B, H, hd, cap, n, (uintptr_t)q | (uintptr_t)k8 | (uintptr_t)v8 | (uintptr_t)k_open |
                             (uintptr_t)v_open | (uintptr_t)out | (uintptr_t)workspace);
    if (rc != VA_OK) return rc;
    VA_CHECK_ARG(group > 0 && group <= 1024 && n * group < (1ll << 24) && B * H * n * group < (1ll << 31), "va_kv8_attn: problem too large");
    VA_CHECK_ARG(ldq >= H * group * hd && (ldq | bsq) % 8 == 0 && bsq >= 0,
                 "va_kv8_attn: the token stride of q must be at least its heads' width, and the strides multiples of 8");
    VA_CHECK_ARG(tokens_per_timestep >= 0 && tokens_per_timestep < (1ll << 30), "va_kv8_attn: tokens per timestep out of range");
    VA_CHECK_ARG(max_len >= 0 && max_len <= cap, "va_kv8_attn: max_len out of range");
    VA_CHECK_ARG(scale > 0.f && scale < 1e30f, "va_kv8_attn: the scale must be positive");
    const int splits = kv8_splits(B, H, n * group, max_len);
    VA_CHECK_ARG(splits == 1 || workspace, "va_kv8_attn: null workspace");
    const Cache c = {(const uint8_t*)k8, (const uint8_t*)v8, k_scale, v_scale, (const bf16_t*)k_open, (const bf16_t*)v_open, lengths, cap};
    AttnArgs a = {(const bf16_t*)q, ldq, bsq, new_tokens, (bf16_t*)out, workspace, nullptr, (int)B, (int)n, (int)H, (int)group,
                  (int)tokens_per_timestep, splits, kv8_tile(B, H, n * group), scale * LOG2E};
    if (splits > 1) a.part_ml = workspace + (int64_t)splits * B * H * n * group * hd;
    return hd == 128 ? kv8_attn<128>(c, a, stream) : kv8_attn<64>(c, a, stream);
}
