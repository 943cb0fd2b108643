// Output stage of the memory layer with its gradient: y = LayerNorm(x) gamma + beta, x = (o * gate) * silu(g), rows of any
// width that is a multiple of 4 (up to 4096), f32 or bf16.
//
// With xn = (x - mean) rstd and w = dy gamma:
//     dx = rstd (w - mean(w) - xn mean(w xn)),     dgamma = sum_rows dy xn,     dbeta = sum_rows dy
//     d_o = dx gate silu(g),   d_gate = dx o silu(g),   d_g = dx o gate s (1 + g (1 - s)),  s = sigmoid(g).
// Bound by memory: forward three values read and one written per element, gradient four read and three written; a row stays
// in registers between its sums and its results, so each is read once.  Up to 1024 columns a wave holds a row (four elements
// per lane and step, rows of a workgroup's waves are independent); wider rows are spread over the four waves of a workgroup
// (more than 16 elements per lane and operand would not stay in registers in the gradient) and their sums meet in LDS.
// A wave keeps its columns' dgamma / dbeta in registers over all its rows; the workgroups' sums go to a workspace and a
// second launch adds them in a fixed order: results do not depend on timing.
// 16 512 rows of 1024, inputs from memory: f32 forward 73 us (3.7 TB/s; 59 where the last-level cache holds some of them),
// gradient 87 + 6 us (5.5 TB/s); bf16 39 us (3.5 TB/s), 61 + 6 us (3.9 TB/s).
#include "common.h"

namespace {

template <typename T> struct gn4;
template <> struct gn4<float> {
    static VA_DEVINL f32x4_t load(const float* p) { return *(const f32x4_t*)p; }
    static VA_DEVINL void store(float* p, f32x4_t v) { *(f32x4_t*)p = v; }
};
template <> struct gn4<bf16_t> {
    static VA_DEVINL f32x4_t load(const bf16_t* p) {
        const u32x2_t w = *(const u32x2_t*)p;
        return (f32x4_t){__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xffff0000u), __uint_as_float(w[1] << 16),
                         __uint_as_float(w[1] & 0xffff0000u)};
    }
    // results of the tensors' own type: one rounding
    static VA_DEVINL void store(bf16_t* p, f32x4_t v) { *(u32x2_t*)p = (u32x2_t){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])}; }
};

VA_DEVINL float gn_sigmoid(float x) { return 1.0f / (1.0f + __expf(-x)); }

// sums over the LANES lanes that hold a row (64: a wave; 256: the workgroup, through LDS)
template <int LANES, int N>
VA_DEVINL void row_sum(float (&s)[N], float (*buf)[4]) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
#pragma unroll
        for (int n = 0; n < N; ++n) s[n] += __shfl_xor(s[n], off);
    if (LANES == 256) {
        __syncthreads();                          // the sums before have been read
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int n = 0; n < N; ++n) buf[n][threadIdx.x >> 6] = s[n];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) s[n] = (buf[n][0] + buf[n][1]) + (buf[n][2] + buf[n][3]);
    }
}

// NV steps of 4 * LANES columns cover a row
template <typename T, int LANES, int NV>
__global__ __launch_bounds__(256) void gated_norm_fwd_kernel(const T* __restrict__ O, const T* __restrict__ GATE, const T* __restrict__ G,
                                                             const float* __restrict__ GAMMA, const float* __restrict__ BETA,
                                                             T* __restrict__ Y, float* __restrict__ MEAN, float* __restrict__ RSTD,
                                                             int64_t M, int D, float eps) {
    __shared__ float buf[1][4];
    const int lane = threadIdx.x % LANES;
    const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (LANES == 64 && row >= M) return;           // LANES == 256: the grid has M workgroups
    const float inv = 1.0f / (float)D;
    f32x4_t x[NV];
    float s[1] = {0.f};
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int c = (n * LANES + lane) * 4;
        x[n] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
        if (c < D) {
            const int64_t at = row * D + c;
            const f32x4_t o = gn4<T>::load(O + at), gate = gn4<T>::load(GATE + at), g = gn4<T>::load(G + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[n][e] = (o[e] * gate[e]) * (g[e] * gn_sigmoid(g[e]));
                s[0] += x[n][e];
            }
        }
    }
    row_sum<LANES>(s, buf);
    const float mean = s[0] * inv;
    float v[1] = {0.f};
#pragma unroll
    for (int n = 0; n < NV; ++n)
        if ((n * LANES + lane) * 4 < D)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[n][e] -= mean;
                v[0] = fmaf(x[n][e], x[n][e], v[0]);
            }
    row_sum<LANES>(v, buf);
    const float rstd = 1.0f / sqrtf(v[0] * inv + eps);
    if (lane == 0 && MEAN != nullptr) {
        MEAN[row] = mean;
        RSTD[row] = rstd;
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int c = (n * LANES + lane) * 4;
        if (c < D) {
            const f32x4_t gm = *(const f32x4_t*)(GAMMA + c), bt = *(const f32x4_t*)(BETA + c);
            f32x4_t y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = fmaf(x[n][e] * rstd, gm[e], bt[e]);
            gn4<T>::store(Y + row * D + c, y);
        }
    }
}

template <typename T, int LANES, int NV>
__global__ __launch_bounds__(256) void gated_norm_bwd_kernel(const T* __restrict__ DY, const T* __restrict__ O, const T* __restrict__ GATE,
                                                             const T* __restrict__ G, const float* __restrict__ GAMMA,
                                                             const float* __restrict__ MEAN, const float* __restrict__ RSTD,
                                                             T* __restrict__ DO, T* __restrict__ DGATE, T* __restrict__ DG,
                                                             float* __restrict__ PART, int64_t M, int D) {
    constexpr int PER = 256 / LANES;               // rows a workgroup handles at a time
    __shared__ float buf[2][4];
    __shared__ f32x4_t wide[PER > 1 ? 3 : 1][64];
    const int lane = threadIdx.x % LANES, sub = threadIdx.x / LANES;
    const float inv = 1.0f / (float)D;
    f32x4_t ag[NV], ab[NV], gm[NV];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int c = (n * LANES + lane) * 4;
        ag[n] = ab[n] = gm[n] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
        if (c < D) gm[n] = *(const f32x4_t*)(GAMMA + c);
    }
    for (int64_t row = (int64_t)blockIdx.x * PER + sub; row < M; row += (int64_t)gridDim.x * PER) {
        const float mean = MEAN[row], rstd = RSTD[row];
        f32x4_t o[NV], gate[NV], g[NV], dy[NV];
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * LANES + lane) * 4;
            o[n] = gate[n] = g[n] = dy[n] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
            if (c < D) {
                const int64_t at = row * D + c;
                o[n] = gn4<T>::load(O + at);
                gate[n] = gn4<T>::load(GATE + at);
                g[n] = gn4<T>::load(G + at);
                dy[n] = gn4<T>::load(DY + at);
            }
        }
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = (o[n][e] * gate[n][e]) * (g[n][e] * gn_sigmoid(g[n][e]));
                const float xn = (x - mean) * rstd, w = dy[n][e] * gm[n][e];
                s[0] += w;                         // columns behind the row's end hold zeros in dy and gamma
                s[1] = fmaf(w, xn, s[1]);
                ag[n][e] = fmaf(dy[n][e], xn, ag[n][e]);
                ab[n][e] += dy[n][e];
            }
        row_sum<LANES>(s, buf);
        const float c1 = s[0] * inv, c2 = s[1] * inv;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = (n * LANES + lane) * 4;
            f32x4_t d_o, d_gate, d_g;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float sg = gn_sigmoid(g[n][e]), silu = g[n][e] * sg, og = o[n][e] * gate[n][e];
                const float xn = (og * silu - mean) * rstd;
                const float dx = rstd * (dy[n][e] * gm[n][e] - c1 - xn * c2);
                d_o[e] = dx * gate[n][e] * silu;
                d_gate[e] = dx * o[n][e] * silu;
                d_g[e] = dx * og * (sg * fmaf(g[n][e], 1.0f - sg, 1.0f));
            }
            if (c < D) {
                const int64_t at = row * D + c;
                gn4<T>::store(DO + at, d_o);
                gn4<T>::store(DGATE + at, d_gate);
                gn4<T>::store(DG + at, d_g);
            }
        }
    }
    // a workgroup's sums: PART[workgroup][dgamma, dbeta][D]
    float* part = PART + (int64_t)blockIdx.x * 2 * D;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int c = (n * LANES + lane) * 4;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            f32x4_t v = k == 0 ? ag[n] : ab[n];
            if (PER > 1) {
                __syncthreads();
                if (sub > 0) wide[sub - 1][lane] = v;
                __syncthreads();
                if (sub > 0) continue;
                v = (v + wide[0][lane]) + (wide[1][lane] + wide[2][lane]);
            }
            if (c < D) *(f32x4_t*)(part + k * D + c) = v;
        }
    }
}

// Sum of the workgroups' rows: 64 columns to a workgroup of 16 waves, each wave adds every sixteenth row.
__global__ __launch_bounds__(1024) void gated_norm_sum_kernel(const float* __restrict__ PART, int parts, int D,
                                                              float* __restrict__ DGAMMA, float* __restrict__ DBETA) {
    __shared__ float buf[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = blockIdx.x * 64 + lane;        // dgamma's columns, then dbeta's
    float s = 0.f;
    if (col < 2 * D)
#pragma unroll 4
        for (int p = wave; p < parts; p += 16) s += PART[(int64_t)p * 2 * D + col];
    buf[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && col < 2 * D) {
        float t = 0.f;
#pragma unroll
        for (int w = 0; w < 16; ++w) t += buf[w][lane];
        if (col < D) DGAMMA[col] = t;
        else DBETA[col - D] = t;
    }
}

// Workgroups of the gradient: three to a CU keep the memory busy, and every one of them leaves a row of sums behind.
int64_t gn_groups(int64_t M, int64_t D) {
    const int64_t rows = D <= 1024 ? 4 : 1, all = (M + rows - 1) / rows;
    return all < 768 ? all : 768;
}

int gn_check(const char* who, int64_t M, int64_t D, uintptr_t bits, int bf16) {
    VA_CHECK_ARG(M > 0 && M < (D <= 1024 ? 1ll << 26 : 1ll << 24), "%s: row count out of range", who);     // lanes of a grid: 2^32
    VA_CHECK_ARG(D > 0 && D % 4 == 0 && D <= 4096, "%s: width %lld not supported (a multiple of 4, at most 4096)", who, (long long)D);
    VA_CHECK_ARG(bits % (bf16 ? 8 : 16) == 0, "%s: misaligned operand", who);
    return VA_OK;
}

template <typename T, int LANES, int NV>
void gn_launch_fwd(const void* o, const void* gate, const void* g, const float* gamma, const float* beta, void* y, float* mean,
                   float* rstd, int64_t M, int64_t D, float eps, hipStream_t stream) {
    const int64_t rows = 256 / LANES;
    hipLaunchKernelGGL((gated_norm_fwd_kernel<T, LANES, NV>), dim3((unsigned)((M + rows - 1) / rows)), dim3(256), 0, stream,
                       (const T*)o, (const T*)gate, (const T*)g, gamma, beta, (T*)y, mean, rstd, M, (int)D, eps);
}
template <typename T, int LANES, int NV>
void gn_launch_bwd(const void* dy, const void* o, const void* gate, const void* g, const float* gamma, const float* mean,
                   const float* rstd, void* d_o, void* d_gate, void* d_g, float* part, int64_t M, int64_t D, hipStream_t stream) {
    hipLaunchKernelGGL((gated_norm_bwd_kernel<T, LANES, NV>), dim3((unsigned)gn_groups(M, D)), dim3(256), 0, stream, (const T*)dy,
                       (const T*)o, (const T*)gate, (const T*)g, gamma, mean, rstd, (T*)d_o, (T*)d_gate, (T*)d_g, part, M, (int)D);
}
#define GN_DISPATCH(launch, T, ...)                         \
    do {                                                    \
        if (D <= 256) launch<T, 64, 1>(__VA_ARGS__);        \
        else if (D <= 512) launch<T, 64, 2>(__VA_ARGS__);   \
        else if (D <= 1024) launch<T, 64, 4>(__VA_ARGS__);  \
        else if (D <= 2048) launch<T, 256, 2>(__VA_ARGS__); \
        else launch<T, 256, 4>(__VA_ARGS__);                \
    } while (0)

}  // namespace

extern "C" int va_gated_layernorm_fwd(const void* o, const void* gate, const void* g, int is_bf16, const float* gamma,
                                      const float* beta, void* y, float* mean, float* rstd, int64_t M, int64_t D, float eps,
                                      hipStream_t stream) {
    VA_CHECK_ARG(o && gate && g && gamma && beta && y, "va_gated_layernorm_fwd: null operand");
    VA_CHECK_ARG((mean == nullptr) == (rstd == nullptr), "va_gated_layernorm_fwd: mean and rstd go together");
    const int rc = gn_check("va_gated_layernorm_fwd", M, D, (uintptr_t)o | (uintptr_t)gate | (uintptr_t)g | (uintptr_t)y, is_bf16);
    if (rc != VA_OK) return rc;
    VA_CHECK_ARG(((uintptr_t)gamma | (uintptr_t)beta) % 16 == 0, "va_gated_layernorm_fwd: misaligned operand");
    if (is_bf16) GN_DISPATCH(gn_launch_fwd, bf16_t, o, gate, g, gamma, beta, y, mean, rstd, M, D, eps, stream);
    else GN_DISPATCH(gn_launch_fwd, float, o, gate, g, gamma, beta, y, mean, rstd, M, D, eps, stream);
    VA_CHECK_LAUNCH("va_gated_layernorm_fwd");
    return VA_OK;
}

extern "C" int64_t va_gated_layernorm_bwd_workspace_floats(int64_t M, int64_t D) {
    return M > 0 && D > 0 ? gn_groups(M, D) * 2 * D : 0;
}

extern "C" int va_gated_layernorm_bwd(const void* dy, const void* o, const void* gate, const void* g, int is_bf16,
                                      const float* gamma, const float* mean, const float* rstd, void* d_o, void* d_gate, void* d_g,
                                      float* dgamma, float* dbeta, float* workspace, int64_t M, int64_t D, hipStream_t stream) {
    VA_CHECK_ARG(dy && o && gate && g && gamma && mean && rstd && d_o && d_gate && d_g && dgamma && dbeta && workspace,
                 "va_gated_layernorm_bwd: null operand");
    const int rc = gn_check("va_gated_layernorm_bwd", M, D, (uintptr_t)dy | (uintptr_t)o | (uintptr_t)gate | (uintptr_t)g |
                            (uintptr_t)d_o | (uintptr_t)d_gate | (uintptr_t)d_g, is_bf16);
    if (rc != VA_OK) return rc;
    VA_CHECK_ARG(((uintptr_t)gamma | (uintptr_t)workspace) % 16 == 0, "va_gated_layernorm_bwd: misaligned operand");
    if (is_bf16) GN_DISPATCH(gn_launch_bwd, bf16_t, dy, o, gate, g, gamma, mean, rstd, d_o, d_gate, d_g, workspace, M, D, stream);
    else GN_DISPATCH(gn_launch_bwd, float, dy, o, gate, g, gamma, mean, rstd, d_o, d_gate, d_g, workspace, M, D, stream);
    VA_CHECK_LAUNCH("va_gated_layernorm_bwd");
    hipLaunchKernelGGL(gated_norm_sum_kernel, dim3((unsigned)((2 * D + 63) / 64)), dim3(1024), 0, stream, (const float*)workspace,
                       (int)gn_groups(M, D), (int)D, dgamma, dbeta);
    VA_CHECK_LAUNCH("va_gated_layernorm_bwd (sums)");
    return VA_OK;
}
