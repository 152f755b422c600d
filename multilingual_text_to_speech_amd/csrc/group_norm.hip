// Group norm + activation + dropout over channel-last activations x[N, L, C] (fp32 or bf16 storage), forward and backward.
//
//   y  = drop(act(gamma * xhat + beta)),  xhat = (x - mean) * rstd; mean and variance of (sample n, group g) run over the sample's
//        lengths[n] valid rows and the group's C / G channels.  Rows behind them are never read; y and dx are zero there.
//   dz = drop'(dy) * act'(z);  dbeta = sum dz,  dgamma = sum dz * xhat  (over all valid rows of all samples)
//   dx = rstd * (gamma dz - mean(gamma dz) - xhat * mean(gamma dz * xhat))
//
// With an 8-bit checkpoint the backward takes x = q * 2^(code - 127) in place of the input; mean and rstd stay those of the forward.
// Statistics are held in fp32 as (count, mean, centred second moment) and merged pairwise, so an offset that is large against the
// spread costs no digits; every sum has a fixed order (no atomics).
//
// This is bytes: read x, write y; read x (or its checkpoint) and dy, write dx.  10 to 30 operations per value.
#include "vec_io.h"

constexpr int GN_T = 256;
constexpr int GN_U = 4;            // row vectors a thread requests before it uses the first
constexpr int GN_CHUNKS = 64;      // most row chunks of a sample (their partial sums are merged by one workgroup)

// ---- activations ------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float gn_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }      // v_rcp_f32: 1 ulp
// tanh through exp loses digits next to zero (1 - e cancels): the odd polynomial there (its next term is 2e-9 of z at 1/4)
__device__ __forceinline__ float gn_tanh(float z) {
    const float e = __expf(-2.f * fabsf(z)), r = copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e), z), s = z * z;
    const float p = z + z * s * (-0.33333333333f + s * (0.13333333333f + s * (-0.05396825397f + s * 0.02186948854f)));
    return fabsf(z) < 0.25f ? p : r;
}
template <int V> __device__ __forceinline__ void gn_act(int act, float (&z)[V]) {
    switch (act) {                       // uniform: one scalar branch for V values
        case MTTS_ACT_RELU:
#pragma unroll
            for (int j = 0; j < V; ++j) z[j] = z[j] < 0.f ? 0.f : z[j];      // NaN stays NaN
            break;
        case MTTS_ACT_TANH:
#pragma unroll
            for (int j = 0; j < V; ++j) z[j] = gn_tanh(z[j]);
            break;
        case MTTS_ACT_SIGMOID:
#pragma unroll
            for (int j = 0; j < V; ++j) z[j] = gn_sigmoid(z[j]);
            break;
        case MTTS_ACT_SILU:
#pragma unroll
            for (int j = 0; j < V; ++j) z[j] *= gn_sigmoid(z[j]);
            break;
        default: break;
    }
}
// d *= act'(z); relu: 0 at z = 0, as the framework's other blocks
template <int V> __device__ __forceinline__ void gn_act_slope(int act, const float (&z)[V], float (&d)[V]) {
    switch (act) {
        case MTTS_ACT_RELU:
#pragma unroll
            for (int j = 0; j < V; ++j) d[j] = z[j] > 0.f ? d[j] : 0.f;
            break;
        case MTTS_ACT_TANH:
#pragma unroll
            for (int j = 0; j < V; ++j) {      // 1 - tanh^2 = 4 e / (1 + e)^2: no cancellation in the tails
                const float e = __expf(-2.f * fabsf(z[j])), r = __builtin_amdgcn_rcpf(1.f + e);
                d[j] *= 4.f * e * r * r;
            }
            break;
        case MTTS_ACT_SIGMOID:
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float e = __expf(-fabsf(z[j])), r = __builtin_amdgcn_rcpf(1.f + e);
                d[j] *= e * r * r;
            }
            break;
        case MTTS_ACT_SILU:
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float p = gn_sigmoid(z[j]);
                d[j] *= p * (1.f + z[j] * (1.f - p));
            }
            break;
        default: break;
    }
}

// ---- statistics -------------------------------------------------------------------------------------------------------------------
struct Moments { float n, mean, m2; };
__device__ __forceinline__ Moments gn_merge(const Moments& a, const Moments& b) {
    const float n = a.n + b.n;
    if (b.n == 0.f) return a;
    if (a.n == 0.f) return b;
    const float d = b.mean - a.mean, w = b.n / n;
    return Moments{n, a.mean + d * w, a.m2 + b.m2 + d * d * a.n * w};
}

__device__ __forceinline__ int gn_length(const GroupNormArgs& p, int n) { return p.lengths ? min(max(p.lengths[n], 0), p.L) : p.L; }

// Workgroup -> (sample n, row chunk, column strip); a thread owns VEC columns and every TY-th row of the chunk.
struct GnTile { int n, chunk, c, ty, TY, r0, r1, len; bool on; };
template <int VEC> __device__ __forceinline__ GnTile gn_tile(const GroupNormArgs& p, int chunks, int strips, int TX) {
    GnTile t;
    const int strip = blockIdx.x % strips, rest = blockIdx.x / strips;
    t.chunk = rest % chunks; t.n = rest / chunks;
    const int tx = threadIdx.x % TX;
    t.ty = threadIdx.x / TX; t.TY = GN_T / TX;
    t.c = (strip * TX + tx) * VEC;
    t.len = gn_length(p, t.n);
    const int per = (p.L + chunks - 1) / chunks;
    t.r0 = t.chunk * per; t.r1 = min(p.L, t.r0 + per);
    t.on = t.c < p.C && t.ty < t.TY;
    return t;
}

// partial moments per (sample, chunk, channel): ws[(n * chunks + chunk) * C + c] = mean, and the second moment N * chunks * C further
template <typename T, int VEC>
__global__ void __launch_bounds__(GN_T) gn_moments_kernel(GroupNormArgs p, int chunks, int strips, int TX) {
    __shared__ float sm[GN_T * VEC], s2[GN_T * VEC];
    __shared__ float sn[GN_T];
    const GnTile t = gn_tile<VEC>(p, chunks, strips, TX);
    const int r1 = min(t.r1, t.len);
    Moments m[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) m[j] = Moments{0.f, 0.f, 0.f};
    if (t.on)
        for (int r = t.r0 + t.ty; r < r1; r += GN_U * t.TY) {
            Raw<T, VEC> v[GN_U];
            const T* base = (const T*)p.x + ((long)t.n * p.L) * p.C + t.c;
#pragma unroll
            for (int u = 0; u < GN_U; ++u) v[u].load(base + (long)min(r + u * t.TY, r1 - 1) * p.C);
            const int k = min(GN_U, (r1 - r + t.TY - 1) / t.TY);
            const float inv = 1.f / (float)k;
            float f[GN_U][VEC];
#pragma unroll
            for (int u = 0; u < GN_U; ++u) get_vec(v[u], f[u]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                float s = 0.f, q = 0.f;
#pragma unroll
                for (int u = 0; u < GN_U; ++u) s += u < k ? f[u][j] : 0.f;
                s *= inv;
#pragma unroll
                for (int u = 0; u < GN_U; ++u) { const float d = f[u][j] - s; q += u < k ? d * d : 0.f; }
                m[j] = gn_merge(m[j], Moments{(float)k, s, q});
            }
        }
    sn[threadIdx.x] = m[0].n;
#pragma unroll
    for (int j = 0; j < VEC; ++j) { sm[j * GN_T + threadIdx.x] = m[j].mean; s2[j * GN_T + threadIdx.x] = m[j].m2; }
    __syncthreads();
    if (t.ty == 0 && t.on) {
        float* ws = p.ws + ((long)t.n * chunks + t.chunk) * p.C + t.c;
        const long half = (long)p.N * chunks * p.C;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            for (int k = 1; k < t.TY; ++k) {
                const int i = threadIdx.x + k * TX;
                m[j] = gn_merge(m[j], Moments{sn[i], sm[j * GN_T + i], s2[j * GN_T + i]});
            }
            ws[j] = m[j].mean; ws[half + j] = m[j].m2;
        }
    }
}

// mean / rstd of one (sample, group): merge over the chunks and the group's channels.  grid N * G, one wave
__global__ void __launch_bounds__(64) gn_stats_kernel(GroupNormArgs p, int chunks) {
    const int n = blockIdx.x / p.G, g = blockIdx.x - n * p.G, Cg = p.C / p.G;
    const int len = gn_length(p, n), per = (p.L + chunks - 1) / chunks;
    const long half = (long)p.N * chunks * p.C;
    Moments m = {0.f, 0.f, 0.f};
    for (int i = threadIdx.x; i < chunks * Cg; i += 64) {
        const int k = i / Cg, c = i - k * Cg;
        const float rows = (float)max(0, min(min(p.L, (k + 1) * per), len) - k * per);
        const float* ws = p.ws + ((long)n * chunks + k) * p.C + (long)g * Cg + c;
        m = gn_merge(m, Moments{rows, ws[0], ws[half]});
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) m = gn_merge(m, Moments{__shfl_xor(m.n, d, 64), __shfl_xor(m.mean, d, 64), __shfl_xor(m.m2, d, 64)});
    if (threadIdx.x == 0) {
        p.mean[(long)n * p.G + g] = m.mean;
        p.rstd[(long)n * p.G + g] = 1.f / sqrtf((m.n > 0.f ? m.m2 / m.n : 0.f) + p.eps);
    }
}

template <int VEC> struct GnCol { float mean[VEC], rstd[VEC], gamma[VEC], beta[VEC]; };
template <int VEC> __device__ __forceinline__ GnCol<VEC> gn_col(const GroupNormArgs& p, int n, int c) {
    GnCol<VEC> k;
    const int Cg = p.C / p.G;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const int cc = min(c + j, p.C - 1);
        const long s = (long)n * p.G + cc / Cg;
        k.mean[j] = p.mean[s]; k.rstd[j] = p.rstd[s]; k.gamma[j] = p.gamma[cc]; k.beta[j] = p.beta[cc];
    }
    return k;
}

// y = drop(act(gamma (x - mean) rstd + beta))
template <typename T, int VEC>
__global__ void __launch_bounds__(GN_T) gn_apply_kernel(GroupNormArgs p, int chunks, int strips, int TX) {
    const GnTile t = gn_tile<VEC>(p, chunks, strips, TX);
    if (!t.on) return;
    const GnCol<VEC> k = gn_col<VEC>(p, t.n, t.c);
    const long base = ((long)t.n * p.L) * p.C + t.c;
    for (int r = t.r0 + t.ty; r < t.r1; r += GN_U * t.TY) {
        Raw<T, VEC> v[GN_U]; Bytes<VEC> keep[GN_U];
#pragma unroll
        for (int u = 0; u < GN_U; ++u) {
            v[u].zero(); keep[u].fill(1);
            const int rr = r + u * t.TY;
            if (rr < min(t.r1, t.len)) {
                v[u].load((const T*)p.x + base + (long)rr * p.C);
                if (p.mask) keep[u].load(p.mask + base + (long)rr * p.C);
            }
        }
#pragma unroll
        for (int u = 0; u < GN_U; ++u) {
            const int rr = r + u * t.TY;
            if (rr >= t.r1) break;
            float f[VEC];
            get_vec(v[u], f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = (f[j] - k.mean[j]) * k.rstd[j] * k.gamma[j] + k.beta[j];
            gn_act<VEC>(p.act, f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                if (p.mask) f[j] = keep[u].get(j) ? f[j] * p.mask_scale : 0.f;
                if (rr >= t.len) f[j] = 0.f;
            }
            store_vec((T*)p.y + base + (long)rr * p.C, f);
        }
    }
}

// one row vector of the backward: xhat and dz
template <typename T, int VEC, bool CK> struct GnBwdRow {
    Raw<T, VEC> x, dy; Bytes<VEC> q, keep; unsigned code;
    __device__ __forceinline__ void load(const GroupNormArgs& p, long row, int c) {
        const long at = row * p.C + c;
        dy.load((const T*)p.dy + at);
        if (CK) { q.load(p.q + at); code = p.q_code[row * ((p.C + CK_BLOCK - 1) / CK_BLOCK) + c / CK_BLOCK]; }
        else x.load((const T*)p.x + at);
        if (p.mask) keep.load(p.mask + at);
    }
    __device__ __forceinline__ void get(const GroupNormArgs& p, const GnCol<VEC>& k, float (&xhat)[VEC], float (&dz)[VEC]) const {
        float z[VEC];
        get_vec(dy, dz);
        if (CK) {
            const float s = ck_scale(code);
#pragma unroll
            for (int j = 0; j < VEC; ++j) xhat[j] = ck_value(q.get(j), s);
        } else get_vec(x, xhat);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            xhat[j] = (xhat[j] - k.mean[j]) * k.rstd[j];
            z[j] = xhat[j] * k.gamma[j] + k.beta[j];
            if (p.mask) dz[j] = keep.get(j) ? dz[j] * p.mask_scale : 0.f;
        }
        gn_act_slope<VEC>(p.act, z, dz);
    }
};

// partial sums per (sample, chunk, channel): ws = sum dz, and N * chunks * C further sum dz * xhat
template <typename T, int VEC, bool CK>
__global__ void __launch_bounds__(GN_T) gn_bwd_sums_kernel(GroupNormArgs p, int chunks, int strips, int TX) {
    __shared__ float s1[GN_T * VEC], s2[GN_T * VEC];
    const GnTile t = gn_tile<VEC>(p, chunks, strips, TX);
    float a[VEC], b[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) a[j] = b[j] = 0.f;
    if (t.on) {
        const int r1 = min(t.r1, t.len);
        const GnCol<VEC> k = gn_col<VEC>(p, t.n, t.c);
        for (int r = t.r0 + t.ty; r < r1; r += GN_U * t.TY) {
            GnBwdRow<T, VEC, CK> w[GN_U];
#pragma unroll
            for (int u = 0; u < GN_U; ++u) w[u].load(p, (long)t.n * p.L + min(r + u * t.TY, r1 - 1), t.c);
#pragma unroll
            for (int u = 0; u < GN_U; ++u) {
                if (r + u * t.TY >= r1) break;
                float xh[VEC], dz[VEC];
                w[u].get(p, k, xh, dz);
#pragma unroll
                for (int j = 0; j < VEC; ++j) { a[j] += dz[j]; b[j] += dz[j] * xh[j]; }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) { s1[j * GN_T + threadIdx.x] = a[j]; s2[j * GN_T + threadIdx.x] = b[j]; }
    __syncthreads();
    if (t.ty == 0 && t.on) {
        float* ws = p.ws + ((long)t.n * chunks + t.chunk) * p.C + t.c;
        const long half = (long)p.N * chunks * p.C;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            for (int i = 1; i < t.TY; ++i) { a[j] += s1[j * GN_T + threadIdx.x + i * TX]; b[j] += s2[j * GN_T + threadIdx.x + i * TX]; }
            ws[j] = a[j]; ws[half + j] = b[j];
        }
    }
}

// mean(gamma dz), mean(gamma dz xhat) of one (sample, group) -> gs[(n * G + g) * 2 ..].  grid N * G, one wave
__global__ void __launch_bounds__(64) gn_bwd_means_kernel(GroupNormArgs p, int chunks, float* gs) {
    const int n = blockIdx.x / p.G, g = blockIdx.x - n * p.G, Cg = p.C / p.G;
    const long half = (long)p.N * chunks * p.C;
    float a = 0.f, b = 0.f;
    for (int i = threadIdx.x; i < chunks * Cg; i += 64) {
        const int k = i / Cg, c = g * Cg + i - k * Cg;
        const float* ws = p.ws + ((long)n * chunks + k) * p.C + c;
        a += p.gamma[c] * ws[0]; b += p.gamma[c] * ws[half];
    }
    a = wave_sum(a); b = wave_sum(b);
    if (threadIdx.x == 0) {
        const float count = (float)gn_length(p, n) * (float)Cg, inv = count > 0.f ? 1.f / count : 0.f;
        gs[2L * blockIdx.x] = a * inv; gs[2L * blockIdx.x + 1] = b * inv;
    }
}

template <typename T, int VEC, bool CK>
__global__ void __launch_bounds__(GN_T) gn_bwd_apply_kernel(GroupNormArgs p, int chunks, int strips, int TX, const float* gs) {
    const GnTile t = gn_tile<VEC>(p, chunks, strips, TX);
    if (!t.on) return;
    const GnCol<VEC> k = gn_col<VEC>(p, t.n, t.c);
    float m1[VEC], m2[VEC];
    const int Cg = p.C / p.G;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const long s = 2 * ((long)t.n * p.G + min(t.c + j, p.C - 1) / Cg);
        m1[j] = gs[s]; m2[j] = gs[s + 1];
    }
    const long base = ((long)t.n * p.L) * p.C + t.c;
    const int rv = min(t.r1, t.len);
    for (int r = t.r0 + t.ty; r < t.r1; r += GN_U * t.TY) {
        GnBwdRow<T, VEC, CK> w[GN_U];
#pragma unroll
        for (int u = 0; u < GN_U; ++u)
            if (r + u * t.TY < rv) w[u].load(p, (long)t.n * p.L + r + u * t.TY, t.c);
#pragma unroll
        for (int u = 0; u < GN_U; ++u) {
            const int rr = r + u * t.TY;
            if (rr >= t.r1) break;
            float xh[VEC], dz[VEC], dx[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) dx[j] = 0.f;
            if (rr < rv) {
                w[u].get(p, k, xh, dz);
#pragma unroll
                for (int j = 0; j < VEC; ++j) dx[j] = k.rstd[j] * (k.gamma[j] * dz[j] - m1[j] - xh[j] * m2[j]);
            }
            store_vec((T*)p.dx + base + (long)rr * p.C, dx);
        }
    }
}

// dgamma, dbeta: sums over the rows of ws[2][rows][C] in row order.  grid ceil(C / 64), block 64 x 16
__global__ void __launch_bounds__(1024) gn_param_grad_kernel(const float* __restrict__ ws, float* __restrict__ dgamma, float* __restrict__ dbeta, long rows, int C) {
    __shared__ float s1[16][64], s2[16][64];
    const int c = blockIdx.x * 64 + threadIdx.x;
    float a = 0.f, b = 0.f;
    if (c < C)
        for (long r = threadIdx.y; r < rows; r += 16 * 8) {
            float u[8], v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const long rr = r + 16 * i < rows ? r + 16 * i : rows - 1;
                u[i] = ws[rr * C + c]; v[i] = ws[(rows + rr) * C + c];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (r + 16 * i < rows) { a += u[i]; b += v[i]; }
        }
    s1[threadIdx.y][threadIdx.x] = a; s2[threadIdx.y][threadIdx.x] = b;
    __syncthreads();
    if (threadIdx.y == 0 && c < C) {
#pragma unroll
        for (int i = 1; i < 16; ++i) { a += s1[i][threadIdx.x]; b += s2[i][threadIdx.x]; }
        if (dbeta) dbeta[c] = a;
        if (dgamma) dgamma[c] = b;
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------------
struct GnPlan { int vec, TX, strips, chunks; unsigned blocks; };
// Row chunks: enough workgroups for the 256 CUs (about four each), never more chunks than 32-row pieces of the sample.
static int gn_chunks(int N, int L, int strips) {
    long want = cdiv(1024, (long)N * strips);
    const long most = cdiv(L, 32);
    if (want > most) want = most;
    if (want > GN_CHUNKS) want = GN_CHUNKS;
    return (int)(want < 1 ? 1 : want);
}
static GnPlan gn_plan(int N, int L, int C, int vec) {
    GnPlan k;
    const int cols = cdiv(C, vec);
    k.vec = vec;
    k.TX = cols < 64 ? cols : 64;
    k.strips = cdiv(cols, k.TX);
    k.chunks = gn_chunks(N, L, k.strips);
    k.blocks = (unsigned)((long)N * k.chunks * k.strips);
    return k;
}
static int gn_check(const GroupNormArgs& p, const char* what) {
    MTTS_REQUIRE(p.N > 0 && p.L > 0 && p.C > 0 && p.G > 0, "%s: empty input (N %d, L %d, C %d, G %d)", what, p.N, p.L, p.C, p.G);
    MTTS_REQUIRE(p.C % p.G == 0, "%s: %d channels are not a multiple of %d groups", what, p.C, p.G);
    MTTS_REQUIRE(p.dtype == MTTS_F32 || p.dtype == MTTS_BF16, "%s: dtype %d is neither MTTS_F32 nor MTTS_BF16", what, p.dtype);
    MTTS_REQUIRE(p.act >= MTTS_ACT_NONE && p.act <= MTTS_ACT_SILU, "%s: unknown activation %d", what, p.act);
    MTTS_REQUIRE(p.gamma && p.beta && p.mean && p.rstd && p.ws, "%s: missing tensor", what);
    // a grid has fewer than 2^32 threads (a sample is cut into chunks only where N * strips is below 1024)
    MTTS_REQUIRE((long)p.N * cdiv(p.C, 64) < (1L << 32) / GN_T && (long)p.N * p.G < (1L << 32) / 64, "%s: %d samples x %d channels are too many for one call", what, p.N, p.C);
    return 0;
}

MTTS_API long mtts_group_norm_workspace_floats(int N, int L, int C, int G) {
    const GnPlan a = gn_plan(N, L, C, 1), b = gn_plan(N, L, C, 4), c = gn_plan(N, L, C, 8);      // the chunk count depends on the width of a strip
    long chunks = a.chunks;
    if (b.chunks > chunks) chunks = b.chunks;
    if (c.chunks > chunks) chunks = c.chunks;
    return 2L * N * chunks * C + 2L * N * G;
}

template <typename T, int VEC> static void gn_fwd_two_pass(const GroupNormArgs& p, hipStream_t s) {
    const GnPlan k = gn_plan(p.N, p.L, p.C, VEC);
    hipLaunchKernelGGL((gn_moments_kernel<T, VEC>), dim3(k.blocks), dim3(GN_T), 0, s, p, k.chunks, k.strips, k.TX);
    hipLaunchKernelGGL(gn_stats_kernel, dim3(p.N * p.G), dim3(64), 0, s, p, k.chunks);
    hipLaunchKernelGGL((gn_apply_kernel<T, VEC>), dim3(k.blocks), dim3(GN_T), 0, s, p, k.chunks, k.strips, k.TX);
}
template <typename T, int VEC, bool CK> static void gn_bwd_two_pass(const GroupNormArgs& p, hipStream_t s) {
    const GnPlan k = gn_plan(p.N, p.L, p.C, VEC);
    const long rows = (long)p.N * k.chunks;
    float* gs = p.ws + 2 * rows * p.C;
    hipLaunchKernelGGL((gn_bwd_sums_kernel<T, VEC, CK>), dim3(k.blocks), dim3(GN_T), 0, s, p, k.chunks, k.strips, k.TX);
    hipLaunchKernelGGL(gn_bwd_means_kernel, dim3(p.N * p.G), dim3(64), 0, s, p, k.chunks, gs);
    hipLaunchKernelGGL((gn_bwd_apply_kernel<T, VEC, CK>), dim3(k.blocks), dim3(GN_T), 0, s, p, k.chunks, k.strips, k.TX, (const float*)gs);
    hipLaunchKernelGGL(gn_param_grad_kernel, dim3(cdiv(p.C, 64)), dim3(64, 16), 0, s, p.ws, p.dgamma, p.dbeta, rows, p.C);
}

MTTS_API int mtts_group_norm_act_fwd(const GroupNormArgs* args, void* stream) {
    const GroupNormArgs p = *args;
    hipStream_t s = (hipStream_t)stream;
    MTTS_TRY(gn_check(p, "mtts_group_norm_act_fwd"));
    MTTS_REQUIRE(p.x && p.y && !p.q == !p.q_code, "mtts_group_norm_act_fwd: missing tensor");
    const int vec = p.dtype == MTTS_F32 ? 4 : 8;
    const bool v = p.C % vec == 0 && aligned_to(p.x, 16) && aligned_to(p.y, 16) && aligned_to(p.mask, vec);
    if (p.dtype == MTTS_F32) v ? gn_fwd_two_pass<float, 4>(p, s) : gn_fwd_two_pass<float, 1>(p, s);
    else v ? gn_fwd_two_pass<bf16_t, 8>(p, s) : gn_fwd_two_pass<bf16_t, 1>(p, s);
    MTTS_CHECK_LAUNCH("group_norm_act_fwd");
    if (p.q) MTTS_TRY(mtts_checkpoint8_pack(p.x, p.lengths, p.q, p.q_code, p.N, p.L, p.C, p.dtype, stream));
    return 0;
}

MTTS_API int mtts_group_norm_act_bwd(const GroupNormArgs* args, void* stream) {
    const GroupNormArgs p = *args;
    hipStream_t s = (hipStream_t)stream;
    MTTS_TRY(gn_check(p, "mtts_group_norm_act_bwd"));
    MTTS_REQUIRE(p.dy && p.dx && (p.q ? p.q_code != nullptr : p.x != nullptr), "mtts_group_norm_act_bwd: missing tensor");
    const int vec = p.dtype == MTTS_F32 ? 4 : 8;
    const bool v = p.C % vec == 0 && aligned_to(p.x, 16) && aligned_to(p.dy, 16) && aligned_to(p.dx, 16) && aligned_to(p.mask, vec) && aligned_to(p.q, vec);
    if (p.dtype == MTTS_F32) {
        if (p.q) v ? gn_bwd_two_pass<float, 4, true>(p, s) : gn_bwd_two_pass<float, 1, true>(p, s);
        else v ? gn_bwd_two_pass<float, 4, false>(p, s) : gn_bwd_two_pass<float, 1, false>(p, s);
    } else {
        if (p.q) v ? gn_bwd_two_pass<bf16_t, 8, true>(p, s) : gn_bwd_two_pass<bf16_t, 1, true>(p, s);
        else v ? gn_bwd_two_pass<bf16_t, 8, false>(p, s) : gn_bwd_two_pass<bf16_t, 1, false>(p, s);
    }
    MTTS_CHECK_LAUNCH("group_norm_act_bwd");
    return 0;
}
