// Group norm + activation + dropout over channel-last activations x[N, L, C] (fp32 or bf16 storage), forward and backward.
//
//   y  = drop(act(gamma * xhat + beta)),  xhat = (x - mean) * rstd; mean and variance of (sample n, group g) run over the sample's
//        lengths[n] valid rows and the group's C / G channels.  Rows behind them are never read; y and dx are zero there.
//   dz = drop'(dy) * act'(z);  dbeta = sum dz,  dgamma = sum dz * xhat  (over all valid rows of all samples)
//   dx = rstd * (gamma dz - mean(gamma dz) - xhat * mean(gamma dz * xhat))
//
// With an 8-bit checkpoint the backward takes x = q * 2^(code - 127) in place of the input; mean and rstd stay those of the forward.
// Every sum has a fixed order (no atomics) and fp32 terms; second moments are centred (an offset that is large against the spread costs
// no digits).
//
// This is bytes: read x, write y; read x (or its checkpoint) and dy, write dx.  Two forms:
//   * resident: one workgroup takes a sample's column strip (whole groups, at least 128 bytes wide), all rows in registers: one pass
//     over memory, one launch each way.  Strips of up to 8192 vectors of 16 bytes (1024 rows of 128 bytes), in the forward 12288 (1536).
//   * two-pass: rows cut into chunks; partial moments (sums) per chunk and group, merged by every workgroup of the second pass; the
//     second reading comes from the 256 MB last-level cache where the tensors fit.
// Widths or addresses that no 16-byte vector fits go one value at a time, in two passes (vectors that straddle rows, with their partial
// ends, were slower: bf16 backward at 64 x 600 x 511 65 us one by one, 158 us so).
//
// GPU time, a copy of 1 GiB running at 5.1 TB/s on the same card (tensors below 256 MB come partly from the last-level cache):
//   64 x 600 x 512 in 16 groups, tanh, fp32: forward with keep flags 44 us (177 MB, 4.0 TB/s), without them and over ragged samples 26 us
//   (138 MB, 5.2 TB/s), backward with flags 51 us (256 MB, 5.0 TB/s).  bf16, silu, ragged, with the checkpoint: forward 28 us (90 MB, 3.2
//   TB/s), backward 36 us (78 MB, 2.2 TB/s): the vector instructions of eight values to a vector, on the rows behind a length too.  Two
//   passes, 4 x 4999 rows of 512, fp32, ragged, with the checkpoint: moments 17 us (45 MB, 2.7 TB/s) + apply 15 us (76 MB, 5.2 TB/s), sums
//   17 us (44 MB, 2.5 TB/s) + apply 16 us (85 MB, 5.2 TB/s): the passes that reduce run at half of the rate of those that write.
//   The sums over samples for the gradients of scale and offset: 4 us.
#include "vec_io.h"

constexpr int GN_T = 256;          // threads of a two-pass workgroup
constexpr int GN_U = 4;            // row vectors a thread requests before it uses the first
constexpr int GN_CHUNKS = 64;      // most row chunks of a sample

// ---- activations ------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float gn_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }      // v_rcp_f32: 1 ulp
// tanh through exp loses digits next to zero (1 - e cancels): the odd polynomial there (its next term is 8.5e-9 of z at 1/4)
__device__ __forceinline__ float gn_tanh(float z) {
    const float e = __expf(-2.f * fabsf(z)), r = copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e), z), s = z * z;
    const float p = z + z * s * (-0.33333333333f + s * (0.13333333333f + s * (-0.05396825397f + s * 0.02186948854f)));
    return fabsf(z) < 0.25f ? p : r;
}
template <int ACT> __device__ __forceinline__ float gn_act(float z) {
    if constexpr (ACT == MTTS_ACT_RELU) return z < 0.f ? 0.f : z;      // NaN stays NaN
    if constexpr (ACT == MTTS_ACT_TANH) return gn_tanh(z);
    if constexpr (ACT == MTTS_ACT_SIGMOID) return gn_sigmoid(z);
    if constexpr (ACT == MTTS_ACT_SILU) return z * gn_sigmoid(z);
    return z;
}
// act'(z) of every activation from one exponential, without a branch (rows in registers, see GN_ROW_DONE): with e = exp(-k |z|),
// w = e / (1 + e)^2 = p (1 - p) and p = sigmoid(k z):  c0 + c1 w + c2 p + c3 z w, nothing at or below `floor`.  tanh: 1 - tanh^2 = 4 w at
// k = 2, no cancellation in the tails; silu: p + z p (1 - p); relu: 1 above zero, as the framework's other blocks.
struct GnSlope {
    float k, c0, c1, c2, c3, floor;
    __device__ __forceinline__ explicit GnSlope(int act) {
        k = act == MTTS_ACT_TANH ? -2.f : -1.f;
        c0 = act == MTTS_ACT_NONE || act == MTTS_ACT_RELU ? 1.f : 0.f;
        c1 = act == MTTS_ACT_TANH ? 4.f : act == MTTS_ACT_SIGMOID ? 1.f : 0.f;
        c2 = c3 = act == MTTS_ACT_SILU ? 1.f : 0.f;
        floor = act == MTTS_ACT_RELU ? 0.f : -__builtin_inff();
    }
    __device__ __forceinline__ float operator()(float z) const {
        const float e = __expf(k * fabsf(z)), r = __builtin_amdgcn_rcpf(1.f + e), w = e * r * r, p = z < 0.f ? e * r : r;
        const float s = c0 + w * (c1 + c3 * fminf(fmaxf(z, -1e30f), 1e30f)) + c2 * p;
        return z <= floor ? 0.f : s;
    }
};
// body(integral constant of the activation): one uniform branch around a whole loop over rows
template <int A> struct GnAct { static constexpr int value = A; };
template <typename F> __device__ __forceinline__ void gn_by_act(int act, F body) {
    switch (act) {
        case MTTS_ACT_RELU: body(GnAct<MTTS_ACT_RELU>()); break;
        case MTTS_ACT_TANH: body(GnAct<MTTS_ACT_TANH>()); break;
        case MTTS_ACT_SIGMOID: body(GnAct<MTTS_ACT_SIGMOID>()); break;
        case MTTS_ACT_SILU: body(GnAct<MTTS_ACT_SILU>()); break;
        default: body(GnAct<MTTS_ACT_NONE>()); break;
    }
}

// ---- geometry ---------------------------------------------------------------------------------------------------------------------
// Strip: W channels (TX vectors) that hold NG whole groups, or, where one group is wider than a workgroup, one of its `parts`.
struct GnGeo { int TX, W, NG, parts, strips, chunks; };

__device__ __forceinline__ int gn_length(const GroupNormArgs& p, int n) { return p.lengths ? min(max(p.lengths[n], 0), p.L) : p.L; }

// This workgroup's sample, chunk and strip [c0, c1), this thread's vector of channels c.. and rows ty, ty + TY, ..
struct GnTile { int n, chunk, strip, g0, c0, c1, c, tx, ty, TY, len; bool on; };
template <int VEC> __device__ __forceinline__ GnTile gn_tile(const GroupNormArgs& p, const GnGeo& k) {
    GnTile t;
    // workgroups go to the eight XCDs in turn; each XCD gets a contiguous run of strips, so that neighbouring strips (which share lines of
    // the checkpoint and pages of the rest) meet in one L2: backward at 64 x 600 x 512, fp32 60.5 -> 55 us
    const unsigned per = gridDim.x >> 3, rem = gridDim.x & 7, xcd = blockIdx.x & 7;
    unsigned b = xcd * per + min(xcd, rem) + (blockIdx.x >> 3);
    t.strip = b % k.strips; b /= k.strips;
    t.chunk = b % k.chunks; t.n = b / k.chunks;
    const int Cg = p.C / p.G;
    if (k.parts > 1) { t.g0 = t.strip / k.parts; t.c0 = t.g0 * Cg + (t.strip - t.g0 * k.parts) * k.W; t.c1 = min(t.c0 + k.W, (t.g0 + 1) * Cg); }
    else { t.c0 = t.strip * k.W; t.g0 = t.c0 / Cg; t.c1 = min(t.c0 + k.W, p.C); }
    t.TY = blockDim.x / k.TX;
    t.ty = threadIdx.x / k.TX; t.tx = threadIdx.x - t.ty * k.TX;
    t.c = t.c0 + t.tx * VEC;
    t.on = t.ty < t.TY && t.c < t.c1;
    t.len = gn_length(p, t.n);
    return t;
}

// out(s) = sum over e < E of in(s, e) for s < S, by the whole workgroup: P = 2^lp neighbouring lanes to a sum.
__device__ __forceinline__ int gn_lanes(int S, int E) {
    int lp = 0;
    while (lp < 6 && (2 << lp) * S <= (int)blockDim.x && (2 << lp) <= E) ++lp;
    return lp;
}
template <typename In, typename Out> __device__ __forceinline__ void gn_block_sums(int S, int E, In in, Out out) {
    const int lp = gn_lanes(S, E), P = 1 << lp, lane = threadIdx.x & (P - 1), each = blockDim.x >> lp;
    for (int s0 = 0; s0 < S; s0 += each) {
        const int s = s0 + (threadIdx.x >> lp);
        float a = 0.f;
        if (s < S)
            for (int e = lane; e < E; e += P) a += in(s, e);
        for (int d = 1; d < P; d *= 2) a += __shfl_xor(a, d, 64);
        if (s < S && lane == 0) out(s, a);
    }
}

// ---- resident form ----------------------------------------------------------------------------------------------------------------
// R row vectors in registers per thread.  Loads and stores go through buffer descriptors of the sample: a load behind the sample's
// length returns zero, a store behind row L is dropped.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t gn_rsrc(const void* base, long offset, long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((char*)const_cast<void*>(base) + offset, 0, (int)bytes, 0x00020000);
}
constexpr unsigned GN_OUT = 0x80000000u;       // an offset behind every sample (they are below 2^31 bytes)

// The register budget of these kernels is the rows they hold: rows are worked off one after the other (the scheduler would otherwise
// interleave them all), and packed words are unpacked again in every phase instead of being kept unpacked.
#define GN_ROW_DONE __builtin_amdgcn_sched_barrier(0)
// TAG keeps the rows of the activations' branches apart: what they have in common must not move in front of the branch for all rows.
template <int TAG = -1, typename V> __device__ __forceinline__ void gn_forget(V& w) {
    constexpr int N = sizeof(V) / 4;
    if constexpr (N == 1) asm volatile("" : "+v"(w) : "n"(TAG));
    else {
#pragma unroll
        for (int i = 0; i < N; ++i) { unsigned u = w[i]; asm volatile("" : "+v"(u) : "n"(TAG)); w[i] = u; }
    }
}

// A running sum is taken here: its additions must not sink, with all their terms, to the place where the sum is used.
__device__ __forceinline__ void gn_pin(float& v) { asm volatile("" : "+v"(v)); }

// Element offsets of a thread's rows in its sample, one after the other; a thread without a vector stays at GN_OUT.
struct GnWalk {
    unsigned at, step; bool on;
    __device__ __forceinline__ GnWalk(const GroupNormArgs& p, const GnTile& t) {
        on = t.on; at = on ? (unsigned)t.ty * p.C + t.c : 0u; step = (unsigned)t.TY * p.C;
    }
    __device__ __forceinline__ void next() { at += step; }
    __device__ __forceinline__ unsigned bytes(int size) const { return on ? at * size : GN_OUT; }
    __device__ __forceinline__ void forget() { asm volatile("" : "+v"(at)); }      // counted again, not kept from the loads
};

__device__ __forceinline__ float gn_drop(const GroupNormArgs& p, unsigned keep, float v) { return !p.mask ? v : keep ? v * p.mask_scale : 0.f; }

// STR: a vector may straddle groups (statistics per channel of the vector, else one set per thread)
template <typename T, int VEC, int R, bool STR>
__global__ void __launch_bounds__(R > 12 ? 512 : 1024) gn_fwd_kernel(GroupNormArgs p, GnGeo k) {
    constexpr int SZ = sizeof(T), K = STR ? VEC : 1;
    extern __shared__ float lds[];
    const GnTile t = gn_tile<VEC>(p, k);
    const int Cg = p.C / p.G, LG = STR ? Cg : Cg / VEC, E = t.TY * LG;      // partial values of a group
    const long base = (long)t.n * p.L * p.C;
    const GnWalk w0(p, t);
    float* const red = lds;                                                   // [2][NG][E]
    float* const stat = lds + 2 * k.NG * E;                                   // [3][NG]: mean, its correction, second moment
    Raw<T, VEC> x[R]; Bytes<VEC> keep[R];
    {
        const __amdgpu_buffer_rsrc_t rx = gn_rsrc(p.x, base * SZ, (long)t.len * p.C * SZ), rm = gn_rsrc(p.mask ? (const void*)p.mask : p.x, p.mask ? base : 0, p.mask ? (long)t.len * p.C : 0);
        GnWalk w = w0;
#pragma unroll
        for (int i = 0; i < R; ++i, w.next()) {
            x[i].load(rx, w.bytes(SZ));
            if (p.mask) keep[i].load(rm, w.bytes(1));
        }
    }
    const int valid = t.on ? (t.len - t.ty + t.TY - 1) / t.TY : 0;            // of this thread's rows
    int gl[K], slot[K];                                                       // group inside the strip; place among its partial values
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const int cc = t.tx * VEC + j;
        gl[j] = STR ? cc / Cg : t.tx / LG;
        slot[j] = gl[j] * E + t.ty * LG + (STR ? cc - gl[j] * Cg : t.tx - gl[j] * LG);
    }
    const float count = (float)t.len * (float)Cg, inv = count > 0.f ? 1.f / count : 0.f;
    // mean
#pragma unroll
    for (int j = 0; j < K; ++j) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            GN_ROW_DONE;
            float v = 0.f;
#pragma unroll
            for (int q = 0; q < VEC / K; ++q) v += x[i].at(STR ? j : q);
            s += v;
            gn_pin(s);
        }
        if (t.ty < t.TY) red[slot[j]] = s;
    }
    __syncthreads();
    gn_block_sums(k.NG, E, [&](int g, int e) { return red[g * E + e]; }, [&](int g, float a) { stat[g] = a * inv; });
    __syncthreads();
    // deviations from it: their sum corrects the mean, their squares are the second moment
    float mean[K], rstd[K];
#pragma unroll
    for (int i = 0; i < R; ++i) gn_forget(x[i].w);
#pragma unroll
    for (int j = 0; j < K; ++j) {
        mean[j] = stat[gl[j]];
        float s = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            GN_ROW_DONE;
#pragma unroll
            for (int q = 0; q < VEC / K; ++q) {
                const float d = i < valid ? x[i].at(STR ? j : q) - mean[j] : 0.f;
                s += d; s2 += d * d;
            }
            gn_pin(s); gn_pin(s2);
        }
        if (t.ty < t.TY) { red[slot[j]] = s; red[k.NG * E + slot[j]] = s2; }
    }
    __syncthreads();
    gn_block_sums(2 * k.NG, E, [&](int g, int e) { return red[g * E + e]; }, [&](int g, float a) { stat[k.NG + g] = a * inv; });
    __syncthreads();
    if (threadIdx.x < k.NG && t.g0 + threadIdx.x < p.G) {
        const float d = stat[k.NG + threadIdx.x], v = stat[2 * k.NG + threadIdx.x] - d * d;
        const long g = (long)t.n * p.G + t.g0 + threadIdx.x;
        p.mean[g] = stat[threadIdx.x] + d; p.rstd[g] = 1.f / sqrtf((v < 0.f ? 0.f : v) + p.eps);      // NaN stays NaN
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const float d = stat[k.NG + gl[j]], v = stat[2 * k.NG + gl[j]] - d * d;
        mean[j] += d; rstd[j] = 1.f / sqrtf((v < 0.f ? 0.f : v) + p.eps);      // NaN stays NaN
    }
    float gamma[VEC], beta[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) { gamma[j] = p.gamma[min(t.c + j, p.C - 1)]; beta[j] = p.beta[min(t.c + j, p.C - 1)]; }
    const __amdgpu_buffer_rsrc_t ry = gn_rsrc(p.y, base * SZ, (long)p.L * p.C * SZ);
    gn_by_act(p.act, [&](auto act) __attribute__((always_inline)) {
        GnWalk w = w0;
        w.forget();
#pragma unroll
        for (int i = 0; i < R; ++i, w.next()) {
            GN_ROW_DONE;
            Raw<T, VEC> v = x[i];
            gn_forget<act.value>(v.w);
            float f[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float z = gn_act<act.value>((v.at(j) - mean[STR ? j : 0]) * rstd[STR ? j : 0] * gamma[j] + beta[j]);
                f[j] = i < valid ? gn_drop(p, keep[i].get(j), z) : 0.f;
            }
            stream_vec(ry, w.bytes(SZ), f);
        }
    });
    if (!p.q) return;
    // the checkpoint: a block's lanes are neighbours (W is a multiple of 32 channels, see gn_plan)
    const int nb = (p.C + CK_BLOCK - 1) / CK_BLOCK;
    const __amdgpu_buffer_rsrc_t rq = gn_rsrc(p.q, base, (long)p.L * p.C), rc = gn_rsrc(p.q_code, (long)t.n * p.L * nb, (long)p.L * nb);
    GnWalk w = w0;
    w.forget();
    unsigned at_c = t.on && (t.c & (CK_BLOCK - 1)) == 0 ? (unsigned)t.ty * nb + t.c / CK_BLOCK : GN_OUT;
    const unsigned step_c = at_c == GN_OUT ? 0u : (unsigned)t.TY * nb;
#pragma unroll
    for (int i = 0; i < R; ++i, w.next()) {
        GN_ROW_DONE;
        Raw<T, VEC> v = x[i];
        gn_forget(v.w);
        unsigned m = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) m = umax_(m, abs_bits(v.at(j)));
        const unsigned code = ck_code(block_max<CK_BLOCK / VEC>(m));
        ck_store(rq, w.bytes(1), v, code);
        __builtin_amdgcn_raw_buffer_store_b8((uint8_t)code, rc, at_c, 0, 0);
        at_c += step_c;
    }
}

// xhat and dz of one row vector
template <typename T, int VEC, int K> __device__ __forceinline__ void gn_dz(const GroupNormArgs& p, const GnSlope& slope, const float (&mean)[K], const float (&rstd)[K], const float (&gamma)[VEC], const float (&beta)[VEC],
                                                                           const Bytes<VEC>& keep, const Raw<T, VEC>& dy, const float (&x)[VEC], float (&xhat)[VEC], float (&dz)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const float u = (x[j] - mean[K > 1 ? j : 0]) * rstd[K > 1 ? j : 0];
        xhat[j] = u;
        dz[j] = gn_drop(p, keep.get(j), dy.at(j)) * slope(u * gamma[j] + beta[j]);
    }
}

// x of one row vector: the input's own, or its checkpoint
template <typename T, int VEC, bool CK> struct GnX;
template <typename T, int VEC> struct GnX<T, VEC, false> {
    Raw<T, VEC> w;
    __device__ __forceinline__ void get(float (&f)[VEC]) const { get_vec(w, f); }
};
template <typename T, int VEC> struct GnX<T, VEC, true> {
    Bytes<VEC> w; unsigned code;
    __device__ __forceinline__ void get(float (&f)[VEC]) const {
        const float s = ck_scale(code);
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = ck_value(w.get(j), s);
    }
};

// The backward keeps x as it lies in memory and dz in fp32; per-channel sums of dz and dz * xhat go to ws [2][N][C], and through gamma
// to the two means of the group.  (bf16, 16 rows, straddling vectors, no checkpoint: 13 registers spill, 56 bytes a lane.)
template <typename T, int VEC, int R, bool STR, bool CK>
__global__ void __launch_bounds__(512) gn_bwd_kernel(GroupNormArgs p, GnGeo k) {
    constexpr int SZ = sizeof(T), K = STR ? VEC : 1;
    extern __shared__ float lds[];
    const GnTile t = gn_tile<VEC>(p, k);
    const int Cg = p.C / p.G, nb = (p.C + CK_BLOCK - 1) / CK_BLOCK, TS = t.TY * k.TX;
    const long base = (long)t.n * p.L * p.C;
    const GnWalk w0(p, t);
    float* const red = lds;                                                   // [2][VEC][TY][TX]
    float* const tot = lds + 2 * VEC * TS;                                    // [2][W]
    float* const mid = tot + 2 * k.W;                                         // [2][NG]
    GnX<T, VEC, CK> x[R]; Raw<T, VEC> dy[R]; Bytes<VEC> keep[R];
    {
        const long rows = t.len;
        const __amdgpu_buffer_rsrc_t rd = gn_rsrc(p.dy, base * SZ, rows * p.C * SZ), rx = CK ? gn_rsrc(p.q, base, rows * p.C) : gn_rsrc(p.x, base * SZ, rows * p.C * SZ);
        const __amdgpu_buffer_rsrc_t rc = CK ? gn_rsrc(p.q_code, (long)t.n * p.L * nb, rows * nb) : rd, rm = gn_rsrc(p.mask ? (const void*)p.mask : p.dy, p.mask ? base : 0, p.mask ? rows * p.C : 0);
        GnWalk w = w0;
        unsigned at_c = t.on ? (unsigned)t.ty * nb + t.c / CK_BLOCK : GN_OUT;
        const unsigned step_c = t.on ? (unsigned)t.TY * nb : 0u;
#pragma unroll
        for (int i = 0; i < R; ++i, w.next()) {
            dy[i].load(rd, w.bytes(SZ));
            x[i].w.load(rx, w.bytes(CK ? 1 : SZ));
            if constexpr (CK) { x[i].code = __builtin_amdgcn_raw_buffer_load_b8(rc, at_c, 0, 0); at_c += step_c; }
            if (p.mask) keep[i].load(rm, w.bytes(1));
        }
    }
    const int valid = t.on ? (t.len - t.ty + t.TY - 1) / t.TY : 0;
    int gl[K]; float mean[K], rstd[K], gamma[VEC], beta[VEC];
#pragma unroll
    for (int j = 0; j < K; ++j) {
        gl[j] = (t.tx * VEC + j) / Cg;
        const long g = (long)t.n * p.G + min(t.g0 + gl[j], p.G - 1);
        mean[j] = p.mean[g]; rstd[j] = p.rstd[g];
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) { gamma[j] = p.gamma[min(t.c + j, p.C - 1)]; beta[j] = p.beta[min(t.c + j, p.C - 1)]; }
    float dz[R][VEC], s1[VEC], s2[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) s1[j] = s2[j] = 0.f;
    const GnSlope slope(p.act);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        GN_ROW_DONE;
        float f[VEC], xh[VEC], d[VEC];
        x[i].get(f);
        gn_dz<T, VEC, K>(p, slope, mean, rstd, gamma, beta, keep[i], dy[i], f, xh, d);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float v = i < valid ? d[j] : 0.f;
            dz[i][j] = v;
            s1[j] += v; s2[j] += i < valid ? v * xh[j] : 0.f;
            gn_pin(s1[j]); gn_pin(s2[j]);
        }
    }
    if (t.ty < t.TY) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) { red[j * TS + threadIdx.x] = s1[j]; red[(VEC + j) * TS + threadIdx.x] = s2[j]; }
    }
    __syncthreads();
    gn_block_sums(2 * k.W, t.TY,
                  [&](int s, int e) { const int h = s >= k.W, cc = s - h * k.W; return red[(h * VEC + cc % VEC) * TS + e * k.TX + cc / VEC]; },
                  [&](int s, float a) {
                      const int h = s >= k.W, cc = s - h * k.W, c = t.c0 + cc;
                      tot[s] = c < p.C ? a * p.gamma[c] : 0.f;
                      if (c < p.C) p.ws[((long)h * p.N + t.n) * p.C + c] = a;
                  });
    __syncthreads();
    const float count = (float)t.len * (float)Cg, inv = count > 0.f ? 1.f / count : 0.f;
    gn_block_sums(2 * k.NG, Cg, [&](int s, int e) { const int h = s >= k.NG; return tot[h * k.W + (s - h * k.NG) * Cg + e]; }, [&](int s, float a) { mid[s] = a * inv; });
    __syncthreads();
    float m1[K], m2[K];
#pragma unroll
    for (int j = 0; j < K; ++j) { m1[j] = mid[gl[j]]; m2[j] = mid[k.NG + gl[j]]; }
    const __amdgpu_buffer_rsrc_t ro = gn_rsrc(p.dx, base * SZ, (long)p.L * p.C * SZ);
    GnWalk w = w0;
    w.forget();
#pragma unroll
    for (int i = 0; i < R; ++i, w.next()) {
        GN_ROW_DONE;
        GnX<T, VEC, CK> xi = x[i];
        gn_forget(xi.w.w);
        float f[VEC], dx[VEC];
        xi.get(f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const int u = STR ? j : 0;
            const float xh = (f[j] - mean[u]) * rstd[u];
            dx[j] = i < valid ? rstd[u] * (gamma[j] * dz[i][j] - m1[u] - xh * m2[u]) : 0.f;
        }
        stream_vec(ro, w.bytes(SZ), dx);
    }
}

// ---- two-pass form ----------------------------------------------------------------------------------------------------------------
struct Moments { float n, mean, m2; };
__device__ __forceinline__ Moments gn_merge(const Moments& a, const Moments& b) {
    const float n = a.n + b.n;
    if (b.n == 0.f) return a;
    if (a.n == 0.f) return b;
    const float d = b.mean - a.mean, w = b.n * __builtin_amdgcn_rcpf(n);
    return Moments{n, a.mean + d * w, a.m2 + b.m2 + d * d * a.n * w};
}
__device__ __forceinline__ Moments gn_wave_merge(Moments m, int P) {
    for (int d = 1; d < P; d *= 2) m = gn_merge(m, Moments{__shfl_xor(m.n, d, 64), __shfl_xor(m.mean, d, 64), __shfl_xor(m.m2, d, 64)});
    return m;
}

// Moments of (sample, group, chunk, part) -> ws[((n * G + g) * chunks + chunk) * parts + part], three floats.  CK: the checkpoint of the
// same rows on the way.
template <typename T, int VEC, bool STR, bool CK>
__global__ void __launch_bounds__(GN_T) gn_moments_kernel(GroupNormArgs p, GnGeo k) {
    constexpr int K = STR ? VEC : 1;
    __shared__ float rn[GN_T * K], rm[GN_T * K], r2[GN_T * K];
    const GnTile t = gn_tile<VEC>(p, k);
    const int per = (p.L + k.chunks - 1) / k.chunks, r0 = t.chunk * per, r1 = min(p.L, r0 + per), rv = min(r1, t.len), nb = (p.C + CK_BLOCK - 1) / CK_BLOCK;
    const long first = (long)t.n * p.L;
    Moments m[K];
#pragma unroll
    for (int j = 0; j < K; ++j) m[j] = Moments{0.f, 0.f, 0.f};
    for (int r = r0 + t.ty; r - t.ty < (CK ? r1 : rv); r += GN_U * t.TY) {      // whole workgroups: the lanes of a block stay together
        Raw<T, VEC> v[GN_U];
#pragma unroll
        for (int u = 0; u < GN_U; ++u) {
            v[u].zero();
            if (t.on && r + u * t.TY < rv) v[u].load((const T*)p.x + (first + r + u * t.TY) * p.C + t.c);
        }
        const int left = (rv - r + t.TY - 1) / t.TY, n = !t.on || r >= rv ? 0 : left < GN_U ? left : GN_U;
        if (n > 0) {
            const float inv = 1.f / (float)(n * (VEC / K));
#pragma unroll
            for (int j = 0; j < K; ++j) {
                float s = 0.f, q = 0.f;
#pragma unroll
                for (int u = 0; u < GN_U; ++u)
#pragma unroll
                    for (int e = 0; e < VEC / K; ++e) s += v[u].at(STR ? j : e);          // zero behind the length
                s *= inv;
#pragma unroll
                for (int u = 0; u < GN_U; ++u)
#pragma unroll
                    for (int e = 0; e < VEC / K; ++e) { const float d = u < n ? v[u].at(STR ? j : e) - s : 0.f; q += d * d; }
                m[j] = gn_merge(m[j], Moments{(float)(n * (VEC / K)), s, q});
            }
        }
        if constexpr (CK) {
#pragma unroll
            for (int u = 0; u < GN_U; ++u) {
                unsigned top = 0;
#pragma unroll
                for (int j = 0; j < VEC; ++j) top = umax_(top, abs_bits(v[u].at(j)));
                const unsigned code = ck_code(block_max<CK_BLOCK / VEC>(top));
                const int rr = r + u * t.TY;
                if (t.on && rr < r1) {
                    ck_store(p.q + (first + rr) * p.C + t.c, v[u], code, VEC);
                    if ((t.c & (CK_BLOCK - 1)) == 0) p.q_code[(first + rr) * nb + t.c / CK_BLOCK] = (uint8_t)code;
                }
            }
        }
    }
    const int Cg = p.C / p.G, wide = k.parts > 1 ? k.W : Cg, LG = STR ? wide : wide / VEC, E = t.TY * LG;
    if (t.ty < t.TY) {
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int cc = STR ? t.tx * VEC + j : t.tx, g = cc / LG, at = g * E + t.ty * LG + cc - g * LG;
            rn[at] = m[j].n; rm[at] = m[j].mean; r2[at] = m[j].m2;
        }
    }
    __syncthreads();
    const int lp = gn_lanes(k.NG, E), P = 1 << lp, lane = threadIdx.x & (P - 1), each = GN_T >> lp, entries = k.chunks * k.parts;
    for (int g0 = 0; g0 < k.NG; g0 += each) {
        const int g = g0 + (threadIdx.x >> lp);
        Moments a = {0.f, 0.f, 0.f};
        if (g < k.NG)
            for (int e = lane; e < E; e += P) a = gn_merge(a, Moments{rn[g * E + e], rm[g * E + e], r2[g * E + e]});
        a = gn_wave_merge(a, P);
        if (g < k.NG && lane == 0 && t.g0 + g < p.G) {
            float* ws = p.ws + 3 * (((long)t.n * p.G + t.g0 + g) * entries + t.chunk * k.parts + (k.parts > 1 ? t.strip - t.g0 * k.parts : 0));
            ws[0] = a.n; ws[1] = a.mean; ws[2] = a.m2;
        }
    }
}

// y = drop(act(gamma (x - mean) rstd + beta)); the groups' moments are merged first
template <typename T, int VEC, bool STR>
__global__ void __launch_bounds__(GN_T) gn_apply_kernel(GroupNormArgs p, GnGeo k) {
    constexpr int K = STR ? VEC : 1;
    __shared__ float stat[2 * GN_T * VEC];
    const GnTile t = gn_tile<VEC>(p, k);
    const int entries = k.chunks * k.parts, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, Cg = p.C / p.G;
    for (int g = wave; g < k.NG && t.g0 + g < p.G; g += GN_T / 64) {
        const long at = (long)t.n * p.G + t.g0 + g;
        const float* ws = p.ws + 3 * at * entries;
        Moments a = {0.f, 0.f, 0.f};
        for (int e = lane; e < entries; e += 64) a = gn_merge(a, Moments{ws[3 * e], ws[3 * e + 1], ws[3 * e + 2]});
        a = gn_wave_merge(a, 64);
        if (lane == 0) {
            const float rstd = 1.f / sqrtf((a.n > 0.f ? a.m2 / a.n : 0.f) + p.eps);
            stat[2 * g] = a.mean; stat[2 * g + 1] = rstd;
            if (t.chunk == 0 && (k.parts == 1 || t.strip == t.g0 * k.parts)) { p.mean[at] = a.mean; p.rstd[at] = rstd; }
        }
    }
    __syncthreads();
    if (!t.on) return;
    float mean[K], rstd[K], gamma[VEC], beta[VEC];
#pragma unroll
    for (int j = 0; j < K; ++j) { const int g = k.parts > 1 ? 0 : (t.tx * VEC + j) / Cg; mean[j] = stat[2 * g]; rstd[j] = stat[2 * g + 1]; }
#pragma unroll
    for (int j = 0; j < VEC; ++j) { gamma[j] = p.gamma[t.c + j]; beta[j] = p.beta[t.c + j]; }
    const int per = (p.L + k.chunks - 1) / k.chunks, r0 = t.chunk * per, r1 = min(p.L, r0 + per), rv = min(r1, t.len);
    const long base = (long)t.n * p.L * p.C + t.c;
    gn_by_act(p.act, [&](auto act) __attribute__((always_inline)) {
        for (int r = r0 + t.ty; r < r1; r += GN_U * t.TY) {
            Raw<T, VEC> v[GN_U]; Bytes<VEC> keep[GN_U];
#pragma unroll
            for (int u = 0; u < GN_U; ++u) {
                const int rr = r + u * t.TY;
                v[u].zero(); keep[u].fill(1);
                if (rr < rv) {
                    v[u].load((const T*)p.x + base + (long)rr * p.C);
                    if (p.mask) keep[u].load(p.mask + base + (long)rr * p.C);
                }
            }
#pragma unroll
            for (int u = 0; u < GN_U; ++u) {
                const int rr = r + u * t.TY;
                if (rr >= r1) break;
                float f[VEC];
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float z = gn_act<act.value>((v[u].at(j) - mean[STR ? j : 0]) * rstd[STR ? j : 0] * gamma[j] + beta[j]);
                    f[j] = rr < rv ? gn_drop(p, keep[u].get(j), z) : 0.f;
                }
                stream_vec((T*)p.y + base + (long)rr * p.C, f);
            }
        }
    });
}

// GN_U rows of the backward, requested together
template <typename T, int VEC, bool CK> struct GnRows {
    GnX<T, VEC, CK> x[GN_U]; Raw<T, VEC> dy[GN_U]; Bytes<VEC> keep[GN_U];
    __device__ __forceinline__ void load(const GroupNormArgs& p, long first, int r, int TY, int rv, int c) {
        const int nb = (p.C + CK_BLOCK - 1) / CK_BLOCK;
#pragma unroll
        for (int u = 0; u < GN_U; ++u) {
            const long row = first + min(r + u * TY, rv - 1), at = row * p.C + c;
            dy[u].load((const T*)p.dy + at);
            if constexpr (CK) { x[u].w.load(p.q + at); x[u].code = p.q_code[row * nb + c / CK_BLOCK]; }
            else x[u].w.load((const T*)p.x + at);
            if (p.mask) keep[u].load(p.mask + at);
        }
    }
};
template <int VEC, int K> struct GnCol {
    float mean[K], rstd[K], gamma[VEC], beta[VEC];
    __device__ __forceinline__ void load(const GroupNormArgs& p, const GnTile& t) {
        const int Cg = p.C / p.G;
#pragma unroll
        for (int j = 0; j < K; ++j) { const long g = (long)t.n * p.G + min(t.c + j, p.C - 1) / Cg; mean[j] = p.mean[g]; rstd[j] = p.rstd[g]; }
#pragma unroll
        for (int j = 0; j < VEC; ++j) { gamma[j] = p.gamma[min(t.c + j, p.C - 1)]; beta[j] = p.beta[min(t.c + j, p.C - 1)]; }
    }
};

// Sums of dz and dz * xhat per (sample, chunk, channel) -> ws [2][N * chunks][C]; through gamma per (sample, group, chunk, part) -> gs
template <typename T, int VEC, bool STR, bool CK>
__global__ void __launch_bounds__(GN_T) gn_bwd_sums_kernel(GroupNormArgs p, GnGeo k, float* gs) {
    __shared__ float red[2 * VEC * GN_T];
    __shared__ float tot[2 * VEC * GN_T];
    const GnTile t = gn_tile<VEC>(p, k);
    const int per = (p.L + k.chunks - 1) / k.chunks, r0 = t.chunk * per, r1 = min(p.L, r0 + per), rv = min(r1, t.len), TS = t.TY * k.TX, Cg = p.C / p.G;
    float s1[VEC], s2[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) s1[j] = s2[j] = 0.f;
    if (t.on) {
        GnCol<VEC, STR ? VEC : 1> col;
        col.load(p, t);
        const GnSlope slope(p.act);
        for (int r = r0 + t.ty; r < rv; r += GN_U * t.TY) {
            GnRows<T, VEC, CK> w;
            w.load(p, (long)t.n * p.L, r, t.TY, rv, t.c);
#pragma unroll
            for (int u = 0; u < GN_U; ++u) {
                if (r + u * t.TY >= rv) break;
                float f[VEC], xh[VEC], dz[VEC];
                w.x[u].get(f);
                gn_dz<T, VEC, STR ? VEC : 1>(p, slope, col.mean, col.rstd, col.gamma, col.beta, w.keep[u], w.dy[u], f, xh, dz);
#pragma unroll
                for (int j = 0; j < VEC; ++j) { s1[j] += dz[j]; s2[j] += dz[j] * xh[j]; }
            }
        }
    }
    if (t.ty < t.TY) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) { red[j * TS + threadIdx.x] = s1[j]; red[(VEC + j) * TS + threadIdx.x] = s2[j]; }
    }
    __syncthreads();
    const long rows = (long)p.N * k.chunks;
    gn_block_sums(2 * k.W, t.TY,
                  [&](int s, int e) { const int h = s >= k.W, cc = s - h * k.W; return red[(h * VEC + cc % VEC) * TS + e * k.TX + cc / VEC]; },
                  [&](int s, float a) {
                      const int h = s >= k.W, cc = s - h * k.W, c = t.c0 + cc;
                      tot[s] = c < t.c1 ? a * p.gamma[c] : 0.f;
                      if (c < t.c1) p.ws[(h * rows + (long)t.n * k.chunks + t.chunk) * p.C + c] = a;
                  });
    __syncthreads();
    const int wide = k.parts > 1 ? k.W : Cg, entries = k.chunks * k.parts;
    gn_block_sums(2 * k.NG, wide, [&](int s, int e) { const int h = s >= k.NG; return tot[h * k.W + (s - h * k.NG) * wide + e]; },
                  [&](int s, float a) {
                      const int h = s >= k.NG, g = t.g0 + s - h * k.NG;
                      if (g < p.G) gs[2 * (((long)t.n * p.G + g) * entries + t.chunk * k.parts + (k.parts > 1 ? t.strip - t.g0 * k.parts : 0)) + h] = a;
                  });
}

template <typename T, int VEC, bool STR, bool CK>
__global__ void __launch_bounds__(GN_T) gn_bwd_apply_kernel(GroupNormArgs p, GnGeo k, const float* gs) {
    constexpr int K = STR ? VEC : 1;
    __shared__ float mid[2 * GN_T * VEC];
    const GnTile t = gn_tile<VEC>(p, k);
    const int entries = k.chunks * k.parts, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, Cg = p.C / p.G;
    const float count = (float)t.len * (float)Cg, inv = count > 0.f ? 1.f / count : 0.f;
    for (int g = wave; g < k.NG && t.g0 + g < p.G; g += GN_T / 64) {
        const float* at = gs + 2 * ((long)t.n * p.G + t.g0 + g) * entries;
        float a = 0.f, b = 0.f;
        for (int e = lane; e < entries; e += 64) { a += at[2 * e]; b += at[2 * e + 1]; }
        a = wave_sum(a); b = wave_sum(b);
        if (lane == 0) { mid[2 * g] = a * inv; mid[2 * g + 1] = b * inv; }
    }
    __syncthreads();
    if (!t.on) return;
    GnCol<VEC, K> col;
    col.load(p, t);
    float m1[K], m2[K];
#pragma unroll
    for (int j = 0; j < K; ++j) { const int g = k.parts > 1 ? 0 : (t.tx * VEC + j) / Cg; m1[j] = mid[2 * g]; m2[j] = mid[2 * g + 1]; }
    const int per = (p.L + k.chunks - 1) / k.chunks, r0 = t.chunk * per, r1 = min(p.L, r0 + per), rv = min(r1, t.len);
    const long base = (long)t.n * p.L * p.C + t.c;
    const GnSlope slope(p.act);
    for (int r = r0 + t.ty; r < r1; r += GN_U * t.TY) {
        GnRows<T, VEC, CK> w;
        if (r < rv) w.load(p, (long)t.n * p.L, r, t.TY, rv, t.c);
#pragma unroll
        for (int u = 0; u < GN_U; ++u) {
            const int rr = r + u * t.TY;
            if (rr >= r1) break;
            float f[VEC], xh[VEC], dz[VEC], dx[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) dx[j] = 0.f;
            if (rr < rv) {
                w.x[u].get(f);
                gn_dz<T, VEC, K>(p, slope, col.mean, col.rstd, col.gamma, col.beta, w.keep[u], w.dy[u], f, xh, dz);
#pragma unroll
                for (int j = 0; j < VEC; ++j) { const int v = STR ? j : 0; dx[j] = col.rstd[v] * (col.gamma[j] * dz[j] - m1[v] - xh[j] * m2[v]); }
            }
            stream_vec((T*)p.dx + base + (long)rr * p.C, dx);
        }
    }
}

// Sums over the rows of ws[2][rows][C] in row order, every `stride`-th row of a piece: into the piece's first row, or (TO_GRAD, one piece)
// into dgamma and dbeta.  grid (ceil(C / 64), pieces), block 64 x 16
constexpr int GN_PIECE = 256;
template <bool TO_GRAD>
__global__ void __launch_bounds__(1024) gn_param_grad_kernel(float* ws, float* __restrict__ dgamma, float* __restrict__ dbeta, long rows, int C, long piece, int stride) {
    __shared__ float s1[16][64], s2[16][64];
    const int c = blockIdx.x * 64 + threadIdx.x;
    const long first = blockIdx.y * piece * stride, n = min(piece, (rows - first + stride - 1) / stride);
    float* const w1 = ws + first * C + c;
    float* const w2 = w1 + rows * C;
    float a = 0.f, b = 0.f;
    if (c < C)
        for (long r = threadIdx.y; r < n; r += 16 * 8) {
            float u[8], v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const long rr = (r + 16 * i < n ? r + 16 * i : n - 1) * stride;
                u[i] = w1[rr * C]; v[i] = w2[rr * C];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (r + 16 * i < n) { a += u[i]; b += v[i]; }
        }
    s1[threadIdx.y][threadIdx.x] = a; s2[threadIdx.y][threadIdx.x] = b;
    __syncthreads();                             // every row of the piece has been read
    if (threadIdx.y == 0 && c < C) {
#pragma unroll
        for (int i = 1; i < 16; ++i) { a += s1[i][threadIdx.x]; b += s2[i][threadIdx.x]; }
        if constexpr (TO_GRAD) {
            if (dbeta) dbeta[c] = a;
            if (dgamma) dgamma[c] = b;
        } else {
            *w1 = a; *w2 = b;
        }
    }
}
// One launch for up to 1024 rows, else pieces first: whole backward at 4096 samples of 16 rows, 512 channels 138 -> 106 us, at 4096 x 16 x 64
// 56 -> 22 us, at 1200 x 1 x 512 33 -> 25 us.
static int gn_param_grad(const GroupNormArgs& p, long rows, hipStream_t s) {
    const int tiles = cdiv(p.C, 64);
    int stride = 1;
    if (rows > 4 * GN_PIECE) {
        const long pieces = (rows + GN_PIECE - 1) / GN_PIECE;
        hipLaunchKernelGGL(gn_param_grad_kernel<false>, dim3(tiles, (unsigned)pieces), dim3(64, 16), 0, s, p.ws, nullptr, nullptr, rows, p.C, (long)GN_PIECE, 1);
        stride = GN_PIECE;
    }
    hipLaunchKernelGGL(gn_param_grad_kernel<true>, dim3(tiles), dim3(64, 16), 0, s, p.ws, p.dgamma, p.dbeta, rows, p.C, rows, stride);
    return 0;
}

// ---- host -------------------------------------------------------------------------------------------------------------------------
struct GnPlan { GnGeo geo; int vec, threads, R; bool resident, str, fuse; unsigned blocks; };
static int gn_lcm(int a, int b) { int x = a, y = b; while (y) { const int r = x % y; x = y; y = r; } return a / x * b; }

// vec: 16-byte vectors where width and addresses allow them, else single values.  slots: most vectors of a resident strip.
static GnPlan gn_plan(const GroupNormArgs& p, bool wide, bool bwd) {
    GnPlan k;
    GnGeo& g = k.geo;
    const int Cg = p.C / p.G, full = p.dtype == MTTS_F32 ? 4 : 8, sz = p.dtype == MTTS_F32 ? 4 : 2;
    wide = wide && p.C % full == 0 && (gn_lcm(Cg, full) <= GN_T * full || Cg % full == 0);
    k.vec = wide ? full : 1;
    k.str = Cg % k.vec != 0;
    // A strip: whole groups and vectors, whole checkpoint blocks where that is not much wider, and at least a 128-byte line of a row (the
    // bf16 backward: 64 bytes and two workgroups to a CU, 41 -> 35 us at 64 x 600 x 512).  The same with and without a checkpoint, so
    // that y does not depend on it.
    const int unit = gn_lcm(Cg, k.vec), line = bwd || sz == 4 ? 32 : 64, blocks = gn_lcm(unit, CK_BLOCK);
    int W = (blocks <= 2 * line || blocks <= 2 * unit) ? blocks : unit;
    W *= cdiv(line, W);
    if (W > p.C) W = p.C;
    // resident: one workgroup, R vectors per thread; offsets in a sample below 2^31 bytes.  Small workgroups with few vectors each where
    // that holds the strip (64 x 117 rows of bf16: 128 threads of 8 vectors 11.8 us, 256 of 4 9.2 us), then up to 12 vectors for 256
    // threads (300 rows, backward: 512 threads of 8 33 us, 256 of 10 23 us), 16 for 512, 12 for the forward's 1024.
    g.parts = 1; g.chunks = 1;
    g.TX = cdiv(W, k.vec);
    k.resident = false;
    if (wide && g.TX <= 512 && (long)p.L * p.C * sz < (1L << 31))
        for (int T = 64; T <= (bwd ? 512 : 1024) && !k.resident; T *= 2) {
            if (T < g.TX) continue;
            const int r = cdiv(p.L, T / g.TX);
            const int most = T < 256 ? 4 : T == 512 ? 16 : 12;
            if (r > most) continue;
            k.threads = T;
            k.R = r <= 1 ? 1 : r <= 4 ? 4 : r <= 8 ? 8 : r <= 10 ? 10 : r <= 12 ? 12 : 16;
            k.resident = ((long)(T / g.TX) * k.R + 1) * p.C * sz < (1L << 32);      // offsets of rows behind the last do not wrap
        }
    if (!k.resident) {
        k.threads = GN_T; k.R = 0;
        if (W > GN_T * k.vec) {                  // at most 256 vectors to a row
            if (unit <= GN_T * k.vec) W = unit;
            else { g.parts = cdiv(Cg, GN_T * k.vec); W = GN_T * k.vec; }
        }
        g.TX = cdiv(W, k.vec);
    }
    g.W = W;
    g.NG = g.parts > 1 ? 1 : W / Cg;
    g.strips = g.parts > 1 ? p.G * g.parts : cdiv(p.C, W);
    if (!k.resident) {
        // enough workgroups for the 256 CUs (about four each), never more chunks than 32-row pieces of the sample
        long want = cdiv(1024, (long)p.N * g.strips);
        if (want > cdiv(p.L, 32)) want = cdiv(p.L, 32);
        if (want > GN_CHUNKS) want = GN_CHUNKS;
        g.chunks = (int)want;
    }
    // a block's lanes are neighbours in a row of lanes that starts at a block
    k.fuse = k.vec > 1 && W % CK_BLOCK == 0 && g.parts == 1;
    k.blocks = (unsigned)((long)p.N * g.chunks * g.strips);
    return k;
}
static int gn_check(const GroupNormArgs& p, const char* what) {
    MTTS_REQUIRE(p.N > 0 && p.L > 0 && p.C > 0 && p.G > 0, "%s: empty input (N %d, L %d, C %d, G %d)", what, p.N, p.L, p.C, p.G);
    MTTS_REQUIRE(p.C % p.G == 0, "%s: %d channels are not a multiple of %d groups", what, p.C, p.G);
    MTTS_REQUIRE(p.dtype == MTTS_F32 || p.dtype == MTTS_BF16, "%s: dtype %d is neither MTTS_F32 nor MTTS_BF16", what, p.dtype);
    MTTS_REQUIRE(p.act >= MTTS_ACT_NONE && p.act <= MTTS_ACT_SILU, "%s: unknown activation %d", what, p.act);
    MTTS_REQUIRE(p.gamma && p.beta && p.mean && p.rstd, "%s: missing tensor", what);
    // a grid has fewer than 2^32 threads; strips are 32 channels wide at least, or the whole row
    MTTS_REQUIRE((long)p.N * cdiv(p.C, 32) * (p.G > cdiv(p.C, 32) ? 2 : 1) < (1L << 32) / 1024, "%s: %d samples x %d channels are too many for one call", what, p.N, p.C);
    MTTS_REQUIRE(p.C <= (1 << 24), "%s: %d channels are too many", what, p.C);
    MTTS_REQUIRE(p.L <= 0x7fff0000, "%s: %d rows are too many for one call", what, p.L);      // a row number plus a workgroup's rows fits an int
    return 0;
}

static bool gn_aligned(const GroupNormArgs& p, bool bwd) {
    const int vec = p.dtype == MTTS_F32 ? 4 : 8;
    return aligned_to(p.mask, vec) && aligned_to(p.q, vec) && (bwd ? (p.q || aligned_to(p.x, 16)) && aligned_to(p.dy, 16) && aligned_to(p.dx, 16) : aligned_to(p.x, 16) && aligned_to(p.y, 16));
}

// What the call with these arguments (all but ws filled in) needs.
MTTS_API long mtts_group_norm_workspace_floats(const GroupNormArgs* args, int backward) {
    const GroupNormArgs& p = *args;
    if (gn_check(p, "mtts_group_norm_workspace_floats")) return -1;
    const GnPlan k = gn_plan(p, gn_aligned(p, backward != 0), backward != 0);
    const long sums = backward ? 2L * p.N * k.geo.chunks * p.C : 0;
    return sums + (k.resident ? 0 : 3L * p.N * p.G * k.geo.chunks * k.geo.parts);
}

template <typename F> static int gn_attr(F fn, size_t lds) {
    if (lds > 64 * 1024) MTTS_CHECK_HIP(hipFuncSetAttribute((const void*)fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    return 0;
}
template <typename T, int VEC, int R, bool STR> static int gn_fwd_go(const GroupNormArgs& p, const GnPlan& k, hipStream_t s) {
    const int TY = k.threads / k.geo.TX, LG = STR ? p.C / p.G : p.C / p.G / VEC;
    const size_t lds = sizeof(float) * (2 * (size_t)k.geo.NG * TY * LG + 3 * k.geo.NG);
    MTTS_TRY(gn_attr(gn_fwd_kernel<T, VEC, R, STR>, lds));
    hipLaunchKernelGGL((gn_fwd_kernel<T, VEC, R, STR>), dim3(k.blocks), dim3(k.threads), lds, s, p, k.geo);
    return 0;
}
template <typename T, int VEC, int R, bool STR, bool CK> static int gn_bwd_go(const GroupNormArgs& p, const GnPlan& k, hipStream_t s) {
    const int TY = k.threads / k.geo.TX;
    const size_t lds = sizeof(float) * (2 * (size_t)VEC * TY * k.geo.TX + 2 * k.geo.W + 2 * k.geo.NG);
    MTTS_TRY(gn_attr(gn_bwd_kernel<T, VEC, R, STR, CK>, lds));
    hipLaunchKernelGGL((gn_bwd_kernel<T, VEC, R, STR, CK>), dim3(k.blocks), dim3(k.threads), lds, s, p, k.geo);
    return 0;
}
template <typename T, int VEC, bool STR> static int gn_fwd_pick(const GroupNormArgs& p, const GnPlan& k, hipStream_t s) {
    if constexpr (VEC > 1) {
        if (k.resident) switch (k.R) {
            case 1: return gn_fwd_go<T, VEC, 1, STR>(p, k, s);
            case 4: return gn_fwd_go<T, VEC, 4, STR>(p, k, s);
            case 8: return gn_fwd_go<T, VEC, 8, STR>(p, k, s);
            case 10: return gn_fwd_go<T, VEC, 10, STR>(p, k, s);
            case 12: return gn_fwd_go<T, VEC, 12, STR>(p, k, s);
            default: return gn_fwd_go<T, VEC, 16, STR>(p, k, s);
        }
        if (p.q) hipLaunchKernelGGL((gn_moments_kernel<T, VEC, STR, true>), dim3(k.blocks), dim3(GN_T), 0, s, p, k.geo);
    }
    if (VEC == 1 || !p.q) hipLaunchKernelGGL((gn_moments_kernel<T, VEC, STR, false>), dim3(k.blocks), dim3(GN_T), 0, s, p, k.geo);
    hipLaunchKernelGGL((gn_apply_kernel<T, VEC, STR>), dim3(k.blocks), dim3(GN_T), 0, s, p, k.geo);
    return 0;
}
template <typename T, int VEC, bool STR, bool CK> static int gn_bwd_pick(const GroupNormArgs& p, const GnPlan& k, hipStream_t s) {
    if constexpr (VEC > 1) {
        if (k.resident) switch (k.R) {
            case 1: return gn_bwd_go<T, VEC, 1, STR, CK>(p, k, s);
            case 4: return gn_bwd_go<T, VEC, 4, STR, CK>(p, k, s);
            case 8: return gn_bwd_go<T, VEC, 8, STR, CK>(p, k, s);
            case 10: return gn_bwd_go<T, VEC, 10, STR, CK>(p, k, s);
            case 12: return gn_bwd_go<T, VEC, 12, STR, CK>(p, k, s);
            default: return gn_bwd_go<T, VEC, 16, STR, CK>(p, k, s);
        }
    }
    float* const gs = p.ws + 2L * p.N * k.geo.chunks * p.C;
    hipLaunchKernelGGL((gn_bwd_sums_kernel<T, VEC, STR, CK>), dim3(k.blocks), dim3(GN_T), 0, s, p, k.geo, gs);
    hipLaunchKernelGGL((gn_bwd_apply_kernel<T, VEC, STR, CK>), dim3(k.blocks), dim3(GN_T), 0, s, p, k.geo, (const float*)gs);
    return 0;
}

MTTS_API int mtts_group_norm_act_fwd(const GroupNormArgs* args, void* stream) {
    GroupNormArgs p = *args;
    hipStream_t s = (hipStream_t)stream;
    MTTS_TRY(gn_check(p, "mtts_group_norm_act_fwd"));
    MTTS_REQUIRE(p.x && p.y && !p.q == !p.q_code, "mtts_group_norm_act_fwd: missing tensor");
    const GnPlan k = gn_plan(p, gn_aligned(p, false), false);
    MTTS_REQUIRE(p.ws || k.resident, "mtts_group_norm_act_fwd: missing workspace");
    int8_t* const q = p.q;
    if (!k.fuse) p.q = nullptr;                  // a pass of its own below
    if (p.dtype == MTTS_F32) {
        if (k.vec == 1) MTTS_TRY((gn_fwd_pick<float, 1, false>(p, k, s)));
        else if (k.str) MTTS_TRY((gn_fwd_pick<float, 4, true>(p, k, s)));
        else MTTS_TRY((gn_fwd_pick<float, 4, false>(p, k, s)));
    } else {
        if (k.vec == 1) MTTS_TRY((gn_fwd_pick<bf16_t, 1, false>(p, k, s)));
        else if (k.str) MTTS_TRY((gn_fwd_pick<bf16_t, 8, true>(p, k, s)));
        else MTTS_TRY((gn_fwd_pick<bf16_t, 8, false>(p, k, s)));
    }
    MTTS_CHECK_LAUNCH("group_norm_act_fwd");
    if (q && !p.q) MTTS_TRY(mtts_checkpoint8_pack(p.x, p.lengths, q, p.q_code, p.N, p.L, p.C, p.dtype, stream));
    return 0;
}

template <typename T, int VEC, bool STR> static int gn_bwd_any(const GroupNormArgs& p, const GnPlan& k, hipStream_t s) {
    return p.q ? gn_bwd_pick<T, VEC, STR, true>(p, k, s) : gn_bwd_pick<T, VEC, STR, false>(p, k, s);
}

MTTS_API int mtts_group_norm_act_bwd(const GroupNormArgs* args, void* stream) {
    const GroupNormArgs p = *args;
    hipStream_t s = (hipStream_t)stream;
    MTTS_TRY(gn_check(p, "mtts_group_norm_act_bwd"));
    MTTS_REQUIRE(p.dy && p.dx && (p.q ? p.q_code != nullptr : p.x != nullptr), "mtts_group_norm_act_bwd: missing tensor");
    MTTS_REQUIRE(p.ws, "mtts_group_norm_act_bwd: missing workspace");
    const GnPlan k = gn_plan(p, gn_aligned(p, true), true);
    if (p.dtype == MTTS_F32) {
        if (k.vec == 1) MTTS_TRY((gn_bwd_any<float, 1, false>(p, k, s)));
        else if (k.str) MTTS_TRY((gn_bwd_any<float, 4, true>(p, k, s)));
        else MTTS_TRY((gn_bwd_any<float, 4, false>(p, k, s)));
    } else {
        if (k.vec == 1) MTTS_TRY((gn_bwd_any<bf16_t, 1, false>(p, k, s)));
        else if (k.str) MTTS_TRY((gn_bwd_any<bf16_t, 8, true>(p, k, s)));
        else MTTS_TRY((gn_bwd_any<bf16_t, 8, false>(p, k, s)));
    }
    if (p.dgamma || p.dbeta) MTTS_TRY(gn_param_grad(p, (long)p.N * k.geo.chunks, s));
    MTTS_CHECK_LAUNCH("group_norm_act_bwd");
    return 0;
}
