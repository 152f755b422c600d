// Weight gradient of a 1-D convolution (or of a linear layer: kernel 1) whose input is held as an 8-bit checkpoint:
//
//   dW[o, c, t] = sum over rows r = (n, l) of dy[r, o] * x[r + shift_t, c],   shift_t = t * dilation - (kernel - 1) * dilation / 2,
//                 x = q * 2^(code - 127), zero outside the sequence; o and c of the same group
//
// A matrix product over the rows: M = output channels, N = (tap, input channel), K = rows; both operands lie with K as the slow index.
// x is exact in bf16 (seven significant bits times a power of two), so an fp32 gradient needs three matrix terms: dy = a1 + a2 + a3, each
// the leading eight bits of what is left (an exact split, 24 bits), against six where both operands are fp32.  fp32 accumulation.
// A bf16 gradient, and an fp32 one in bf16 mode (rounded to nearest even), takes one term.
//
// Tile TM x TN x 32 rows per workgroup, v_mfma_f32_32x32x16_bf16.  A thread takes 8 rows x 4 columns: the transposition happens in
// registers, and 8 rows of one column are the 16 bytes that a lane feeds to the matrix instruction.  LDS holds these 16-byte units in
// fragment order, [32-column block][row octet][column], the column XORed with (column / 8) & 3 so that the stores (four columns per
// lane) and the reads (one column per lane) both touch every bank equally.
// The rows are split over grid.z; partial tiles go to a workspace and are added in split order.
#include "vec_io.h"

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;

constexpr int WG_BK = 32;          // rows of a K step

__device__ __forceinline__ int wg_unit(int octet, int col) { return ((col >> 5) * 4 + octet) * 32 + ((col & 31) ^ ((col >> 3) & 3)); }
__device__ __forceinline__ unsigned top_halves(float lo, float hi) {      // the leading 16 bits of two fp32, as two bf16
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302);
}
__device__ __forceinline__ float bf16_head(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }

// TERMS 3: exact split of fp32; 1: bf16 gradient, or fp32 rounded.  VEC: quads of columns are loaded at once (else element by element).
template <typename T, int TERMS, int TM, int TN, int WM, int WN, bool VEC>
__global__ void __launch_bounds__((TM / WM) * (TN / WN) * 64) wgrad8_kernel(Wgrad8Args p, int splits, int tiles_n, int steps_per) {
    constexpr int THREADS = (TM / WM) * (TN / WN) * 64, FM = WM / 32, FN = WN / 32;
    static_assert(TM + TN <= THREADS, "one 8 x 4 piece of an operand tile per thread");
    __shared__ u32x4 sa[TERMS][TM * 4];
    __shared__ u32x4 sb[TN * 4];
    const int Og = p.O / p.groups, Cg = p.I / p.groups, Nn = p.kernel * Cg, nb = (p.I + CK_BLOCK - 1) / CK_BLOCK;
    const int split = blockIdx.z % splits, g = blockIdx.z / splits;
    const int tm = blockIdx.x / tiles_n, tn = blockIdx.x - tm * tiles_n;
    const int m0 = tm * TM, n0 = tn * TN;
    const long R = (long)p.N * p.L;
    const long k_begin = (long)split * steps_per * WG_BK, k_end = min(R, k_begin + (long)steps_per * WG_BK);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = (wave / (TN / WN)) * WM, wn = (wave % (TN / WN)) * WN;

    // this thread's piece: threads [0, TM) stage dy, [TM, TM + TN) stage x; 4 columns, row octet `oct` of the step
    const bool is_a = tid < TM, is_b = !is_a && tid < TM + TN;
    const int piece = is_a ? tid : tid - TM, quads = (is_a ? TM : TN) / 4;
    const int oct = piece / quads, col = (piece - oct * quads) * 4;
    int bt[4], bc[4]; bool bon[4];               // x columns: tap, channel
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int jn = n0 + col + j;
        bon[j] = is_b && jn < Nn;
        bt[j] = bon[j] ? jn / Cg : 0; bc[j] = bon[j] ? jn - bt[j] * Cg + g * Cg : 0;
    }
    const int pad = (p.kernel - 1) * p.dilation / 2;

    f32x16 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    for (long k0 = k_begin; k0 < k_end; k0 += WG_BK) {
        float f[8][4];
        const long r0 = k0 + oct * 8;
        if (is_a) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const long r = r0 + i;
                const T* row = (const T*)p.dy + r * p.O + g * Og + m0 + col;
                if (VEC && r < k_end && m0 + col < Og) {
                    if (sizeof(T) == 4) {
                        const f32x4 v = *reinterpret_cast<const f32x4*>(row);
#pragma unroll
                        for (int j = 0; j < 4; ++j) f[i][j] = v[j];
                    } else {
                        const u32x2 v = *reinterpret_cast<const u32x2*>(row);
                        f[i][0] = bf16_lo(v[0]); f[i][1] = bf16_hi(v[0]); f[i][2] = bf16_lo(v[1]); f[i][3] = bf16_hi(v[1]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        f[i][j] = 0.f;
                        if (!VEC && r < k_end && m0 + col + j < Og) { Raw<T, 1> v; v.load(row + j); v.get(&f[i][j]); }
                    }
                }
            }
        } else if (is_b) {
            int l = (int)(r0 % p.L);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const long r = r0 + i;
#pragma unroll
                for (int j = 0; j < 4; ++j) f[i][j] = 0.f;
                if (r < k_end) {
                    if (VEC) {
                        const int ls = l + bt[0] * p.dilation - pad;
                        if (bon[0] && ls >= 0 && ls < p.L) {
                            const long row = r + bt[0] * p.dilation - pad;
                            const float s = ck_scale(p.q_code[row * nb + bc[0] / CK_BLOCK]);
                            Bytes<4> q; q.load(p.q + row * p.I + bc[0]);
#pragma unroll
                            for (int j = 0; j < 4; ++j) f[i][j] = ck_value(q.get(j), s);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int ls = l + bt[j] * p.dilation - pad;
                            if (bon[j] && ls >= 0 && ls < p.L) {
                                const long row = r + bt[j] * p.dilation - pad;
                                f[i][j] = ck_value((uint8_t)p.q[row * p.I + bc[j]], ck_scale(p.q_code[row * nb + bc[j] / CK_BLOCK]));
                            }
                        }
                    }
                }
                l = l + 1 == p.L ? 0 : l + 1;
            }
        }
        __syncthreads();                     // the previous step's fragments have been read
        if (is_a) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = wg_unit(oct, col + j);
                if (TERMS == 1) {
                    sa[0][at] = u32x4{bf16_pack(f[0][j], f[1][j]), bf16_pack(f[2][j], f[3][j]), bf16_pack(f[4][j], f[5][j]), bf16_pack(f[6][j], f[7][j])};
                } else {
#pragma unroll
                    for (int t = 0; t < TERMS; ++t) {
                        u32x4 w;
#pragma unroll
                        for (int h = 0; h < 4; ++h) w[h] = top_halves(f[2 * h][j], f[2 * h + 1][j]);
                        sa[t][at] = w;
#pragma unroll
                        for (int i = 0; i < 8; ++i) f[i][j] -= bf16_head(f[i][j]);
                    }
                }
            }
        } else if (is_b) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                sb[wg_unit(oct, col + j)] = u32x4{top_halves(f[0][j], f[1][j]), top_halves(f[2][j], f[3][j]), top_halves(f[4][j], f[5][j]), top_halves(f[6][j], f[7][j])};
        }
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            bf16x8_t b[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) b[j] = __builtin_bit_cast(bf16x8_t, sb[wg_unit(ks * 2 + (lane >> 5), wn + j * 32 + (lane & 31))]);
#pragma unroll
            for (int t = TERMS - 1; t >= 0; --t)          // small terms first
#pragma unroll
                for (int i = 0; i < FM; ++i) {
                    const bf16x8_t a = __builtin_bit_cast(bf16x8_t, sa[t][wg_unit(ks * 2 + (lane >> 5), wm + i * 32 + (lane & 31))]);
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b[j], acc[i][j], 0, 0, 0);
                }
        }
    }

    // element e of a 32 x 32 tile: row 8 * (e / 4) + 4 * (lane / 32) + e % 4, column lane % 32
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int m = m0 + wm + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3), n = n0 + wn + j * 32 + (lane & 31);
                if (m < Og && n < Nn) {
                    const long o = (long)g * Og + m;
                    if (splits > 1) p.ws[((long)split * p.O + o) * Nn + n] = acc[i][j][e];
                    else if (p.packed) p.dw[o * Nn + n] = acc[i][j][e];
                    else { const int t = n / Cg; p.dw[(o * Cg + n - t * Cg) * p.kernel + t] = acc[i][j][e]; }
                }
            }
}

// dw = sum over the splits, in split order; [O, kernel, Cg] -> the same (packed) or [O, Cg, kernel]
__global__ void __launch_bounds__(256) wgrad8_sum_kernel(Wgrad8Args p, int splits) {
    const int Cg = p.I / p.groups, Nn = p.kernel * Cg;
    const long total = (long)p.O * Nn, stride = (long)gridDim.x * 256;
    GridRC rc((long)blockIdx.x * 256 + threadIdx.x, stride, Nn);
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += stride, rc.next()) {
        float s = 0.f;
        for (int k0 = 0; k0 < splits; k0 += 8) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = p.ws[(long)min(k0 + k, splits - 1) * total + i];
#pragma unroll
            for (int k = 0; k < 8; ++k) if (k0 + k < splits) s += v[k];
        }
        if (p.packed) p.dw[i] = s;
        else { const int t = rc.col / Cg; p.dw[(rc.row * Cg + rc.col - t * Cg) * p.kernel + t] = s; }
    }
}

struct WgPlan { int tiles_m, tiles_n, splits, steps_per; };
static WgPlan wg_plan(const Wgrad8Args& p, int TM, int TN) {
    WgPlan k;
    const long R = (long)p.N * p.L;
    const int steps = cdiv(R, WG_BK);
    k.tiles_m = cdiv(p.O / p.groups, TM); k.tiles_n = cdiv((long)p.kernel * (p.I / p.groups), TN);
    // enough workgroups for two to a CU, at least eight steps each
    const long tiles = (long)k.tiles_m * k.tiles_n * p.groups;
    long want = cdiv(512, tiles);
    if (want > steps / 8) want = steps / 8;
    if (want < 1) want = 1;
    k.steps_per = cdiv(steps, want);
    k.splits = cdiv(steps, k.steps_per);
    return k;
}

static int wg_check(const Wgrad8Args& p) {
    MTTS_REQUIRE(p.N > 0 && p.L > 0 && p.I > 0 && p.O > 0 && p.kernel > 0 && p.dilation > 0 && p.groups > 0,
                 "mtts_conv_weight_grad8: empty shape (N %d, L %d, I %d, O %d, kernel %d, dilation %d, groups %d)", p.N, p.L, p.I, p.O, p.kernel, p.dilation, p.groups);
    MTTS_REQUIRE(p.I % p.groups == 0 && p.O % p.groups == 0, "mtts_conv_weight_grad8: %d x %d channels are not a multiple of %d groups", p.I, p.O, p.groups);
    MTTS_REQUIRE(p.dtype == MTTS_F32 || p.dtype == MTTS_BF16, "mtts_conv_weight_grad8: dtype %d is neither MTTS_F32 nor MTTS_BF16", p.dtype);
    MTTS_REQUIRE((long)p.kernel * (p.I / p.groups) < (1L << 28) && (long)(p.kernel - 1) * p.dilation < (1L << 30), "mtts_conv_weight_grad8: kernel %d with dilation %d is too large", p.kernel, p.dilation);
    const WgPlan k = wg_plan(p, 128, 128);
    MTTS_REQUIRE((long)k.tiles_m * k.tiles_n * 256 < (1L << 32) && (long)k.splits * p.groups < 65536, "mtts_conv_weight_grad8: too many tiles for one call");
    return 0;
}

MTTS_API long mtts_conv_weight_grad8_workspace_floats(const Wgrad8Args* args) {
    if (wg_check(*args)) return -1;
    const WgPlan k = wg_plan(*args, 128, 128);
    return k.splits > 1 ? (long)k.splits * args->O * args->kernel * (args->I / args->groups) : 0;
}

template <typename T, int TERMS, bool VEC> static void wg_go(const Wgrad8Args& p, hipStream_t s) {
    const WgPlan k = wg_plan(p, 128, 128);
    hipLaunchKernelGGL((wgrad8_kernel<T, TERMS, 128, 128, 64, 64, VEC>), dim3(k.tiles_m * k.tiles_n, 1, k.splits * p.groups), dim3(256), 0, s, p, k.splits, k.tiles_n, k.steps_per);
    if (k.splits > 1) {
        const long total = (long)p.O * p.kernel * (p.I / p.groups);
        const long blocks = cdiv(total, 256);
        hipLaunchKernelGGL(wgrad8_sum_kernel, dim3((unsigned)(blocks > 4096 ? 4096 : blocks)), dim3(256), 0, s, p, k.splits);
    }
}

MTTS_API int mtts_conv_weight_grad8(const Wgrad8Args* args, void* stream) {
    const Wgrad8Args p = *args;
    hipStream_t s = (hipStream_t)stream;
    MTTS_TRY(wg_check(p));
    MTTS_REQUIRE(p.q && p.q_code && p.dy && p.dw && (p.ws || mtts_conv_weight_grad8_workspace_floats(&p) == 0), "mtts_conv_weight_grad8: missing tensor");
    const bool f32 = p.dtype == MTTS_F32;
    const int Og = p.O / p.groups, Cg = p.I / p.groups;
    // whole quads of columns inside a group and a tap, at addresses that a quad may start at
    const bool v = Og % 4 == 0 && Cg % 4 == 0 && aligned_to(p.dy, f32 ? 16 : 8) && aligned_to(p.q, 4);
    const int prec = p.precision ? p.precision : (mtts_get_precision() == 1 ? 1 : 2);      // as GemmArgs.precision
    if (!f32) v ? wg_go<bf16_t, 1, true>(p, s) : wg_go<bf16_t, 1, false>(p, s);
    else if (prec == 1) v ? wg_go<float, 1, true>(p, s) : wg_go<float, 1, false>(p, s);
    else v ? wg_go<float, 3, true>(p, s) : wg_go<float, 3, false>(p, s);
    MTTS_CHECK_LAUNCH("conv_weight_grad8");
    return 0;
}
