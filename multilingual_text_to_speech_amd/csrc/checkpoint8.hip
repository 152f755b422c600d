// 8-bit activation checkpoints: pack x[N, L, C] (fp32 or bf16) into q[N, L, C] (signed bytes) + code[N, L, ceil(C / 32)] (biased
// exponents), and the values they stand for.  The arithmetic is in vec_io.h.
//
// One pass over memory each way, nothing else: 4 (2) bytes read, 1 + 1/32 written per value.  A block's 32 channels sit in 8 (fp32) or 4
// (bf16) neighbouring lanes, so its maximum is three (two) DPP steps; a row's last, partial block is padded with idle lanes.
#include "vec_io.h"

constexpr int CK_T = 256;
constexpr int CK_U = 4;          // vectors a thread requests before it uses the first

// n-th sample, its rows x P lane slots (P = slots of a row, a whole number of blocks); grid N * chunks
template <typename T, int VEC>
__global__ void __launch_bounds__(CK_T) ck_pack_kernel(const T* __restrict__ x, const int* __restrict__ lengths, int8_t* __restrict__ q,
                                                       uint8_t* __restrict__ code, int L, int C, int P, int chunks) {
    constexpr int LANES = CK_BLOCK / VEC;
    const int n = blockIdx.x / chunks, chunk = blockIdx.x - n * chunks;
    const int len = lengths ? min(max(lengths[n], 0), L) : L;
    const long row0 = (long)n * L, total = (long)L * P;
    const int nb = P / LANES;
    const long i0 = (long)chunk * CK_T + threadIdx.x, stride = (long)chunks * CK_T;
    GridRC rc(i0, stride, P);
    for (long i = i0; i - (long)threadIdx.x < total; ) {              // whole workgroups: the lanes of a block stay together
        Raw<T, VEC> v[CK_U];
        long row[CK_U]; int col[CK_U]; bool in[CK_U];
#pragma unroll
        for (int u = 0; u < CK_U; ++u) {
            row[u] = rc.row; col[u] = rc.col * VEC; in[u] = i < total;
            v[u].zero();
            if (in[u] && rc.row < len && col[u] < C) v[u].load(x + (row0 + rc.row) * C + col[u]);
            rc.next(); i += stride;
        }
#pragma unroll
        for (int u = 0; u < CK_U; ++u) {
            unsigned m = 0;
#pragma unroll
            for (int j = 0; j < VEC; ++j) m = umax_(m, abs_bits(v[u].at(j)));
            if (VEC == 1) {
#pragma unroll
                for (int d = 1; d < CK_BLOCK; d *= 2) m = umax_(m, (unsigned)__shfl_xor((int)m, d, 64));
            } else {
                m = block_max<LANES == 4 ? 4 : 8>(m);
            }
            const unsigned c = ck_code(m);
            if (in[u]) {
                const long at = row0 + row[u];
                if (col[u] < C) {
                    if constexpr (VEC == 1) q[at * C + col[u]] = (int8_t)ck_quantise(v[u].at(0), c);
                    else ck_store(q + at * C + col[u], v[u], c);
                }
                if ((col[u] & (CK_BLOCK - 1)) == 0) code[at * nb + col[u] / CK_BLOCK] = (uint8_t)c;
            }
        }
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(CK_T) ck_unpack_kernel(const int8_t* __restrict__ q, const uint8_t* __restrict__ code, T* __restrict__ x,
                                                         long rows, int C) {
    const int P = C / VEC, nb = (C + CK_BLOCK - 1) / CK_BLOCK;
    const long total = rows * P, i0 = (long)blockIdx.x * CK_T + threadIdx.x, stride = (long)gridDim.x * CK_T;
    GridRC rc(i0, stride, P);
    for (long i = i0; i < total; ) {
        Bytes<VEC> v[CK_U]; unsigned c[CK_U]; long at[CK_U];
#pragma unroll
        for (int u = 0; u < CK_U; ++u) {
            at[u] = -1;
            if (i < total) {
                at[u] = rc.row * C + rc.col * VEC;
                v[u].load(q + at[u]);
                c[u] = code[rc.row * nb + rc.col * VEC / CK_BLOCK];
            }
            rc.next(); i += stride;
        }
#pragma unroll
        for (int u = 0; u < CK_U; ++u)
            if (at[u] >= 0) {
                float f[VEC]; const float s = ck_scale(c[u]);
#pragma unroll
                for (int j = 0; j < VEC; ++j) f[j] = ck_value(v[u].get(j), s);
                store_vec(x + at[u], f);
            }
    }
}

template <typename T, int VEC>
static void ck_pack_go(const void* x, const int* lengths, int8_t* q, uint8_t* code, int N, int L, int C, hipStream_t s) {
    const int P = cdiv(C, CK_BLOCK) * (CK_BLOCK / VEC);
    const long per = cdiv((long)L * P, (long)CK_T * CK_U);              // chunks that give every thread one round
    const int chunks = (int)(per < 1 ? 1 : per);
    hipLaunchKernelGGL((ck_pack_kernel<T, VEC>), dim3((unsigned)((long)N * chunks)), dim3(CK_T), 0, s, (const T*)x, lengths, q, code, L, C, P, chunks);
}

template <typename T, int VEC>
static void ck_unpack_go(const int8_t* q, const uint8_t* code, void* x, long rows, int C, hipStream_t s) {
    const long want = cdiv(rows * (C / VEC), (long)CK_T * CK_U);
    const int blocks = (int)(want < 1 ? 1 : want);
    hipLaunchKernelGGL((ck_unpack_kernel<T, VEC>), dim3(blocks), dim3(CK_T), 0, s, q, code, (T*)x, rows, C);
}

// a grid has fewer than 2^32 threads, one for CK_U lane slots (a slot holds one value at least)
static bool ck_fits(long N, long rows, long C) { return rows * ((C + CK_BLOCK - 1) / CK_BLOCK * CK_BLOCK) / (CK_T * CK_U) + N < (1L << 32) / CK_T; }

MTTS_API int mtts_checkpoint8_pack(const void* x, const int* lengths, int8_t* q, uint8_t* code, int N, int L, int C, int dtype, void* stream) {
    MTTS_REQUIRE(x && q && code, "mtts_checkpoint8_pack: missing tensor");
    MTTS_REQUIRE(N > 0 && L > 0 && C > 0 && (dtype == MTTS_F32 || dtype == MTTS_BF16), "mtts_checkpoint8_pack: bad shape or type (N %d, L %d, C %d, dtype %d)", N, L, C, dtype);
    MTTS_REQUIRE(ck_fits(N, (long)N * L, C), "mtts_checkpoint8_pack: %d x %d x %d values are too many for one call", N, L, C);
    hipStream_t s = (hipStream_t)stream;
    const bool f32 = dtype == MTTS_F32;
    const int vec = f32 ? 4 : 8;
    const bool v = C % vec == 0 && aligned_to(x, 16) && aligned_to(q, vec);       // rows start where a vector may: C is a whole number of them
    if (f32) v ? ck_pack_go<float, 4>(x, lengths, q, code, N, L, C, s) : ck_pack_go<float, 1>(x, lengths, q, code, N, L, C, s);
    else v ? ck_pack_go<bf16_t, 8>(x, lengths, q, code, N, L, C, s) : ck_pack_go<bf16_t, 1>(x, lengths, q, code, N, L, C, s);
    MTTS_CHECK_LAUNCH("checkpoint8_pack");
    return 0;
}

MTTS_API int mtts_checkpoint8_unpack(const int8_t* q, const uint8_t* code, void* x, long rows, int C, int dtype, void* stream) {
    MTTS_REQUIRE(x && q && code, "mtts_checkpoint8_unpack: missing tensor");
    MTTS_REQUIRE(rows > 0 && C > 0 && (dtype == MTTS_F32 || dtype == MTTS_BF16), "mtts_checkpoint8_unpack: bad shape or type (rows %ld, C %d, dtype %d)", rows, C, dtype);
    MTTS_REQUIRE(ck_fits(1, rows, C), "mtts_checkpoint8_unpack: %ld x %d values are too many for one call", rows, C);
    hipStream_t s = (hipStream_t)stream;
    const bool f32 = dtype == MTTS_F32;
    const int vec = f32 ? 4 : 8;
    const bool v = C % vec == 0 && aligned_to(x, 16) && aligned_to(q, vec);
    if (f32) v ? ck_unpack_go<float, 4>(q, code, x, rows, C, s) : ck_unpack_go<float, 1>(q, code, x, rows, C, s);
    else v ? ck_unpack_go<bf16_t, 8>(q, code, x, rows, C, s) : ck_unpack_go<bf16_t, 1>(q, code, x, rows, C, s);
    MTTS_CHECK_LAUNCH("checkpoint8_unpack");
    return 0;
}
