// 8-bit activation checkpoints: pack x[N, L, C] (fp32 or bf16) into q[N, L, C] (signed bytes) + code[N, L, ceil(C / 32)] (biased
// exponents), and the values they stand for.  The arithmetic is in vec_io.h.
//
// One pass over memory each way, nothing else: 4 (2) bytes read, 1 + 1/32 written per value.  A block's 32 channels sit in 8 (fp32) or 4
// (bf16) neighbouring lanes, so its maximum is three (two) DPP steps; a row's last, partial block is padded with idle lanes.  Vectors
// start at any element and a row's last one may be partial (64 x 600 x 511 fp32, pack: 30 us element by element, 19 us so).
//
// 64 x 600 x 512: fp32 (99 MB each way) pack 18.8 us, unpack 17.2 us, 5.3 and 5.8 TB/s, with inputs that partly come from the last-level
// cache; pack with lengths from 300 to 600 (79 MB) 17 us.  bf16 (60 MB): pack 15.3 us, 3.9 TB/s (the vector instructions of the rounding),
// unpack 10.9 us, 5.5 TB/s.  A copy of 1 GiB runs at 5.1 TB/s on the same card.
#include "vec_io.h"

constexpr int CK_T = 256;
constexpr int CK_U = 8;          // rows a thread requests before it uses the first

// Workgroup -> (sample, row chunk, strip of TX lane slots); a thread takes one slot of CK_U rows, TY apart.  One 32-bit division per
// thread: flat indices over the whole tensor cost two 64-bit divisions, more than the work on four vectors.
struct CkGeo { int TX, strips, chunks; unsigned blocks; };
struct CkAt { int n, row, TY, slot; bool on; };
__device__ __forceinline__ CkAt ck_at(const CkGeo& k) {
    unsigned b = blockIdx.x;
    const int strip = b % k.strips; b /= k.strips;
    const int chunk = b % k.chunks, n = b / k.chunks, TY = CK_T / k.TX, ty = threadIdx.x / k.TX;
    return CkAt{n, chunk * TY * CK_U + ty, TY, strip * k.TX + (int)threadIdx.x - ty * k.TX, ty < TY};      // lanes behind the last whole row of lanes: off
}

// P lane slots to a row, a whole number of blocks
template <typename T, int VEC>
__global__ void __launch_bounds__(CK_T) ck_pack_kernel(const T* __restrict__ x, const int* __restrict__ lengths, int8_t* __restrict__ q,
                                                       uint8_t* __restrict__ code, int L, int C, int P, CkGeo k) {
    constexpr int LANES = CK_BLOCK / VEC;
    const CkAt t = ck_at(k);
    const int len = lengths ? min(max(lengths[t.n], 0), L) : L, c = t.slot * VEC, nb = P / LANES, left = C - c;      // values of this slot (none: <= 0)
    const long row0 = (long)t.n * L;
    Raw<T, VEC> v[CK_U];
#pragma unroll
    for (int u = 0; u < CK_U; ++u) {
        const int r = t.row + u * t.TY;
        v[u].zero();
        if (t.on && r < len && left > 0) load_any(v[u], x + (row0 + r) * C + c, left);
    }
#pragma unroll
    for (int u = 0; u < CK_U; ++u) {
        const int r = t.row + u * t.TY;
        unsigned m = 0;
#pragma unroll
        for (int j = 0; j < VEC; ++j) m = umax_(m, abs_bits(v[u].at(j)));
        m = block_max<LANES>(m);
        const unsigned e = ck_code(m);
        if (t.on && r < L && t.slot < P) {
            const long at = row0 + r;
            if (left > 0) ck_store(q + at * C + c, v[u], e, left);
            if ((c & (CK_BLOCK - 1)) == 0) code[at * nb + c / CK_BLOCK] = (uint8_t)e;
        }
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(CK_T) ck_unpack_kernel(const int8_t* __restrict__ q, const uint8_t* __restrict__ code, T* __restrict__ x,
                                                         long rows, int C, CkGeo k) {
    const CkAt t = ck_at(k);                     // n: chunks of 2^20 rows, so that rows of one fit an int
    const long row0 = (long)t.n << 20;
    const int c = t.slot * VEC, nb = (C + CK_BLOCK - 1) / CK_BLOCK, L = (int)min(rows - row0, 1L << 20), left = C - c;
    Bytes<VEC> v[CK_U]; unsigned e[CK_U];
#pragma unroll
    for (int u = 0; u < CK_U; ++u) {
        const int r = t.row + u * t.TY;
        if (t.on && r < L && left > 0) { load_any(v[u], q + (row0 + r) * C + c, left); e[u] = code[(row0 + r) * nb + c / CK_BLOCK]; }
    }
#pragma unroll
    for (int u = 0; u < CK_U; ++u) {
        const int r = t.row + u * t.TY;
        if (t.on && r < L && left > 0) {
            float f[VEC]; const float s = ck_scale(e[u]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = ck_value(v[u].get(j), s);
            stream_any(x + (row0 + r) * C + c, f, left);
        }
    }
}

// N samples of L rows of P slots; false where a grid would have 2^32 threads or more
static bool ck_geo(CkGeo& k, long N, long L, long P) {
    k.TX = (int)(P < CK_T ? P : CK_T);
    k.strips = cdiv(P, k.TX);
    const long chunks = (L + (long)CK_T / k.TX * CK_U - 1) / ((long)CK_T / k.TX * CK_U);
    k.chunks = (int)chunks;
    const long blocks = N * chunks;
    k.blocks = (unsigned)(blocks * k.strips);
    return blocks < (1L << 32) / CK_T && blocks * k.strips < (1L << 32) / CK_T;
}

template <typename T, int VEC>
static int ck_pack_go(const void* x, const int* lengths, int8_t* q, uint8_t* code, int N, int L, int C, hipStream_t s) {
    const int P = cdiv(C, CK_BLOCK) * (CK_BLOCK / VEC);
    CkGeo k;
    MTTS_REQUIRE(ck_geo(k, N, L, P), "mtts_checkpoint8_pack: %d x %d x %d values are too many for one call", N, L, C);
    hipLaunchKernelGGL((ck_pack_kernel<T, VEC>), dim3(k.blocks), dim3(CK_T), 0, s, (const T*)x, lengths, q, code, L, C, P, k);
    return 0;
}

template <typename T, int VEC>
static int ck_unpack_go(const int8_t* q, const uint8_t* code, void* x, long rows, int C, hipStream_t s) {
    CkGeo k;
    const long piece = 1L << 20;
    MTTS_REQUIRE(ck_geo(k, (rows + piece - 1) / piece, rows < piece ? rows : piece, cdiv(C, VEC)), "mtts_checkpoint8_unpack: %ld x %d values are too many for one call", rows, C);
    hipLaunchKernelGGL((ck_unpack_kernel<T, VEC>), dim3(k.blocks), dim3(CK_T), 0, s, q, code, (T*)x, rows, C, k);
    return 0;
}

MTTS_API int mtts_checkpoint8_pack(const void* x, const int* lengths, int8_t* q, uint8_t* code, int N, int L, int C, int dtype, void* stream) {
    MTTS_REQUIRE(x && q && code, "mtts_checkpoint8_pack: missing tensor");
    MTTS_REQUIRE(N > 0 && L > 0 && C > 0 && (dtype == MTTS_F32 || dtype == MTTS_BF16), "mtts_checkpoint8_pack: bad shape or type (N %d, L %d, C %d, dtype %d)", N, L, C, dtype);
    MTTS_REQUIRE(L <= 0x7fff0000 && C <= 0x7fff0000, "mtts_checkpoint8_pack: %d x %d x %d values are too many for one call", N, L, C);      // rows of a chunk fit an int
    hipStream_t s = (hipStream_t)stream;
    if (dtype == MTTS_F32) MTTS_TRY((ck_pack_go<float, 4>(x, lengths, q, code, N, L, C, s)));
    else MTTS_TRY((ck_pack_go<bf16_t, 8>(x, lengths, q, code, N, L, C, s)));
    MTTS_CHECK_LAUNCH("checkpoint8_pack");
    return 0;
}

MTTS_API int mtts_checkpoint8_unpack(const int8_t* q, const uint8_t* code, void* x, long rows, int C, int dtype, void* stream) {
    MTTS_REQUIRE(x && q && code, "mtts_checkpoint8_unpack: missing tensor");
    MTTS_REQUIRE(rows > 0 && C > 0 && (dtype == MTTS_F32 || dtype == MTTS_BF16), "mtts_checkpoint8_unpack: bad shape or type (rows %ld, C %d, dtype %d)", rows, C, dtype);
    MTTS_REQUIRE(rows < 1L << 50 && C <= 0x7fff0000, "mtts_checkpoint8_unpack: %ld x %d values are too many for one call", rows, C);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == MTTS_F32) MTTS_TRY((ck_unpack_go<float, 4>(q, code, x, rows, C, s)));
    else MTTS_TRY((ck_unpack_go<bf16_t, 8>(q, code, x, rows, C, s)));
    MTTS_CHECK_LAUNCH("checkpoint8_unpack");
    return 0;
}
