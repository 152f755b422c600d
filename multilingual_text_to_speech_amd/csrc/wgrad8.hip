// Weight gradient of a 1-D convolution (or of a linear layer: kernel 1) whose input is held as an 8-bit checkpoint:
//
//   dW[o, c, t] = sum over rows r = (n, l) of dy[r, o] * x[r + shift_t, c],   shift_t = t * dilation - (kernel - 1) * dilation / 2,
//                 x = q * 2^(code - 127), zero outside the sequence; o and c of the same group
//
// A matrix product over the rows: M = output channels, N = (tap, input channel), K = rows; both operands lie with K as the slow index.
// x is exact in bf16 (seven significant bits times a power of two), so an fp32 gradient needs three matrix terms: dy = a1 + a2 + a3, each
// the leading eight bits of what is left (an exact split, 24 bits), against six where both operands are fp32.  fp32 accumulation.
// A bf16 gradient, and an fp32 one in bf16 mode (rounded to nearest even), takes one term.
// The split's limits: bits of dy worth less than 2^-133, the smallest bf16 number, are lost (magnitudes of 2^-110 and more keep all 24
// bits), and an infinite dy makes its output channel's sums NaN (infinity minus its leading bits), where one term sums infinities.
//
// What bounds it: the matrix pipes.  At 38400 rows, 512 -> 512 channels, kernel 5 (100.7 GFLOP, three terms) the whole call takes 235 us
// where three of four inputs are zeros, as behind a rectifier and dropout, and 250 us where none are: 1210-1290 TFLOP/s of bf16 products
// where a plain bf16 library product of 8192^3 reaches 1330 on the same card.  One term: bf16 gradients 116-120 us, 840-870 TFLOP/s, fp32
// ones in bf16 mode 127-129 us: a step's 1024 cycles of matrix instructions stand beside 1024 cycles of LDS reads and writes (at 128 bytes a
// cycle) and 900 of vector instructions, two thirds of them for the checkpoint.  At 7680 rows, bf16 (20 GFLOP) 44 us: half of that is
// the partial tiles' way through memory (63 MB out and in at twelve splits).  Kernel 1 at 38400 rows, fp32: 67-70 us for 45 us of matrix
// instructions, the same way for sixty-four splits of 1 MB.
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

// One thread's 8 rows x 4 columns, at(row, column), -> four (per plane) 16-byte units.  ROUND: fp32 to the nearest bf16; otherwise TERMS
// planes of eight bits each (3: all of an fp32; 1: all of a bf16).
template <int TERMS, bool ROUND, int PLANE, typename F> __device__ __forceinline__ void wg_put(u32x4* to, int oct, int col, F at) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = at(i, j);
        const int unit = wg_unit(oct, col + j);
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
            if constexpr (ROUND) to[unit] = u32x4{bf16_pack(c[0], c[1]), bf16_pack(c[2], c[3]), bf16_pack(c[4], c[5]), bf16_pack(c[6], c[7])};
            else to[t * PLANE + unit] = u32x4{top_halves(c[0], c[1]), top_halves(c[2], c[3]), top_halves(c[4], c[5]), top_halves(c[6], c[7])};
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] -= bf16_head(c[i]);
        }
    }
}

// the matrix instructions of one half (16 rows) of a K step
template <int TERMS, int PLANE, int FM, int FN>
__device__ __forceinline__ void wg_mfma(const u32x4* sa, const u32x4* sb, int ks, int wm, int wn, int lane, f32x16 (&acc)[FM][FN]) {
    bf16x8_t b[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) b[j] = __builtin_bit_cast(bf16x8_t, sb[wg_unit(ks * 2 + (lane >> 5), wn + j * 32 + (lane & 31))]);
#pragma unroll
    for (int t = TERMS - 1; t >= 0; --t)          // small terms first
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const bf16x8_t a = __builtin_bit_cast(bf16x8_t, sa[t * PLANE + wg_unit(ks * 2 + (lane >> 5), wm + i * 32 + (lane & 31))]);
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b[j], acc[i][j], 0, 0, 0);
        }
}

// Columns of the product: per tap, the quads of channels (at whole multiples of four, so that a quad lies in one checkpoint block) that
// touch the group: Cp = quad columns, the first one at channel `first`; the channels of other groups in the outer quads are not stored.
struct WgCols { int Cp, first, skip; };
__host__ __device__ inline int wg_quad_columns(int Cg) { return Cg % 4 == 0 ? Cg : ((Cg + 6) & ~3); }
__device__ __forceinline__ WgCols wg_cols(const Wgrad8Args& p, int g) {
    const int Cg = p.I / p.groups;
    return WgCols{wg_quad_columns(Cg), g * Cg & ~3, g * Cg & 3};
}

// element e of a 32 x 32 tile: row 8 * (e / 4) + 4 * (lane / 32) + e % 4, column lane % 32
template <int FM, int FN>
__device__ __forceinline__ void wg_store(const Wgrad8Args& p, int splits, int split, int g, int m0, int n0, int lane, const f32x16 (&acc)[FM][FN]) {
    const int Og = p.O / p.groups, Cg = p.I / p.groups, Nn = p.kernel * Cg;
    const WgCols cols = wg_cols(p, g);
    const bool plain = splits > 1 || p.packed;                       // [O, kernel, Cg] slabs / result, or [O, Cg, kernel]
    float* const out = splits > 1 ? p.ws + (long)split * p.O * Nn : p.dw;
    const int mine = m0 + 4 * (lane >> 5), left = Og - mine;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const int n = n0 + j * 32 + (lane & 31), t = n / cols.Cp, c = n - t * cols.Cp - cols.skip;
        if (t >= p.kernel || c < 0 || c >= Cg) continue;
        float* at = out + ((long)g * Og + mine) * Nn + (plain ? t * Cg + c : c * p.kernel + t);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i * 32 + e4 * 8 + e < left) at[(long)e * Nn] = acc[i][j][e4 * 4 + e];
                at += 8L * Nn;
            }
    }
}
template <int FM, int FN> __device__ __forceinline__ void wg_clear(f32x16 (&acc)[FM][FN]) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
}

// Workgroup -> (split, group, tile).  Workgroups go to the eight XCDs in turn; the ones of an XCD get a contiguous run of work, so that
// the tiles of one split (which read the same rows) share an L2.
struct WgAt { int split, g, tm, tn; };
__device__ __forceinline__ WgAt wg_at(int tiles_m, int tiles_n, int groups, int total) {
    const int per = total >> 3, rem = total & 7, x = blockIdx.x & 7, k = blockIdx.x >> 3;
    int id = x * per + min(x, rem) + k;
    WgAt a;
    a.tn = id % tiles_n; id /= tiles_n;
    a.tm = id % tiles_m; id /= tiles_m;
    a.g = id % groups; a.split = id / groups;
    return a;
}

// Any size (dilations whose offsets pass 2^31): element loads, no overlap of loads and products.  128 x 128 x 32, four waves.
template <typename T, int TERMS>
__global__ void __launch_bounds__(256) wgrad8_edge_kernel(Wgrad8Args p, int splits, int tiles_m, int tiles_n, int steps_per) {
    __shared__ u32x4 sa[TERMS * 512];
    __shared__ u32x4 sb[512];
    const int Og = p.O / p.groups, nb = (p.I + CK_BLOCK - 1) / CK_BLOCK;
    const WgAt w = wg_at(tiles_m, tiles_n, p.groups, gridDim.x);
    const WgCols cols = wg_cols(p, w.g);
    const int m0 = w.tm * 128, n0 = w.tn * 128, pad = (p.kernel - 1) * p.dilation / 2;
    const long R = (long)p.N * p.L, k_begin = (long)w.split * steps_per * WG_BK, k_end = min(R, k_begin + (long)steps_per * WG_BK);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    const bool is_a = tid < 128;
    const int oct = (tid & 127) >> 5, col = (tid & 31) * 4;
    int bt[4], bc[4]; bool on[4];                // columns of x: tap, channel
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int jn = (is_a ? m0 : n0) + col + j;
        on[j] = jn < (is_a ? Og : p.kernel * cols.Cp);
        bt[j] = is_a || !on[j] ? 0 : jn / cols.Cp; bc[j] = is_a || !on[j] ? 0 : jn - bt[j] * cols.Cp + cols.first;
        if (bc[j] >= p.I) on[j] = false;
    }
    f32x16 acc[2][2];
    wg_clear(acc);
    for (long k0 = k_begin; k0 < k_end; k0 += WG_BK) {
        float f[8][4];
        const long r0 = k0 + oct * 8;
        int l = (int)(r0 % p.L);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const long r = r0 + i;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float v = 0.f;
                if (on[j] && r < k_end) {
                    if (is_a) {
                        Raw<T, 1> e; e.load((const T*)p.dy + r * p.O + (long)w.g * Og + m0 + col + j); v = e.at(0);
                    } else {
                        const long sh = (long)bt[j] * p.dilation - pad, ls = l + sh, row = r + sh;
                        if (ls >= 0 && ls < p.L) v = ck_value((uint8_t)p.q[row * p.I + bc[j]], ck_scale(p.q_code[row * nb + bc[j] / CK_BLOCK]));
                    }
                }
                f[i][j] = v;
            }
            l = l + 1 == p.L ? 0 : l + 1;
        }
        __syncthreads();                     // the previous step's fragments have been read
        const auto at = [&](int i, int j) { return f[i][j]; };
        if (is_a) wg_put<TERMS, TERMS == 1 && sizeof(T) == 4, 512>(sa, oct, col, at); else wg_put<1, false, 512>(sb, oct, col, at);
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) wg_mfma<TERMS, 512, 2, 2>(sa, sb, ks, wm, wn, lane, acc);
    }
    wg_store<2, 2>(p, splits, w.split, w.g, m0 + wm, n0 + wn, lane, acc);
}

// The pipelined form.  Two LDS stages: while the matrix instructions of step k run, the piece of step k + 1 is split and stored to the
// other stage and the next loads are under way; one barrier a step.  The first TM threads stage dy, the other TN threads x, each half of the waves runs its own copy of the loop.
// Loads go through buffer descriptors of the split's rows, which return zero behind the end; a row outside its sample is sent there.
// ODD: quads of x or of a bf16 dy may start at any byte; the aligned words around them are loaded and shifted together.
template <int S> struct WgSet { static constexpr int value = S; };

// KP: 32-row blocks of a step; each has waves of its own over the whole tile, whose accumulators are added at the end (through LDS).
template <typename T, int TERMS, int TM, int TN, int WM, int WN, int KP, bool ODD>
__global__ void __launch_bounds__((TM + TN) * KP) wgrad8_kernel(Wgrad8Args p, int splits, int tiles_m, int tiles_n, int steps_per) {
    static_assert((TM / WM) * (TN / WN) * 64 == TM + TN && TM % 64 == 0, "one 8 x 4 piece of an operand tile per thread, whole waves to each operand");
    constexpr int FM = WM / 32, FN = WN / 32, PLANE = TM * 4, BLOCK = TERMS * PLANE + TN * 4, STAGE = KP * BLOCK, BK = WG_BK * KP, SETS = TERMS == 1 || TM == 128 ? 2 : 1, WAVES = (TM / WM) * (TN / WN);
    extern __shared__ u32x4 lds[];           // [2][KP][BLOCK]
    const int Og = p.O / p.groups, nb = (p.I + CK_BLOCK - 1) / CK_BLOCK;
    const WgAt w = wg_at(tiles_m, tiles_n, p.groups, gridDim.x);
    const int m0 = w.tm * TM, n0 = w.tn * TN, pad = (p.kernel - 1) * p.dilation / 2;
    const long R = (long)p.N * p.L, k_begin = (long)w.split * steps_per * WG_BK, k_end = min(R, k_begin + (long)steps_per * WG_BK);
    const int steps = (int)((k_end - k_begin + BK - 1) / BK);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), kp = wave / WAVES;
    const int wm = (wave % WAVES / (TN / WN)) * WM, wn = (wave % (TN / WN)) * WN;
    f32x16 acc[FM][FN];
    wg_clear(acc);

    // load(k, S): the rows of step k into register set S; put(S, stage).  With two sets the loads have a step and a half to arrive: a bf16
    // step of 256 x 256 x 32 is half a microsecond of matrix instructions, less than the way to memory.
    auto loop = [&](auto load, auto put) {
        load(WgSet<0>());
        put(WgSet<0>(), lds);
        if constexpr (SETS == 2) load(WgSet<1>());
        __syncthreads();
        auto step = [&](int odd, auto ahead, auto behind) __attribute__((always_inline)) {      // sets of the next loads and of the next stage
            u32x4* const now = lds + odd * STAGE + kp * BLOCK;
            load(ahead);
            __builtin_amdgcn_sched_barrier(0);
            wg_mfma<TERMS, PLANE, FM, FN>(now, now + TERMS * PLANE, 0, wm, wn, lane, acc);
            wg_mfma<TERMS, PLANE, FM, FN>(now, now + TERMS * PLANE, 1, wm, wn, lane, acc);
            put(behind, lds + (odd ^ 1) * STAGE);
#pragma unroll
            for (int i = 0; i < 2 * TERMS * FM * FN; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);       // a matrix instruction,
                __builtin_amdgcn_sched_group_barrier(0x002, 12, 0);      // twelve vector instructions beside it (eight, second half only: 125 against 120 us in bf16)
            }
            __syncthreads();
        };
        if constexpr (SETS == 2) {
            for (int k = 0; k < steps; k += 2) {
                step(0, WgSet<0>(), WgSet<1>());
                if (k + 1 < steps) step(1, WgSet<1>(), WgSet<0>());
            }
        } else {
            for (int k = 0; k < steps; ++k) step(k & 1, WgSet<0>(), WgSet<0>());
        }
    };
    if (wave < TM * KP / 64) {
        constexpr int SZ = sizeof(T);
        const int octs = tid / (TM / 4), oct = octs & 3, block = (octs >> 2) * BLOCK, col = (tid % (TM / 4)) * 4;
        const long first = (long)w.g * Og + m0;                          // columns behind the group's or the row's end are not stored
        const char* const from = (const char*)p.dy + (k_begin * p.O + first) * SZ;
        const unsigned lead = ODD && SZ == 2 ? (unsigned)((uintptr_t)from & 3) : 0u;      // descriptors start at a whole word
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(from) - lead, 0, (int)((((k_end - k_begin) * p.O - first) * SZ + lead + 3) & ~3L), 0x00020000);
        const unsigned row = (unsigned)p.O * SZ, base = (unsigned)octs * 8 * row + (unsigned)col * SZ + lead;
        unsigned at = base;                                              // of the next load's first row
        if constexpr (ODD && SZ == 2) {
            u32x3 r[SETS][8]; unsigned odd[SETS][8];
            // the word that the last value shares with whatever follows the tensor: as a row behind the end it has to be zero, not a NaN
            const unsigned end = (unsigned)(((k_end - k_begin) * p.O - first) * SZ) + lead;
            loop([&](auto set) __attribute__((always_inline)) {
#pragma unroll
                     for (int i = 0; i < 8; ++i) {
                         const unsigned o = at + (unsigned)i * row;
                         odd[set.value][i] = o & 2; r[set.value][i] = __builtin_amdgcn_raw_buffer_load_b96(rs, o < end ? o & ~3u : 0x80000000u, 0, 0);
                     }
                     at += BK * row;
                 },
                 [&](auto set, u32x4* to) __attribute__((always_inline)) {
                     wg_put<1, false, PLANE>(to + block, oct, col, [&](int i, int j) {
                         const unsigned w = __builtin_amdgcn_alignbyte(r[set.value][i][(j >> 1) + 1], r[set.value][i][j >> 1], odd[set.value][i]);
                         return j & 1 ? bf16_hi(w) : bf16_lo(w);
                     });
                 });
        } else {
            Raw<T, 4> r[SETS][8];
            loop([&](auto set) __attribute__((always_inline)) {
#pragma unroll
                     for (int i = 0; i < 8; ++i) r[set.value][i].load(rs, at + (unsigned)i * row);
                     at += BK * row;
                 },
                 [&](auto set, u32x4* to) __attribute__((always_inline)) {
                     wg_put<TERMS, TERMS == 1 && SZ == 4, PLANE>(to + block, oct, col, [&](int i, int j) { return r[set.value][i].at(j); });
                 });
        }
    } else {
        const int t2 = tid - TM * KP, octs = t2 / (TN / 4), oct = octs & 3, block = (octs >> 2) * BLOCK, col = (t2 % (TN / 4)) * 4;
        const WgCols cols = wg_cols(p, w.g);
        const int tap = (n0 + col) / cols.Cp, ch = n0 + col - tap * cols.Cp + cols.first;
        const bool on = tap < p.kernel && ch < p.I;
        const int shift = on ? tap * p.dilation - pad : 0x60000000;      // a column that does not exist: never inside a sample
        const long b0 = max(0L, k_begin - pad), b1 = min(R, k_end - pad + (long)(p.kernel - 1) * p.dilation);
        const int8_t* const from = p.q + b0 * p.I;
        const unsigned lead = ODD ? (unsigned)((uintptr_t)from & 3) : 0u;
        const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(from) - lead, 0, (int)(((b1 - b0) * p.I + lead + 3) & ~3L), 0x00020000);
        const __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.q_code + b0 * nb), 0, (int)((b1 - b0) * nb), 0x00020000);
        const int row0 = (int)(k_begin - b0) + octs * 8 + (on ? shift : 0), step = BK % p.L;
        unsigned at_q = (unsigned)(row0 * p.I + ch) + lead, at_c = (unsigned)(row0 * nb + ch / CK_BLOCK);      // of the next load's first row
        int l0 = (int)((k_begin + octs * 8) % p.L);                       // and its place in its sample
        unsigned q[SETS][8], c[SETS][8];
        u32x2 wide[SETS][ODD ? 8 : 1];
        loop([&](auto set) __attribute__((always_inline)) {
                 constexpr int S = set.value;
                 int l = l0;
#pragma unroll
                 for (int i = 0; i < 8; ++i) {
                     const unsigned out = (unsigned)(l + shift) < (unsigned)p.L ? 0u : 0x80000000u;      // behind the end of either buffer
                     const unsigned o = at_q + (unsigned)(i * p.I);
                     if constexpr (ODD) { wide[S][i] = __builtin_amdgcn_raw_buffer_load_b64(rq, (o & ~3u) | out, 0, 0); q[S][i] = o; }
                     else q[S][i] = __builtin_amdgcn_raw_buffer_load_b32(rq, o | out, 0, 0);
                     c[S][i] = __builtin_amdgcn_raw_buffer_load_b8(rc, (at_c + (unsigned)(i * nb)) | out, 0, 0);
                     l = l + 1 == p.L ? 0 : l + 1;
                 }
                 at_q += (unsigned)(BK * p.I); at_c += (unsigned)(BK * nb);
                 l0 += step;
                 if (l0 >= p.L) l0 -= p.L;
             },
             [&](auto set, u32x4* to) __attribute__((always_inline)) {
                 constexpr int S = set.value;
                 if constexpr (ODD)
#pragma unroll
                     for (int i = 0; i < 8; ++i) q[S][i] = __builtin_amdgcn_alignbyte(wide[S][i][1], wide[S][i][0], q[S][i]);
                 wg_put<1, false, TN * 4>(to + block + TERMS * PLANE, oct, col, [&](int i, int j) { return ck_value((q[S][i] >> (8 * j)) & 0xffu, ck_scale(c[S][i])); });      // exact
             });
    }
    if constexpr (KP > 1) {
        static_assert(KP == 2 && FM * FN * 16 * WAVES * 64 <= 2 * STAGE * 4, "the second half's accumulators fit the stages");
        float* const other = reinterpret_cast<float*>(lds) + (wave % WAVES) * FM * FN * 16 * 64 + lane;      // the loop ended with a barrier
        if (kp == 1) {
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) other[((i * FN + j) * 16 + e) * 64] = acc[i][j][e];
        }
        __syncthreads();
        if (kp == 1) return;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] += other[((i * FN + j) * 16 + e) * 64];
    }
    wg_store<FM, FN>(p, splits, w.split, w.g, m0 + wm, n0 + wn, lane, acc);
}

// dw = sum over the splits, in split order; slabs [O, kernel, Cg] -> the same (packed) or [O, Cg, kernel].  A workgroup takes one output
// channel and CC input channels with all their taps: the sums cross over in LDS, so that reads and writes are both contiguous.
template <int VEC, int U>
__global__ void __launch_bounds__(512) wgrad8_sum_kernel(Wgrad8Args p, int splits, int CC, int chunks) {
    extern __shared__ float tile[];          // [CC][kernel]
    const int Cg = p.I / p.groups, k = p.kernel, Nn = k * Cg;
    const int o = blockIdx.x / chunks, c0 = (blockIdx.x - o * chunks) * CC, cc = min(CC, Cg - c0), quads = (cc + VEC - 1) / VEC;
    const long slab = (long)p.O * Nn;
    const float* const ws = p.ws + (long)o * Nn + c0;
    for (int i = threadIdx.x; i < quads * k; i += blockDim.x) {
        const int t = i / quads, c = (i - t * quads) * VEC;
        float s[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[j] = 0.f;
        for (int k0 = 0; k0 < splits; k0 += U) {                         // U slabs requested per round trip, added in slab order
            Raw<float, VEC> v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u].load(ws + min(k0 + u, splits - 1) * slab + (long)t * Cg + c);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (k0 + u < splits)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) s[j] += v[u].at(j);
        }
        if (p.packed) store_vec(p.dw + (long)o * Nn + (long)t * Cg + c0 + c, s);
        else
#pragma unroll
            for (int j = 0; j < VEC; ++j) tile[(c + j) * k + t] = s[j];
    }
    if (p.packed) return;
    __syncthreads();
    for (int i = threadIdx.x; i < cc * k; i += blockDim.x) p.dw[(long)o * Nn + (long)c0 * k + i] = tile[i];
}
static int wg_sum(const Wgrad8Args& p, int splits, hipStream_t s) {
    const int Cg = p.I / p.groups;
    int CC = 8192 / p.kernel < 256 ? 8192 / p.kernel : 256;              // at most 32 KB of sums (one channel at least: see wg_check)
    if (CC >= 4) CC &= ~3;
    const int chunks = cdiv(Cg, CC);
    const bool v = Cg % 4 == 0 && CC % 4 == 0 && aligned_to(p.ws, 16) && (!p.packed || aligned_to(p.dw, 16));
    const size_t lds = p.packed ? 0 : (size_t)CC * p.kernel * 4;
    const dim3 grid((unsigned)((long)p.O * chunks));
    // Sixteen slabs a round trip where there are more: 38400 rows, 64 -> 64 channels, kernel 3 (128 slabs): 29.6 -> 24.2 us for the whole call.
    // A vector per thread where 512 hold them: 127 -> 255 channels, kernel 3, 28 splits: 36.2 -> 33.2 us for the whole call
    const int vectors = (Cg < CC ? Cg : CC) * p.kernel / (v ? 4 : 1), threads = vectors >= 512 ? 512 : (vectors + 63) & ~63;
    if (v && splits > 16) hipLaunchKernelGGL((wgrad8_sum_kernel<4, 16>), grid, dim3(threads), lds, s, p, splits, CC, chunks);
    else if (v) hipLaunchKernelGGL((wgrad8_sum_kernel<4, 4>), grid, dim3(threads), lds, s, p, splits, CC, chunks);
    else hipLaunchKernelGGL((wgrad8_sum_kernel<1, 16>), grid, dim3(threads), lds, s, p, splits, CC, chunks);
    return 0;
}

struct WgPlan { int tile, tiles_m, tiles_n, splits, steps_per; bool pipe, odd; };
static WgPlan wg_plan(const Wgrad8Args& p) {
    WgPlan k;
    const long R = (long)p.N * p.L;
    const int Og = p.O / p.groups, Cg = p.I / p.groups, steps = cdiv(R, WG_BK), sz = p.dtype == MTTS_F32 ? 4 : 2;
    // quads of x and of a bf16 dy at whole words
    k.odd = p.I % 4 != 0 || !aligned_to(p.q, 4) || (sz == 2 && (p.O % 4 != 0 || Og % 4 != 0 || !aligned_to(p.dy, 8)));
    k.pipe = true;                               // offsets in a split's rows below 2^31
    const long span = (long)(p.kernel - 1) * p.dilation + 8 * WG_BK, wide = (long)p.O * sz > p.I ? (long)p.O * sz : p.I;
    const long most = (((1L << 31) - 8) / wide - span) / WG_BK;          // steps whose offsets fit
    if (most < 8) k.pipe = false;
    const long Nn = (long)p.kernel * wg_quad_columns(Cg);
    auto tiles = [&](long t) { return cdiv(Og, t) * (long)cdiv(Nn, t) * p.groups; };
    auto split = [&](long t) {                   // one workgroup to a CU; at least six steps each
        long want = tiles(t) > 256 ? 1 : 256 / tiles(t);
        if (want > steps / 6) want = steps / 6;
        return want < 1 ? 1 : want;
    };
    // Six steps at least: 1030 rows, 49 -> 199 channels, kernel 1: 15.7 us, with eight 17.0, four 14.7; 7777 rows, 122 -> 97, kernel 3, bf16:
    // 16.7, 17.3, 19; 256 rows, 512 -> 512, kernel 5 (eight steps in all): 14.6, 14.6, 18.
    // 256 x 256 tiles where they fill three quarters of the CUs with sixteen steps or more each (a partial tile costs its way through
    // memory) and waste less than 0.3 of their area, 128 x 128 of two half steps elsewhere.  Rows, I -> O,
    // kernel, fp32 (bf16) gradients, us of 256 / 128: 38400, 512 -> 512, 5: 245 / 302 (120 / 178); 7680: 69 / 72 (47 / 49); 38400,
    // kernel 1: 72 / 72; 38400, 127 -> 255, 3 (nine steps each): 64 / 46 (54 / 37); 1920, 512 -> 512, 5 (140 workgroups): 40 / 32;
    // 38400, 256 -> 256, 1 (150): 45 / 32; 14400, 128 -> 320, 5 (0.52 of the area): 44 / 35; 38400, 512 -> 80, 5 (0.31): 131 / 87
    const bool big = k.pipe && tiles(256) * split(256) >= 192 && steps >= 16 * split(256) && 10.0 * Og * Nn >= 7.0 * 65536 * (double)(tiles(256) / p.groups);
    k.tile = big ? 256 : 128;
    k.tiles_m = cdiv(Og, k.tile); k.tiles_n = cdiv(Nn, k.tile);
    long want = split(k.tile);
    if (k.pipe && cdiv(steps, want) > most) want = cdiv(steps, most);
    k.steps_per = cdiv(steps, want);
    if (!big && k.steps_per < steps) k.steps_per += k.steps_per & 1;      // whole double steps
    k.splits = cdiv(steps, k.steps_per);
    return k;
}

static int wg_check(const Wgrad8Args& p) {
    MTTS_REQUIRE(p.N > 0 && p.L > 0 && p.I > 0 && p.O > 0 && p.kernel > 0 && p.dilation > 0 && p.groups > 0,
                 "mtts_conv_weight_grad8: empty shape (N %d, L %d, I %d, O %d, kernel %d, dilation %d, groups %d)", p.N, p.L, p.I, p.O, p.kernel, p.dilation, p.groups);
    MTTS_REQUIRE(p.I % p.groups == 0 && p.O % p.groups == 0, "mtts_conv_weight_grad8: %d x %d channels are not a multiple of %d groups", p.I, p.O, p.groups);
    MTTS_REQUIRE(p.dtype == MTTS_F32 || p.dtype == MTTS_BF16, "mtts_conv_weight_grad8: dtype %d is neither MTTS_F32 nor MTTS_BF16", p.dtype);
    MTTS_REQUIRE((long)p.kernel * (p.I / p.groups) < (1L << 28) && (long)(p.kernel - 1) * p.dilation < (1L << 30), "mtts_conv_weight_grad8: kernel %d with dilation %d is too large", p.kernel, p.dilation);
    MTTS_REQUIRE(p.kernel <= 8192 && (long)p.O * (p.I / p.groups) < (1L << 32) / 256, "mtts_conv_weight_grad8: %d output x %d input channels of %d taps are too many for one call", p.O, p.I / p.groups, p.kernel);
    MTTS_REQUIRE(p.L <= 0x7fff0000, "mtts_conv_weight_grad8: %d rows are too many for one call", p.L);      // a row number plus a step's rows fits an int
    const WgPlan k = wg_plan(p);
    MTTS_REQUIRE((long)k.tiles_m * k.tiles_n * p.groups * k.splits < (1L << 32) / 512, "mtts_conv_weight_grad8: too many tiles for one call");
    return 0;
}

MTTS_API long mtts_conv_weight_grad8_workspace_floats(const Wgrad8Args* args) {
    if (wg_check(*args)) return -1;
    const WgPlan k = wg_plan(*args);
    return k.splits > 1 ? (long)k.splits * args->O * args->kernel * (args->I / args->groups) : 0;
}

template <typename T, int TERMS, int TM, int TN, int WM, int WN, int KP, bool ODD> static int wg_launch(const Wgrad8Args& p, const WgPlan& k, hipStream_t s) {
    const size_t lds = 2 * KP * (TERMS * TM * 4 + TN * 4) * sizeof(u32x4);
    const void* fn = (const void*)wgrad8_kernel<T, TERMS, TM, TN, WM, WN, KP, ODD>;
    if (lds > 64 * 1024) MTTS_CHECK_HIP(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    hipLaunchKernelGGL((wgrad8_kernel<T, TERMS, TM, TN, WM, WN, KP, ODD>), dim3(k.tiles_m * k.tiles_n * p.groups * k.splits), dim3((TM + TN) * KP), lds, s, p, k.splits, k.tiles_m, k.tiles_n, k.steps_per);
    return 0;
}
template <typename T, int TERMS, int TM, int TN, int WM, int WN, int KP> static int wg_pipe(const Wgrad8Args& p, const WgPlan& k, hipStream_t s) {
    return k.odd ? wg_launch<T, TERMS, TM, TN, WM, WN, KP, true>(p, k, s) : wg_launch<T, TERMS, TM, TN, WM, WN, KP, false>(p, k, s);
}
template <typename T, int TERMS> static int wg_go(const Wgrad8Args& p, hipStream_t s) {
    const WgPlan k = wg_plan(p);
    if (k.pipe && k.tile == 256) MTTS_TRY((wg_pipe<T, TERMS, 256, 256, 64, 128, 1>(p, k, s)));
    else if (k.pipe) MTTS_TRY((wg_pipe<T, TERMS, 128, 128, 64, 64, 2>(p, k, s)));
    else hipLaunchKernelGGL((wgrad8_edge_kernel<T, TERMS>), dim3(k.tiles_m * k.tiles_n * p.groups * k.splits), dim3(256), 0, s, p, k.splits, k.tiles_m, k.tiles_n, k.steps_per);
    if (k.splits > 1) MTTS_TRY(wg_sum(p, k.splits, s));
    MTTS_CHECK_LAUNCH("conv_weight_grad8");
    return 0;
}

MTTS_API int mtts_conv_weight_grad8(const Wgrad8Args* args, void* stream) {
    const Wgrad8Args p = *args;
    hipStream_t s = (hipStream_t)stream;
    MTTS_TRY(wg_check(p));
    MTTS_REQUIRE(p.q && p.q_code && p.dy && p.dw && (p.ws || mtts_conv_weight_grad8_workspace_floats(&p) == 0), "mtts_conv_weight_grad8: missing tensor");
    const int prec = p.precision ? p.precision : (mtts_get_precision() == 1 ? 1 : 2);      // as GemmArgs.precision
    if (p.dtype == MTTS_BF16) return wg_go<bf16_t, 1>(p, s);
    return prec == 1 ? wg_go<float, 1>(p, s) : wg_go<float, 3>(p, s);
}
