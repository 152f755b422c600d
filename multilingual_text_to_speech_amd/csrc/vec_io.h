// Typed vector access to channel-last activations (fp32 or bf16 storage, fp32 arithmetic) and the 8-bit checkpoint arithmetic, shared by
// group_norm.hip, checkpoint8.hip and wgrad8.hip.
#pragma once
#include "common.h"

typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
// Cache policy of streamed stores (non-temporal): results of 78 MB push the inputs out of L2 otherwise.  Producer, group norm forward and
// backward, consumer in a row at 64 x 600 x 512 fp32: 156 -> 143 us, the forward alone 38.5 -> 28.2 us.
constexpr int BUF_NT = 2;
typedef __attribute__((ext_vector_type(3))) unsigned u32x3;
typedef __attribute__((ext_vector_type(2))) unsigned u32x2;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
typedef __attribute__((ext_vector_type(2))) float f32x2_t;

typedef f32x4 __attribute__((aligned(4))) f32x4_at4;      // at any element
typedef u32x4 __attribute__((aligned(2))) u32x4_at2;

struct bf16_t { uint16_t v; };                 // storage type of MTTS_BF16 tensors

__device__ __forceinline__ float bf16_lo(unsigned w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(unsigned w) { return __uint_as_float(w & 0xffff0000u); }
// two fp32 -> two bf16 in one word, round to nearest even (v_cvt_pk_bf16_f32): off by half a step at most, 2^-8 of the value
__device__ __forceinline__ unsigned bf16_pack(float a, float b) {
    const f32x2_t f = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f, bf16x2_t));
}

// VEC values as they lie in memory: one 16-byte access (4 fp32 / 8 bf16), or one element (VEC = 1).
template <typename T, int VEC> struct Raw;
template <> struct Raw<float, 4> {
    u32x4 w;
    __device__ __forceinline__ void load(const float* p) { w = *reinterpret_cast<const u32x4*>(p); }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, unsigned at) { w = __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0); }
    __device__ __forceinline__ float at(int j) const { return __uint_as_float(w[j]); }
    __device__ __forceinline__ void zero() { w = u32x4{0, 0, 0, 0}; }
};
template <> struct Raw<bf16_t, 4> {
    u32x2 w;
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, unsigned at) { w = __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0); }
    __device__ __forceinline__ float at(int j) const { return j & 1 ? bf16_hi(w[j >> 1]) : bf16_lo(w[j >> 1]); }
};
template <> struct Raw<bf16_t, 8> {
    u32x4 w;
    __device__ __forceinline__ void load(const bf16_t* p) { w = *reinterpret_cast<const u32x4*>(p); }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, unsigned at) { w = __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0); }
    __device__ __forceinline__ float at(int j) const { return j & 1 ? bf16_hi(w[j >> 1]) : bf16_lo(w[j >> 1]); }
    __device__ __forceinline__ void zero() { w = u32x4{0, 0, 0, 0}; }
};
template <> struct Raw<float, 1> {
    float w;
    __device__ __forceinline__ void load(const float* p) { w = *p; }
    __device__ __forceinline__ float at(int) const { return w; }
    __device__ __forceinline__ void zero() { w = 0.f; }
};
template <> struct Raw<bf16_t, 1> {
    uint16_t w;
    __device__ __forceinline__ void load(const bf16_t* p) { w = p->v; }
    __device__ __forceinline__ float at(int) const { return __uint_as_float((unsigned)w << 16); }
    __device__ __forceinline__ void zero() { w = 0; }
};

// The same from any address, and n of VEC elements (the others zero): rows of a width that is no whole number of vectors.  (The hardware
// takes wide accesses at any byte; the compiler makes them of these copies.)
__device__ __forceinline__ void load_any(Raw<float, 4>& r, const float* p, int n) {
    if (n >= 4) { __builtin_memcpy(&r.w, p, 16); return; }
    r.zero();
#pragma unroll
    for (int j = 0; j < 3; ++j) if (j < n) r.w[j] = __float_as_uint(p[j]);
}
__device__ __forceinline__ void load_any(Raw<bf16_t, 8>& r, const bf16_t* p, int n) {
    if (n >= 8) { __builtin_memcpy(&r.w, p, 16); return; }
    r.zero();
#pragma unroll
    for (int j = 0; j < 7; ++j) if (j < n) r.w[j >> 1] |= (unsigned)p[j].v << (16 * (j & 1));
}

template <typename T, int VEC> __device__ __forceinline__ void get_vec(const Raw<T, VEC>& r, float (&f)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = r.at(j);
}

__device__ __forceinline__ void store_vec(float* p, const float (&f)[4]) { *reinterpret_cast<f32x4*>(p) = f32x4{f[0], f[1], f[2], f[3]}; }
__device__ __forceinline__ void stream_vec(float* p, const float (&f)[4]) { const f32x4 v = {f[0], f[1], f[2], f[3]}; __builtin_nontemporal_store(v, reinterpret_cast<f32x4*>(p)); }
__device__ __forceinline__ void stream_vec(float* p, const float (&f)[1]) { *p = f[0]; }
__device__ __forceinline__ void stream_vec(bf16_t* p, const float (&f)[1]) { p->v = (uint16_t)bf16_pack(f[0], 0.f); }
__device__ __forceinline__ void stream_any(float* p, const float (&f)[4], int n) {
    if (n >= 4) { const f32x4 v = {f[0], f[1], f[2], f[3]}; __builtin_nontemporal_store(v, reinterpret_cast<f32x4_at4*>(p)); return; }
#pragma unroll
    for (int j = 0; j < 3; ++j) if (j < n) p[j] = f[j];
}
__device__ __forceinline__ void store_vec(float* p, const float (&f)[1]) { *p = f[0]; }
__device__ __forceinline__ u32x4 pack_vec(const float (&f)[8]) { return u32x4{bf16_pack(f[0], f[1]), bf16_pack(f[2], f[3]), bf16_pack(f[4], f[5]), bf16_pack(f[6], f[7])}; }
__device__ __forceinline__ void stream_vec(bf16_t* p, const float (&f)[8]) { __builtin_nontemporal_store(pack_vec(f), reinterpret_cast<u32x4*>(p)); }
__device__ __forceinline__ void stream_any(bf16_t* p, const float (&f)[8], int n) {
    const u32x4 v = pack_vec(f);
    if (n >= 8) { __builtin_nontemporal_store(v, reinterpret_cast<u32x4_at2*>(p)); return; }
#pragma unroll
    for (int j = 0; j < 7; ++j) if (j < n) p[j].v = (uint16_t)(v[j >> 1] >> (16 * (j & 1)));
}
__device__ __forceinline__ void stream_vec(__amdgpu_buffer_rsrc_t r, unsigned at, const float (&f)[4]) {
    __builtin_amdgcn_raw_buffer_store_b128(u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])}, r, at, 0, BUF_NT);
}
__device__ __forceinline__ void stream_vec(__amdgpu_buffer_rsrc_t r, unsigned at, const float (&f)[8]) { __builtin_amdgcn_raw_buffer_store_b128(pack_vec(f), r, at, 0, BUF_NT); }

// VEC bytes (8-bit values, keep flags)
template <int VEC> struct Bytes;
template <> struct Bytes<1> {
    uint8_t w;
    __device__ __forceinline__ void load(const void* p) { w = *(const uint8_t*)p; }
    __device__ __forceinline__ unsigned get(int) const { return w; }
    __device__ __forceinline__ void fill(unsigned v) { w = (uint8_t)v; }
};
template <> struct Bytes<4> {
    unsigned w;
    __device__ __forceinline__ void load(const void* p) { w = *(const unsigned*)p; }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, unsigned at) { w = __builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0); }
    __device__ __forceinline__ unsigned get(int j) const { return (w >> (8 * j)) & 0xffu; }
    __device__ __forceinline__ void fill(unsigned v) { w = v * 0x01010101u; }
};
template <> struct Bytes<8> {
    u32x2 w;
    __device__ __forceinline__ void load(const void* p) { w = *(const u32x2*)p; }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, unsigned at) { w = __builtin_amdgcn_raw_buffer_load_b64(r, at, 0, 0); }
    __device__ __forceinline__ unsigned get(int j) const { return (w[j >> 2] >> (8 * (j & 3))) & 0xffu; }
    __device__ __forceinline__ void fill(unsigned v) { w = u32x2{v * 0x01010101u, v * 0x01010101u}; }
};

__device__ __forceinline__ void load_any(Bytes<4>& r, const void* p, int n) {
    if (n >= 4) { __builtin_memcpy(&r.w, p, 4); return; }
    r.w = 0;
#pragma unroll
    for (int j = 0; j < 3; ++j) if (j < n) r.w |= (unsigned)((const uint8_t*)p)[j] << (8 * j);
}
__device__ __forceinline__ void load_any(Bytes<8>& r, const void* p, int n) {
    if (n >= 8) { __builtin_memcpy(&r.w, p, 8); return; }
    r.w = u32x2{0, 0};
#pragma unroll
    for (int j = 0; j < 7; ++j) if (j < n) r.w[j >> 2] |= (unsigned)((const uint8_t*)p)[j] << (8 * (j & 3));
}

// ---- 8-bit checkpoint: blocks of 32 channels of a row, value = q * 2^(code - 127) -----------------------------------------------------
// code is the smallest exponent that keeps |round(x / s)| <= 127: with amax = m 2^k, m in [1, 2), amax / 2^(k-6) = 64 m rounds to 128
// exactly when m >= 255/128, i.e. when adding 0x10000 to amax's bits carries into the exponent.  code >= 1 (s >= 2^-126, a normal
// number); a block with an infinity or a NaN has code 255 and q = 0: 0 * inf, it stands for NaN in every place.  The topmost binade
// (code 249) would round up to 64 * 2^122 = 2^128: its quotient stops at 63.  s is a power of two, so x / s and q * s are exact, and
// q * s with its seven significant bits is exact in bf16.
constexpr int CK_BLOCK = 32;
__device__ __forceinline__ unsigned ck_code(unsigned amax_bits) {
    if (amax_bits >= 0x7f800000u) return 255u;
    const int e = (int)((amax_bits + 0x10000u) >> 23) - 6;
    return (unsigned)(e < 1 ? 1 : e);
}
__device__ __forceinline__ int ck_quantise(float x, unsigned code) {
    if (code == 255u) return 0;
    const float inv = __uint_as_float((254u - code) << 23);          // 2^(127 - code): exact for code <= 249
    const float top = code == 249u ? 63.f : 127.f;
    return (int)fminf(fmaxf(rintf(x * inv), -top), top);
}
// four (h = 0) or eight values of a vector, as bytes
template <typename R> __device__ __forceinline__ unsigned ck_word(const R& x, int h, unsigned code) {
    unsigned w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) w |= ((unsigned)ck_quantise(x.at(4 * h + j), code) & 0xffu) << (8 * j);
    return w;
}
// n of the vector's values, to any address
__device__ __forceinline__ void ck_store(int8_t* q, const Raw<float, 4>& x, unsigned code, int n) {
    const unsigned w = ck_word(x, 0, code);
    if (n >= 4) { __builtin_memcpy(q, &w, 4); return; }
#pragma unroll
    for (int j = 0; j < 3; ++j) if (j < n) q[j] = (int8_t)(w >> (8 * j));
}
__device__ __forceinline__ void ck_store(int8_t* q, const Raw<bf16_t, 8>& x, unsigned code, int n) {
    const u32x2 w = {ck_word(x, 0, code), ck_word(x, 1, code)};
    if (n >= 8) { __builtin_memcpy(q, &w, 8); return; }
#pragma unroll
    for (int j = 0; j < 7; ++j) if (j < n) q[j] = (int8_t)(w[j >> 2] >> (8 * (j & 3)));
}
__device__ __forceinline__ void ck_store(__amdgpu_buffer_rsrc_t r, unsigned at, const Raw<float, 4>& x, unsigned code) {
    __builtin_amdgcn_raw_buffer_store_b32(ck_word(x, 0, code), r, at, 0, 0);      // 32-byte pieces of a line, gathered in L2: 44 -> 36 us for the call
}
__device__ __forceinline__ void ck_store(__amdgpu_buffer_rsrc_t r, unsigned at, const Raw<bf16_t, 8>& x, unsigned code) {
    __builtin_amdgcn_raw_buffer_store_b64(u32x2{ck_word(x, 0, code), ck_word(x, 1, code)}, r, at, 0, BUF_NT);
}
__device__ __forceinline__ float ck_scale(unsigned code) { return __uint_as_float(code << 23); }      // 255: infinity
__device__ __forceinline__ float ck_value(unsigned byte, float scale) { return (float)(int)(int8_t)byte * scale; }
__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }    // NaN > infinity > every number
__device__ __forceinline__ unsigned umax_(unsigned a, unsigned b) { return a > b ? a : b; }
template <int CTRL> __device__ __forceinline__ unsigned dpp_u(unsigned x) {
    return (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xF, 0xF, false);
}
// maximum over LANES = 4 or 8 consecutive lanes (the lanes that hold one block); every lane gets it
template <int LANES> __device__ __forceinline__ unsigned block_max(unsigned m) {
    m = umax_(m, dpp_u<0xB1>(m));       // quad_perm [1,0,3,2]
    m = umax_(m, dpp_u<0x4E>(m));       // quad_perm [2,3,0,1]
    if (LANES == 8) m = umax_(m, dpp_u<0x141>(m));      // row_half_mirror
    return m;
}

static inline bool aligned_to(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
