// q8.hip -- activations and weights held in 8 bits with one power-of-two scale per block of 128, the matrix product that reads them and
// the backward passes that read them instead of 16-bit activations.
//
// The format.  A block is 128 neighbouring channels of one row of an [M, C] matrix (a channels-last map is one, M = N*H*W), or a 128 x 128
// tile of a weight matrix.  With a = the largest finite magnitude of the block,
//     e = max(-111, smallest e with a <= 448 * 2^e),       code = e4m3(x / 2^e), round to nearest even,      x^ = code * 2^e.
// Why a power of two: x / 2^e and x^ are exact, so rounding to the code is the ONLY rounding (relative 2^-4 down to 2^-6 * 2^e); x^ has 4
// significant bits and is therefore a bf16 number (and an fp16 number, if x was one), so the 16-bit matrix cores consume it without a
// second rounding; and 2^e is what the block-scaled MFMA of gfx950 takes as its E8M0 operand, so a scale costs the product no VALU work.
// The smallest e keeps x^ in (224, 448] * 2^e for the largest element: nothing saturates, the top element keeps its 2^-4 as well.
//   magnitudes above the largest e4m3 multiple of the source type (1.875 * 2^127; fp16 1.875 * 2^15) count as that number -- rounding up
//   would give the type's infinity; NaN and infinities become the NaN code, and take no part in a; e >= -111 keeps every scale and every
//   non-zero x^ (>= 2^-120) a normal fp32 number: magnitudes under 2^-121 are zero.
//
// Layout: codes [M][ldc] bytes, ldc = C rounded up to 16 (the tail is zero: 16-byte loads never need a column mask); scales
// [ceil(C/128)][lds] bytes, lds = M rounded up to 16, biased by 127 -- block-major, so that a tile's rows of one block are one contiguous
// run.  A weight matrix has the same layout (a 128 x 128 tile's scale repeated for its 128 rows): both operands of the product are read by
// the same code, and because a tile's scale serves rows and columns alike the transposed matrix has the same values.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "h16.h"
#include "mgnet_hip.h"

namespace {

constexpr int TPB = 256;
constexpr int BLK = 128;                  // channels per scale
constexpr int RPG = 8;                    // rows per lane group of the streaming kernels: 8 loads in flight, 8 scale bytes per store
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_ptr;
constexpr int OOB = (int)0x80000000;      // an offset no buffer descriptor below admits: such a load returns (or leaves in LDS) zeros

#ifdef MGN_F16
constexpr float TOP16 = 61440.f;          // largest e4m3 multiple below the type's largest finite number
#else
constexpr float TOP16 = 1.875f * 1.7014118346046923e38f;
#endif
constexpr float TOP32 = 1.875f * 1.7014118346046923e38f;

// This block's number among those of flat_grid() below.  One dimension of a launch holds less than 2^32 work items: what is beyond that is
// dropped without an error.
constexpr int GRID_X_LOG2 = 20;
__device__ __forceinline__ long block_id() { return ((long)blockIdx.y << GRID_X_LOG2) | blockIdx.x; }
// blocks from the number that was asked for up to the grid's own have nothing to do and say so themselves
inline bool flat_grid(long blocks, int threads, dim3* grid) {
    if (blocks * threads <= 0xffffffffL) { *grid = dim3((unsigned)blocks); return true; }
    const long rows = (blocks + (1L << GRID_X_LOG2) - 1) >> GRID_X_LOG2;
    *grid = dim3(1u << GRID_X_LOG2, (unsigned)rows);
    return rows <= 65535;
}

__device__ __forceinline__ float pow2(uint32_t biased) { return __uint_as_float(biased << 23); }
// biased exponent of the scale: a <= 1.75 * 2^E  <=>  the mantissa bits of a do not exceed 0x600000
__device__ __forceinline__ uint32_t scale_of(uint32_t amax_bits) {
    const uint32_t e = (amax_bits + 0x1fffffu) >> 23;
    return e < 24u ? 16u : e - 8u;
}
__device__ __forceinline__ float inv_scale(uint32_t s) { return pow2(254u - s); }

// eight values -> their codes; |v| <= top for finite ones
__device__ __forceinline__ uint2 encode8(const float (&f)[8], float inv, float top) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float c = __builtin_amdgcn_fmed3f(f[k], -top, top) * inv;
        v[k] = (__float_as_uint(f[k]) & 0x7fffffffu) < 0x7f800000u ? c : __uint_as_float(0x7fc00000u);
    }
    uint2 r;
    r.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    r.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], (int)r.x, true);
    r.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
    r.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], (int)r.y, true);
    return r;
}
__device__ __forceinline__ void decode8(uint2 c, float sc, float (&v)[8]) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.x, true);
    const f32x2 d = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.y, false), e = __builtin_amdgcn_cvt_pk_f32_fp8((int)c.y, true);
    v[0] = a[0] * sc; v[1] = a[1] * sc; v[2] = b[0] * sc; v[3] = b[1] * sc;
    v[4] = d[0] * sc; v[5] = d[1] * sc; v[6] = e[0] * sc; v[7] = e[1] * sc;
}
__device__ __forceinline__ uint32_t amax8(const float (&f)[8], float top) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const uint32_t u = __float_as_uint(f[k]) & 0x7fffffffu;
        const uint32_t w = u < 0x7f800000u ? u : 0u;
        m = m > w ? m : w;
    }
    const uint32_t t = __float_as_uint(top);
    return m < t ? m : t;
}
// maximum over LPB neighbouring lanes (4, 8 or 16: inside one DPP row), left in all of them
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t m) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, CTRL, 0xf, 0xf, true);
    return m > o ? m : o;
}
template <int LPB>
__device__ __forceinline__ uint32_t group_max(uint32_t m) {
    m = dpp_max<0xB1>(m);                 // quad: neighbour
    m = dpp_max<0x4E>(m);                 // quad: other pair
    if (LPB >= 8) m = dpp_max<0x141>(m);  // half row mirrored
    if (LPB >= 16) m = dpp_max<0x140>(m); // row mirrored
    return m;
}

__device__ __forceinline__ void unpack8(const uint4& r, float (&v)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) { v[2 * k] = mgn_lo2f(w[k]); v[2 * k + 1] = mgn_hi2f(w[k]); }
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
    return make_uint4(mgn_pack2(v[0], v[1]), mgn_pack2(v[2], v[3]), mgn_pack2(v[4], v[5]), mgn_pack2(v[6], v[7]));
}

// one block's share of a lane, eight 16-bit values: scale of the block (LPB lanes) and codes.  The maximum is taken on the 16-bit words
// (packed), and the conversion divides by the scale itself: a third of the instructions of the general form, which is left for blocks with a
// NaN, an infinity or a magnitude beyond the last e4m3 multiple (all of the group's lanes go one way)
#ifdef MGN_F16
constexpr uint32_t TOPWORD = 0x7b80u;
#define MGN_CVT_FP8(OLD, W, SC, HI) __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(OLD, __builtin_bit_cast(h16x2, W), SC, HI)
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t word_bits(uint32_t m) { return __float_as_uint(mgn_h2f((uint16_t)m)); }
#else
constexpr uint32_t TOPWORD = 0x7f70u;
#define MGN_CVT_FP8(OLD, W, SC, HI) __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(OLD, __builtin_bit_cast(h16x2, W), SC, HI)
typedef __bf16 h16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t word_bits(uint32_t m) { return m << 16; }
#endif
template <int LPB>
__device__ __forceinline__ uint2 quantize8(const uint4& q, uint32_t& s) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    const u16x2 a = __builtin_bit_cast(u16x2, q.x & 0x7fff7fffu), b = __builtin_bit_cast(u16x2, q.y & 0x7fff7fffu);
    const u16x2 c = __builtin_bit_cast(u16x2, q.z & 0x7fff7fffu), d = __builtin_bit_cast(u16x2, q.w & 0x7fff7fffu);
    const u16x2 t = __builtin_elementwise_max(__builtin_elementwise_max(a, b), __builtin_elementwise_max(c, d));
    const uint32_t m = group_max<LPB>(t[0] > t[1] ? t[0] : t[1]);
    if (__builtin_expect(m > TOPWORD, 0)) {
        float f[8];
        unpack8(q, f);
        s = scale_of(group_max<LPB>(amax8(f, TOP16)));
        return encode8(f, inv_scale(s), TOP16);
    }
    s = scale_of(word_bits(m));
    const float sc = pow2(s);
    s16x2 lo = {0, 0}, hi = {0, 0};
    lo = MGN_CVT_FP8(lo, q.x, sc, false);
    lo = MGN_CVT_FP8(lo, q.y, sc, true);
    hi = MGN_CVT_FP8(hi, q.z, sc, false);
    hi = MGN_CVT_FP8(hi, q.w, sc, true);
    return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}

// ------------------------------------------------------------------------------------------------------
// x -> codes, scales.  One pass: a group of LPB lanes owns one block of 8 consecutive rows (8 channels a lane), so a block's maximum is
// four DPP steps and its eight scales leave in one store; the 8 rows are 8 independent 16-byte loads per lane.  Bound by HBM (3 bytes per
// 16-bit value): 262144 x 256 bf16 in 39.6 us, 5.1 TB/s, the rate of a large copy (5.12); back in 30.2 us, the codes still in the last cache.
// ------------------------------------------------------------------------------------------------------
struct RowMap {                           // row r of the matrix = pixel (n, h, w) of a map with these strides (elements)
    long sn, sh, sw;
    int H, W;
    int flat;                             // 1: row r starts at r * sw
};
__device__ __forceinline__ long row_offset(const RowMap& m, int r) {
    if (m.flat) return (long)r * m.sw;
    const int q = r / m.W, w = r - q * m.W, n = q / m.H, h = q - n * m.H;
    return (long)n * m.sn + (long)h * m.sh + (long)w * m.sw;
}

// 16, 8 and 4 bytes at any address that suits an element: global loads and stores need no more, so that rows of any pitch move alike
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32_any __attribute__((aligned(2)));

template <typename T> struct Src;
template <> struct Src<float> {
    struct Raw { u32x4_any a, b; };
    static constexpr float TOP = TOP32;
    __device__ static Raw zero() { return Raw{}; }
    __device__ static float one(const float* p) { return *p; }
    __device__ static Raw load(const float* p) { return Raw{*reinterpret_cast<const u32x4_any*>(p), *reinterpret_cast<const u32x4_any*>(p + 4)}; }
    __device__ static Raw tail(const float* p, int t) {   // t < 8 values, zeros behind them
        Raw r{};
        u32x4_any v = {0, 0, 0, 0};
        if (t & 4) { r.a = *reinterpret_cast<const u32x4_any*>(p); p += 4; }
        if (t & 2) { const u32x2_any w = *reinterpret_cast<const u32x2_any*>(p); v.x = w.x; v.y = w.y; p += 2; }
        if (t & 1) { if (t & 2) v.z = __float_as_uint(*p); else v.x = __float_as_uint(*p); }
        if (t & 4) r.b = v; else r.a = v;
        return r;
    }
    __device__ static void get(const Raw& r, float (&v)[8]) {
#pragma unroll
        for (int k = 0; k < 4; ++k) { v[k] = __uint_as_float(r.a[k]); v[k + 4] = __uint_as_float(r.b[k]); }
    }
};
template <> struct Src<uint16_t> {
    struct Raw { uint4 a; };
    static constexpr float TOP = TOP16;
    __device__ static Raw zero() { return Raw{make_uint4(0, 0, 0, 0)}; }
    __device__ static float one(const uint16_t* p) { return mgn_h2f(*p); }
    __device__ static void get(const Raw& r, float (&v)[8]) { unpack8(r.a, v); }
    __device__ static Raw load(const uint16_t* p) { const u32x4_any v = *reinterpret_cast<const u32x4_any*>(p); return Raw{make_uint4(v.x, v.y, v.z, v.w)}; }
    __device__ static Raw tail(const uint16_t* p, int t) {
        u32x2_any lo = {0, 0};
        uint32_t x = 0, y = 0;
        if (t & 4) { lo = *reinterpret_cast<const u32x2_any*>(p); p += 4; }
        if (t & 2) { x = *reinterpret_cast<const u32_any*>(p); p += 2; }
        if (t & 1) { if (t & 2) y = *p; else x = *p; }
        return (t & 4) ? Raw{make_uint4(lo.x, lo.y, x, y)} : Raw{make_uint4(x, y, 0, 0)};
    }
};

template <typename T, int LPB>
__global__ __launch_bounds__(TPB) void q8_pack(const T* __restrict__ x, RowMap map, int M, int C, int nb, int ldc, long lds,
                                               unsigned char* __restrict__ codes, unsigned char* __restrict__ scales) {
    const long gid = block_id() * (TPB / LPB) + threadIdx.x / LPB;
    const int l = threadIdx.x % LPB;
    const int kb = (int)(gid % nb);
    const long r0l = gid / nb * RPG;
    if (r0l >= M) return;                 // (whole groups leave together: the DPP steps below stay inside one group)
    const int r0 = (int)r0l, c0 = kb * BLK + l * 8;
    uint32_t sb[RPG];
    typename Src<T>::Raw q[RPG];
    if (c0 + 8 <= C || c0 >= C) {
#pragma unroll
        for (int j = 0; j < RPG; ++j) q[j] = (r0 + j < M && c0 < C) ? Src<T>::load(x + row_offset(map, r0 + j) + c0) : Src<T>::zero();
    } else {
#pragma unroll
        for (int j = 0; j < RPG; ++j) q[j] = r0 + j < M ? Src<T>::tail(x + row_offset(map, r0 + j) + c0, C - c0) : Src<T>::zero();
    }
#pragma unroll
    for (int j = 0; j < RPG; ++j) {
        uint2 e;
        if constexpr (sizeof(T) == 2) {
            e = quantize8<LPB>(q[j].a, sb[j]);
        } else {
            float f[8];
            Src<T>::get(q[j], f);
            sb[j] = scale_of(group_max<LPB>(amax8(f, Src<T>::TOP)));
            e = encode8(f, inv_scale(sb[j]), Src<T>::TOP);
        }
        if (r0 + j < M && c0 < ldc) *reinterpret_cast<uint2*>(codes + (long)(r0 + j) * ldc + c0) = e;
    }
    if (l == 0) {                         // lds is a multiple of 16: eight bytes from a row that is a multiple of 8 stay inside it
        const uint2 w = make_uint2(sb[0] | (sb[1] << 8) | (sb[2] << 16) | (sb[3] << 24), sb[4] | (sb[5] << 8) | (sb[6] << 16) | (sb[7] << 24));
        *reinterpret_cast<uint2*>(scales + kb * lds + r0) = w;
    }
}

// codes, scales -> x^ [M][C] (rows of C contiguous values); the mirror image of q8_pack.  A lane writes 16 bytes at a time, neighbours side by
// side: of 16-bit values its 8 channels, of 32-bit ones 4 channels in either half of the block (60M values: 62 us against 75
// with 8 in a row, whose two stores lie 32 bytes apart)
template <typename T, int LPB>
__global__ __launch_bounds__(TPB) void q8_unpack(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales, int M, int C,
                                                 int nb, int ldc, long lds, T* __restrict__ y) {
    const long gid = block_id() * (TPB / LPB) + threadIdx.x / LPB;
    const int l = threadIdx.x % LPB;
    const int kb = (int)(gid % nb);
    const long r0l = gid / nb * RPG;
    if (r0l >= M) return;
    constexpr bool HALF = sizeof(T) == 2;
    const int r0 = (int)r0l, c0 = kb * BLK + l * (HALF ? 8 : 4), c1 = c0 + (HALF ? 4 : 4 * LPB);   // two runs of 4 channels
    if (c0 >= C) return;
    const uint2 w = *reinterpret_cast<const uint2*>(scales + kb * lds + r0);
    uint2 q[RPG];
#pragma unroll
    for (int j = 0; j < RPG; ++j) {
        const unsigned char* p = codes + (long)(r0 + j) * ldc;
        if (r0 + j >= M) q[j] = make_uint2(0, 0);
        else if (HALF) q[j] = *reinterpret_cast<const uint2*>(p + c0);
        else q[j] = make_uint2(*reinterpret_cast<const uint32_t*>(p + c0), c1 < C ? *reinterpret_cast<const uint32_t*>(p + c1) : 0);
    }
#pragma unroll
    for (int j = 0; j < RPG; ++j) {
        if (r0 + j >= M) break;
        float v[8];
        decode8(q[j], pow2(((j < 4 ? w.x : w.y) >> (8 * (j & 3))) & 0xffu), v);
        T* row = y + (long)(r0 + j) * C;
        if constexpr (HALF) {
            const uint4 o = pack8(v);
            T* p = row + c0;
            if (c0 + 8 <= C) {
                *reinterpret_cast<u32x4_any*>(p) = u32x4_any{o.x, o.y, o.z, o.w};
            } else {
                const int t = C - c0;
                uint32_t a = o.x, b = o.y;
                if (t & 4) { *reinterpret_cast<u32x2_any*>(p) = u32x2_any{a, b}; a = o.z; b = o.w; p += 4; }
                if (t & 2) { *reinterpret_cast<u32_any*>(p) = a; a = b; p += 2; }
                if (t & 1) *p = (T)a;
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int c = h ? c1 : c0;
                if (c + 4 <= C) {
                    *reinterpret_cast<u32x4_any*>(row + c) = u32x4_any{__float_as_uint(v[4 * h]), __float_as_uint(v[4 * h + 1]), __float_as_uint(v[4 * h + 2]), __float_as_uint(v[4 * h + 3])};
                } else {
#pragma unroll
                    for (int k = 0; k < 3; ++k) if (c + k < C) row[c + k] = v[4 * h + k];
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------
// a weight matrix W [N][K] (any strides) -> codes [N][ldc(K)] + scales [ceil(K/128)][lds(N)], and the same values transposed: codes
// [K][ldc(N)] + scales [ceil(N/128)][lds(K)] (what the data gradient multiplies by).  A block per 128 x 128 tile; the tile goes through
// LDS once so that both outputs leave in 16-byte stores.  A layer has few tiles: 256 x 256 fp32 takes 5.5 us, the latency of one block's load,
// maximum, conversion and two stores (8.2 with a scalar load and a byte store to LDS for each value); 8192 x 8192 takes 85 us, 3.9 TB/s.
// ------------------------------------------------------------------------------------------------------
constexpr int TILE_TPB = 1024;            // 16 values a thread (64: 11 us for the same layer)
template <typename T>
__global__ __launch_bounds__(TILE_TPB) void q8_pack_tile(const T* __restrict__ w, long sr, long sc, int N, int K, unsigned char* __restrict__ codes,
                                                    unsigned char* __restrict__ scales, unsigned char* __restrict__ codes_t,
                                                    unsigned char* __restrict__ scales_t) {
    constexpr int PITCH = BLK + 4;        // (33 words: the transposing byte reads spread over the banks)
    __shared__ uint32_t tile[BLK * PITCH / 4];
    __shared__ uint32_t part[TILE_TPB / 64];
    const int n0 = blockIdx.x * BLK, k0 = blockIdx.y * BLK, tid = threadIdx.x;
    const int ldk = (K + 15) & ~15, ldn = (N + 15) & ~15;
    // A thread has 16 neighbours along the fast axis, the contiguous one.  Along it the codes leave from registers; the transposed ones go
    // through LDS.
    const bool kfast = sc == 1 || sr != 1;
    const int ns = kfast ? N : K, nf = kfast ? K : N, s0 = kfast ? n0 : k0, f0 = kfast ? k0 : n0, lds = kfast ? ldn : ldk, ldf = kfast ? ldk : ldn;
    const long ss = kfast ? sr : sc, sf = kfast ? sc : sr;
    unsigned char *const direct = kfast ? codes : codes_t, *const turned = kfast ? codes_t : codes;
    const int row = tid >> 3, ch = (tid & 7) * 16;
    const T* p = w + (long)(s0 + row) * ss + (long)(f0 + ch) * sf;
    float f[2][8];
    if (s0 + row < ns && sf == 1 && f0 + ch + 16 <= nf) {
        const typename Src<T>::Raw a = Src<T>::load(p), b = Src<T>::load(p + 8);
        Src<T>::get(a, f[0]);
        Src<T>::get(b, f[1]);
    } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) f[k >> 3][k & 7] = (s0 + row < ns && f0 + ch + k < nf) ? Src<T>::one(p + k * sf) : 0.f;
    }
    uint32_t m = amax8(f[0], Src<T>::TOP);
    const uint32_t m1 = amax8(f[1], Src<T>::TOP);
    m = group_max<16>(m > m1 ? m : m1);
#pragma unroll
    for (int d = 16; d < 64; d <<= 1) { const uint32_t o = (uint32_t)__shfl_xor((int)m, d); m = m > o ? m : o; }
    if ((tid & 63) == 0) part[tid >> 6] = m;
    __syncthreads();
    m = part[0];
#pragma unroll
    for (int k = 1; k < TILE_TPB / 64; ++k) m = m > part[k] ? m : part[k];
    const uint32_t s = scale_of(m);
    const float inv = inv_scale(s);
    const uint2 e0 = encode8(f[0], inv, Src<T>::TOP), e1 = encode8(f[1], inv, Src<T>::TOP);
    if (direct && s0 + row < ns && f0 + ch < ldf) *reinterpret_cast<uint4*>(direct + (long)(s0 + row) * ldf + f0 + ch) = make_uint4(e0.x, e0.y, e1.x, e1.y);
    if (turned) {
        uint32_t* d = tile + (row * PITCH + ch) / 4;
        d[0] = e0.x, d[1] = e0.y, d[2] = e1.x, d[3] = e1.y;
        __syncthreads();
        if (f0 + row < nf && s0 + ch < lds) {
            const unsigned char* t = reinterpret_cast<const unsigned char*>(tile) + ch * PITCH + row;
            uint32_t o[4];
#pragma unroll
            for (int q = 0; q < 4; ++q, t += 4 * PITCH)
                o[q] = (uint32_t)t[0] | ((uint32_t)t[PITCH] << 8) | ((uint32_t)t[2 * PITCH] << 16) | ((uint32_t)t[3 * PITCH] << 24);
            *reinterpret_cast<uint4*>(turned + (long)(f0 + row) * lds + s0 + ch) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
    if (tid < BLK) {
        if (codes && n0 + tid < N) scales[(long)blockIdx.y * ldn + n0 + tid] = (unsigned char)s;
        if (codes_t && k0 + tid < K) scales_t[(long)blockIdx.x * ldk + k0 + tid] = (unsigned char)s;
    }
}

// ------------------------------------------------------------------------------------------------------
// out[m][n] = act( sum_k A[m][k] B[n][k] + bias[n] )
//   v_mfma_scale_f32_32x32x64_f8f6f4 with the two blocks' exponents as its E8M0 operands: products of codes scaled in the matrix core,
//   fp32 accumulation, one rounding at the end.  B's rows are the instruction's rows and A's its columns, so a lane ends up with 4
//   consecutive n of one m.  The k order inside a block is free (both operands are read alike and share the block's scale).
//   Precision, measured on the instruction: it adds the products of 8 neighbouring k before they join the fp32 accumulator, each cut
//   towards zero to a multiple of 2^-13 of the largest one's binade.  1.3e-5 of a result (2-norm, Gaussian operands): far below the
//   rounding to 16 bits (1.7e-3 / 2.1e-4) and the operands' own (2.6e-2); a 32-bit result carries it.
//   Kernels, by size (the rules stand in mgn_q8_matmul): q8_mm_small for few tiles, q8_stream_* for K <= 512 and many rows, q8_mm_128x32 for
//   N <= 32, q8_mm_128x128 and q8_mm_256x256.
// ------------------------------------------------------------------------------------------------------
// act(v) without a branch: ReLU is lo = 0, neg = 1; leaky ReLU lo = -inf, neg = slope (0 < slope <= 1); none lo = -inf, neg = 1.  `maximum`
// passes a NaN on.
struct Act { float lo, neg; };
__device__ __forceinline__ float activate(float v, const Act& a) {
    v = __builtin_elementwise_maximum(v, a.lo);
    return __builtin_elementwise_maximum(v, v * a.neg);
}
inline Act make_act(int act, float slope) {
    const bool relu = act == 1 || (act == 2 && slope == 0.f);
    return Act{relu ? 0.f : -__builtin_inff(), act == 2 && !relu ? slope : 1.f};
}
inline bool act_ok(int act, float slope) { return act == 0 || act == 1 || (act == 2 && slope >= 0.f && slope <= 1.f); }
struct MmParams {
    const unsigned char *a, *sa, *b, *sb;
    const float* bias;
    void* out;
    int M, N, K, nb, ld;                  // ld: bytes per code row (both operands)
    long lda_s, ldb_s, ldo;               // scale rows; elements per row of out
    Act act;
    int out32;
    int mt, nt;
};
MGN_PLAN_RO(MmParams, MGN_RO(a) MGN_RO(sa) MGN_RO(b) MGN_RO(sb) MGN_RO(bias))

// four consecutive n of row m
template <typename P>
__device__ __forceinline__ void mm_emit(const P& p, long m, int n, const float (&v)[4]) {
    float r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float b = (p.bias && n + e < p.N) ? p.bias[n + e] : 0.f;
        r[e] = activate(v[e] + b, p.act);
    }
    if (p.out32) {
        float* o = (float*)p.out + m * p.ldo + n;
        if (n + 3 < p.N) { *reinterpret_cast<u32x4_any*>(o) = __builtin_bit_cast(u32x4_any, make_float4(r[0], r[1], r[2], r[3])); return; }
#pragma unroll
        for (int e = 0; e < 4; ++e) if (n + e < p.N) o[e] = r[e];
    } else {
        uint16_t* o = (uint16_t*)p.out + m * p.ldo + n;
        const uint2 w = make_uint2(mgn_pack2(r[0], r[1]), mgn_pack2(r[2], r[3]));
        if (n + 3 < p.N) { *reinterpret_cast<u32x2_any*>(o) = u32x2_any{w.x, w.y}; return; }
#pragma unroll
        for (int e = 0; e < 4; ++e) if (n + e < p.N) o[e] = (uint16_t)((e < 2 ? w.x : w.y) >> (16 * (e & 1)));
    }
}

template <int BM, int BN, int WVM, int WVN, int ST>
struct MmTile {
    static constexpr int NW = WVM * WVN, TM = BM / WVM / 32, TN = BN / WVN / 32;
    static constexpr int ABYTES = BM * BLK, STAGE = (BM + BN) * BLK, SCALES = 512;   // [256 rows of A][256 rows of B]
    static constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW;                           // 1-KB pieces (8 rows) per wave and stage
    static constexpr int LDS = ST * (STAGE + SCALES), OUT = 32 * (TN * 32 * 4 + 16);     // OUT: a wave's share on the way out
    static_assert(NW * OUT <= LDS && PA * NW * 8 == BM && (PB * NW * 8 == BN) && BM <= 256 && BN <= 256 && NW % 2 == 0, "tile shape");
};

// the accumulators of TM x TN 32 x 32 tiles (channels by 4 in a lane, rows over lanes) as rows of out from (m0, n0); `sm`: the wave's own LDS
template <int TM, int TN, typename T>
__device__ __forceinline__ void mm_store(const MmParams& p, const f32x16 (&acc)[TN][TM], unsigned char* sm, long m0, int n0, int lane) {
    constexpr int E = 16 / sizeof(T), PITCH = TN * 32 * sizeof(T) + 16, CHUNKS = TN * 32 / E, ROWS = 64 / CHUNKS;
    const int lr = lane & 31, hi = lane >> 5, row = lane / CHUNKS, n = n0 + lane % CHUNKS * E;
    float bias[TN][16];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int c = n0 + i * 32 + 8 * (e >> 2) + 4 * hi + (e & 3);
            bias[i][e] = (p.bias && c < p.N) ? p.bias[c] : 0.f;
        }
#pragma unroll
    for (int j = 0; j < TM; ++j) {
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float r[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] = activate(acc[i][j][4 * q + e] + bias[i][4 * q + e], p.act);
                unsigned char* d = sm + lr * PITCH + (i * 32 + 8 * q + 4 * hi) * sizeof(T);
                if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(d) = make_float4(r[0], r[1], r[2], r[3]);
                else *reinterpret_cast<uint2*>(d) = make_uint2(mgn_pack2(r[0], r[1]), mgn_pack2(r[2], r[3]));
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (LDS keeps a wave's order: the next 32 rows need no wait)
#pragma unroll
        for (int it = 0; it < 32 / ROWS; ++it) {
            const long m = m0 + j * 32 + it * ROWS + row;
            const uint4 w = *reinterpret_cast<const uint4*>(sm + (it * ROWS + row) * PITCH + lane % CHUNKS * 16);
            if (m >= p.M || n >= p.N) continue;
            T* o = (T*)p.out + m * p.ldo + n;
            if (n + E <= p.N) {
                *reinterpret_cast<u32x4_any*>(o) = u32x4_any{w.x, w.y, w.z, w.w};
            } else {
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (n + e < p.N) {
                        if constexpr (sizeof(T) == 4) o[e] = __builtin_bit_cast(float, u[e]);
                        else o[e] = (uint16_t)(u[e >> 1] >> (16 * (e & 1)));
                    }
            }
        }
        asm volatile("" ::: "memory");
    }
}

// The tile of this block.  Tiles are counted through groups of 4 row tiles, in a group column by column; XCD x (= blockIdx % 8) takes the
// x-th eighth of that sequence, so that the XCDs have equal shares and the tiles in flight on one share rows and columns in its L2.
__device__ __forceinline__ bool mm_tile(const MmParams& p, int& mtile, int& ntile) {
    constexpr int G = 4;
    const long total = (long)p.mt * p.nt, id = block_id();
    const int x = (int)id & 7;
    const long first = total * x >> 3;
    if (first + (id >> 3) >= total * (x + 1) >> 3) return false;
    const int t = (int)(first + (id >> 3));
    const int g = t / (G * p.nt), in = t - g * G * p.nt, rows = p.mt - g * G < G ? p.mt - g * G : G;
    ntile = in / rows, mtile = g * G + in - ntile * rows;
    return true;
}

constexpr int loads_left(int n) { return (n & 15) | ((n >> 4) << 14) | 0x0070; }   // s_waitcnt vmcnt(n) lgkmcnt(0)

// A block computes a BM x BN tile; a step covers one block of 128 k.  Rows travel HBM/L2 -> LDS by LDS-DMA (16 bytes a lane, 8 rows a
// piece), ST stages; 16-byte chunk c of row r lies at position c ^ ((r >> 1) & 7), so that the 16-byte fragment reads of 16 neighbouring
// rows cover every bank once.  128 x 128: two stages leave room for two blocks a CU, whose matrix and load phases fill each other's gaps
// (four stages and one block: 8192^3 631 us against 490); 2048^3 15.3 us, 1.1 PFLOP/s, 256 blocks, one a CU and its step's latency.
// 128 x 32: bound by reading A, three stages (100000 x 8 x 4096: 90 us against 106 with two; its 410 MB take 80 at the rate of a copy).
template <int BM, int BN, int WVM, int WVN, int ST>
__device__ __forceinline__ void q8_mm_body(const MmParams& p) {
    using Tl = MmTile<BM, BN, WVM, WVN, ST>;
    extern __shared__ __attribute__((aligned(16))) unsigned char q8_sm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int mtile, ntile;
    if (!mm_tile(p, mtile, ntile)) return;
    const long m0 = (long)mtile * BM;
    const int n0 = ntile * BN;
    const int rowsA = (int)(p.M - m0 < BM ? p.M - m0 : BM), rowsB = p.N - n0 < BN ? p.N - n0 : BN;
    const __amdgpu_buffer_rsrc_t rsA = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.a + m0 * p.ld), 0, (uint32_t)(rowsA * p.ld), 0x00020000);
    const __amdgpu_buffer_rsrc_t rsB = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.b + (long)n0 * p.ld), 0, (uint32_t)(rowsB * p.ld), 0x00020000);
    // scale rows: 4 bytes a lane from row 4 * lane; rows are padded to 16, so whole words of this tile's rows never leave the scale row
    const int sra = (rowsA + 3) >> 2, srb = (rowsB + 3) >> 2;

    int offA[Tl::PA], offB[Tl::PB];
    const int col = ((lane & 7) ^ ((wave * 4 + (lane >> 4)) & 7)) << 4;   // (the swizzle of row r is the same for all pieces of a wave)
#pragma unroll
    for (int q = 0; q < Tl::PA; ++q) {
        const int r = (wave + Tl::NW * q) * 8 + (lane >> 3);
        offA[q] = r < rowsA ? r * p.ld + col : OOB;
    }
#pragma unroll
    for (int q = 0; q < Tl::PB; ++q) {
        const int r = (wave + Tl::NW * q) * 8 + (lane >> 3);
        offB[q] = r < rowsB ? r * p.ld + col : OOB;
    }
    auto issue = [&](int kb, unsigned char* st) {
        const int k0 = kb * BLK;
        const bool in = k0 + col < p.ld;   // (OOB + k0 stays beyond every descriptor; steps behind the last one load nothing)
#pragma unroll
        for (int q = 0; q < Tl::PA; ++q)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsA, (lds_ptr)(st + (wave + Tl::NW * q) * 1024), 16, in ? offA[q] + k0 : OOB, 0, 0, 0);
#pragma unroll
        for (int q = 0; q < Tl::PB; ++q)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsB, (lds_ptr)(st + Tl::ABYTES + (wave + Tl::NW * q) * 1024), 16, in ? offB[q] + k0 : OOB, 0, 0, 0);
        if (wave < 2) {                   // wave 0: A's scales, wave 1: B's
            const unsigned char* s = wave == 0 ? p.sa + (long)kb * p.lda_s + m0 : p.sb + (long)kb * p.ldb_s + n0;
            const int words = kb < p.nb ? (wave == 0 ? sra : srb) : 0;
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(s), 0, (uint32_t)(words * 4), 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(st + Tl::STAGE + wave * 256), 4, lane < words ? lane * 4 : OOB, 0, 0, 0);
        }
    };

    const int wm = wave / WVN, wn = wave % WVN, lr = lane & 31, hi = lane >> 5;
    f32x16 acc[Tl::TN][Tl::TM];
#pragma unroll
    for (int i = 0; i < Tl::TN; ++i)
#pragma unroll
        for (int j = 0; j < Tl::TM; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    const int sw = (lr >> 1) & 7;         // (tile bases are multiples of 32 rows)
    // One step: start the next stage's loads, multiply this one.  The two pointers are restrict (and the waits outside) because the compiler
    // otherwise takes every LDS read after an LDS-DMA for a read of its target and puts a full s_waitcnt vmcnt(0) between the two, which
    // makes the two stages one: measured 1.9x on a large product.
    auto step = [&](int kb, const unsigned char* __restrict__ st, unsigned char* __restrict__ next) {
        issue(kb + ST - 1, next);
        int xs[Tl::TM], ws[Tl::TN];
#pragma unroll
        for (int j = 0; j < Tl::TM; ++j) xs[j] = st[Tl::STAGE + (wm * Tl::TM + j) * 32 + lr];
#pragma unroll
        for (int i = 0; i < Tl::TN; ++i) ws[i] = st[Tl::STAGE + 256 + (wn * Tl::TN + i) * 32 + lr];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const int c0 = ((kk * 4 + hi * 2) ^ sw) << 4, c1 = ((kk * 4 + hi * 2 + 1) ^ sw) << 4;
            i32x8 x[Tl::TM], w[Tl::TN];
#pragma unroll
            for (int j = 0; j < Tl::TM; ++j) {
                const unsigned char* row = st + ((wm * Tl::TM + j) * 32 + lr) * BLK;
                const int4 u = *reinterpret_cast<const int4*>(row + c0), v = *reinterpret_cast<const int4*>(row + c1);
                x[j] = i32x8{u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
            }
#pragma unroll
            for (int i = 0; i < Tl::TN; ++i) {
                const unsigned char* row = st + Tl::ABYTES + ((wn * Tl::TN + i) * 32 + lr) * BLK;
                const int4 u = *reinterpret_cast<const int4*>(row + c0), v = *reinterpret_cast<const int4*>(row + c1);
                w[i] = i32x8{u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
            }
#pragma unroll
            for (int i = 0; i < Tl::TN; ++i)
#pragma unroll
                for (int j = 0; j < Tl::TM; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[i], x[j], acc[i][j], 0, 0, 0, ws[i], 0, xs[j]);
        }
    };
    // `ahead` stages' loads are in flight behind the one that is waited for: PA + PB each, one more in the two waves of the scales.  (This
    // wave's reads of the step before are through as well: their stage is the next to be loaded.)
    auto landed = [&]() {
        constexpr int ahead = ST - 2;
        if (wave < 2) __builtin_amdgcn_s_waitcnt(loads_left(ahead * (Tl::PA + Tl::PB + 1)));
        else __builtin_amdgcn_s_waitcnt(loads_left(ahead * (Tl::PA + Tl::PB)));
        asm volatile("" ::: "memory");
    };
#pragma unroll
    for (int k = 0; k < ST - 1; ++k) issue(k, q8_sm + k * (Tl::STAGE + Tl::SCALES));
    int cur = 0;
    for (int kb = 0; kb < p.nb; ++kb) {
        landed();
        __builtin_amdgcn_s_barrier();     // everyone's rows of step kb have landed, and step kb - 1 has been read
        const int nxt = cur == 0 ? ST - 1 : cur - 1;
        step(kb, q8_sm + cur * (Tl::STAGE + Tl::SCALES), q8_sm + nxt * (Tl::STAGE + Tl::SCALES));
        cur = cur == ST - 1 ? 0 : cur + 1;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (empty loads behind the last step write their stages as well)
    // A wave's 32 rows of 32 TN channels go through LDS, so that they leave as whole row segments, 16 bytes a lane: with 8-byte stores of
    // each lane's own 4 channels (16 bytes of a row side by side) the write-back of short products is bound by the number of requests.
    // Rows of out need no alignment beyond their element's (global stores take any address).
    __syncthreads();                      // the last stage has been read
    if (p.out32) mm_store<Tl::TM, Tl::TN, float>(p, acc, q8_sm + wave * Tl::OUT, m0 + wm * Tl::TM * 32, n0 + wn * Tl::TN * 32, lane);
    else mm_store<Tl::TM, Tl::TN, uint16_t>(p, acc, q8_sm + wave * Tl::OUT, m0 + wm * Tl::TM * 32, n0 + wn * Tl::TN * 32, lane);
}

// Large products: 256 x 256 outputs by eight waves (each 128 x 64: 4 x 2 MFMA tiles), 64 k at a time through a ring of four LDS stages.
// The waves work in two groups, one slot apart: while one group multiplies (8 MFMAs), the other one reads its next 64 k from LDS and starts
// the loads of three stages later, so that matrix cores, LDS and loads run together.  Group 0 reads stage h in slot 2h and multiplies in
// slot 2h + 1, group 1 a slot later; a barrier ends each slot.  Stage h + 3 takes the place of stage h - 1, which group 1 read in slot 2h - 1;
// every wave has waited for its part of stage h + 1 when slot 2h + 1 ends.
// 8192^3: 421-455 us, 2.4-2.6 PFLOP/s (the library's product with one scale per tensor 2.6).  The matrix cores are busy in 70 % of the
// cycles, and the clock is down to 1.7-2.0 GHz: what is left is bound by power.  (One slot for all waves, two stages of 128 k: 10 % more
// cycles; without any loads of the next stage 330 us, without LDS reads 370, without MFMAs 308.)
struct Mm256 {
    static constexpr int ABYTES = 256 * 64, STAGE = 2 * ABYTES + 512, ST = 4, TM = 4, TN = 2, OUT = 32 * (TN * 32 * 4 + 16);
    static constexpr int LDS = ST * STAGE;
    static_assert(8 * OUT <= LDS, "the way out");
};
__global__ __launch_bounds__(512, 1) void q8_mm_256x256(MmParams p) {
    using Tl = Mm256;
    constexpr int TM = Tl::TM, TN = Tl::TN;
    extern __shared__ __attribute__((aligned(16))) unsigned char q8_sm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 31, hi = lane >> 5;
    int mtile, ntile;
    if (!mm_tile(p, mtile, ntile)) return;
    const long m0 = (long)mtile * 256;
    const int n0 = ntile * 256;
    const int rowsA = (int)(p.M - m0 < 256 ? p.M - m0 : 256), rowsB = p.N - n0 < 256 ? p.N - n0 : 256;
    const __amdgpu_buffer_rsrc_t rsA = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.a + m0 * p.ld), 0, (uint32_t)(rowsA * p.ld), 0x00020000);
    const __amdgpu_buffer_rsrc_t rsB = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.b + (long)n0 * p.ld), 0, (uint32_t)(rowsB * p.ld), 0x00020000);
    const int nh = (p.ld + 63) >> 6;
    // 16-byte chunk c of row r at c ^ ((r >> 2) & 3): 16 neighbouring rows cover every bank once
    const int col = ((lane & 3) ^ ((lane >> 4) & 3)) << 4;
    int offA[2], offB[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int r = (wave + 8 * q) * 16 + (lane >> 2);
        offA[q] = r < rowsA ? r * p.ld + col : OOB;
        offB[q] = r < rowsB ? r * p.ld + col : OOB;
    }
    auto issue = [&](int h, unsigned char* st) {
        // (offsets with the top bit set stay beyond every descriptor; stages behind the last one load nothing)
        const int k0 = h * 64, out = k0 + col < p.ld ? 0 : OOB;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsA, (lds_ptr)(st + (wave + 8 * q) * 1024), 16, (offA[q] | out) + k0, 0, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsB, (lds_ptr)(st + Tl::ABYTES + (wave + 8 * q) * 1024), 16, (offB[q] | out) + k0, 0, 0, 0);
        }
    };
    // scales, in even stages: wave 0 A's, wave 1 B's
    const unsigned char* const sbase = wave == 0 ? p.sa + m0 : p.sb + n0;
    const long spitch = wave == 0 ? p.lda_s : p.ldb_s;
    const uint32_t sbytes = (uint32_t)(((wave == 0 ? rowsA : rowsB) + 3) & ~3);
    auto issue_scales = [&](int h, unsigned char* st) {
        if (wave < 2) {
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(sbase + (long)(h >> 1) * spitch), 0, h < nh ? sbytes : 0u, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(st + 2 * Tl::ABYTES + wave * 256), 4, lane * 4, 0, 0, 0);
        }
    };
    const int wm = wave >> 2, wn = wave & 3, group = wave >> 2, sw = (lr >> 2) & 3;
    const int c0 = ((hi * 2) ^ sw) << 4, c1 = ((hi * 2 + 1) ^ sw) << 4;
    f32x16 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    i32x8 x[TM], w[TN];
    int xs[TM], ws[TN];
    auto meet = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    // the two stages behind the next one may be in flight: 4 loads each, and the scales of the even one in their two waves
    auto landed = [&]() {
        if (wave < 2) __builtin_amdgcn_s_waitcnt(loads_left(9));
        else __builtin_amdgcn_s_waitcnt(loads_left(8));
        asm volatile("" ::: "memory");
    };
    auto fetch = [&](auto even, int h, const unsigned char* __restrict__ st, unsigned char* __restrict__ next) {
        if constexpr (decltype(even)::value) {
#pragma unroll
            for (int j = 0; j < TM; ++j) xs[j] = st[2 * Tl::ABYTES + (wm * TM + j) * 32 + lr];
#pragma unroll
            for (int i = 0; i < TN; ++i) ws[i] = st[2 * Tl::ABYTES + 256 + (wn * TN + i) * 32 + lr];
        }
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            const unsigned char* row = st + ((wm * TM + j) * 32 + lr) * 64;
            const int4 u = *reinterpret_cast<const int4*>(row + c0), v = *reinterpret_cast<const int4*>(row + c1);
            x[j] = i32x8{u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
        }
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            const unsigned char* row = st + Tl::ABYTES + ((wn * TN + i) * 32 + lr) * 64;
            const int4 u = *reinterpret_cast<const int4*>(row + c0), v = *reinterpret_cast<const int4*>(row + c1);
            w[i] = i32x8{u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
        }
        issue(h + 3, next);
        if constexpr (!decltype(even)::value) issue_scales(h + 3, next);
    };
    auto half = [&](auto grp, auto even, int h) {
        fetch(even, h, q8_sm + (h & 3) * Tl::STAGE, q8_sm + ((h + 3) & 3) * Tl::STAGE);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if constexpr (decltype(grp)::value) landed();
        meet();
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[i], x[j], acc[i][j], 0, 0, 0, ws[i], 0, xs[j]);
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) asm volatile("" : "+v"(acc[i][j]));   // (here, not behind the next branch)
        if constexpr (!decltype(grp)::value) landed();
        meet();
    };
    auto run = [&](auto grp) {
        for (int h = 0; h < nh; h += 2) {
            half(grp, std::true_type{}, h);
            if (h + 1 < nh) half(grp, std::false_type{}, h + 1);
        }
    };
    issue(0, q8_sm), issue_scales(0, q8_sm);
    issue(1, q8_sm + Tl::STAGE);
    issue(2, q8_sm + 2 * Tl::STAGE), issue_scales(2, q8_sm + 2 * Tl::STAGE);
    landed();
    meet();
    if (group) {
        meet();
        run(std::true_type{});
    } else {
        run(std::false_type{});
        meet();
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (empty loads behind the last stage write LDS as well)
    __syncthreads();
    if (p.out32) mm_store<TM, TN, float>(p, acc, q8_sm + wave * Tl::OUT, m0 + wm * TM * 32, n0 + wn * TN * 32, lane);
    else mm_store<TM, TN, uint16_t>(p, acc, q8_sm + wave * Tl::OUT, m0 + wm * TM * 32, n0 + wn * TN * 32, lane);
}
__global__ __launch_bounds__(256, 2) void q8_mm_128x128(MmParams p) { q8_mm_body<128, 128, 2, 2, 2>(p); }
__global__ __launch_bounds__(256, 2) void q8_mm_128x32(MmParams p) { q8_mm_body<128, 32, 4, 1, 3>(p); }

// The product for short k (K <= 512) and many rows -- every 1x1 convolution of the network: bound by HBM (256 -> 256 at 1/8 resolution: 201 MB
// for 34 GFLOP), so rows are streamed once through persistent blocks that keep their weights in REGISTERS.
//   * a block owns 32 * NT * WN output channels; its waves hold the fragments of all KB blocks of k (NT * KB * 16 VGPRs);
//   * a tile is BM whole rows (32 KB of source).  The next tile's rows are loaded into registers while the current one is multiplied, then
//     become codes in one of two LDS tiles.  SRC 1 / 2: the source is 16-bit and the codes are made here exactly as q8_pack does (16 lanes
//     per block of a row, four DPP steps) -- x is read once, and q8_pack's own pass (read x, write codes, read codes) disappears; SRC 2
//     also stores codes and scales for the backward pass.  SRC 0: the source is packed already;
//   * 16-byte chunk c of LDS row r at c ^ (r & 15) (KB = 1: c ^ ((r >> 1) & 7)): fragment reads of 16 neighbouring rows cover each bank once;
//   * a lane ends up with 4 + 4 consecutive channels of a pixel; v_permlane32_swap joins them to 16-byte stores.
// grid (row blocks, N / (32 NT WN)); the blocks of one row range sit on one XCD (grid.x % 8 == 0) and share its rows through L2.
// 262144 x 256 x 256: packed source 45-50 us (201 MB, 39 at the rate of a copy), 16-bit source 60-63 (269 MB, 52), with codes kept 64-69
// (336 MB, 65).
struct StreamParams {
    const unsigned char* src;             // codes, or 16-bit rows of `ld` elements
    const unsigned char* src_scales;
    unsigned char *codes, *scales;        // SRC 2
    const unsigned char *b, *sb;
    const float* bias;
    void* out;
    int M, K, N, ld, ldc, ldb, ntiles;
    long lds, ldb_s, ldo;
    Act act;
    int out32;
};
MGN_PLAN_RO(StreamParams, MGN_RO(src) MGN_RO(src_scales) MGN_RO(b) MGN_RO(sb) MGN_RO(bias))

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// a lane's accumulators of NT 32-channel tiles: channels n0 + 32 t + 8 q + 4 hi + 0..3 of row m; `bias` in LDS, from channel n0 on.
// VEC: 16-byte stores of 8 channels through `rs` (rows of the tile from its first one on; what lies outside is dropped): no branch, so that
// the number of stores in flight is known where the next tile's loads are waited for.
template <int NT, bool VEC>
__device__ __forceinline__ void stream_store(const StreamParams& p, __amdgpu_buffer_rsrc_t rs, long m0, int r, int n0, int hi, const float* bias, const f32x16 (&acc)[NT]) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float v[16];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float4 b = *reinterpret_cast<const float4*>(bias + t * 32 + 8 * q + 4 * hi);
            v[4 * q] = activate(acc[t][4 * q] + b.x, p.act);
            v[4 * q + 1] = activate(acc[t][4 * q + 1] + b.y, p.act);
            v[4 * q + 2] = activate(acc[t][4 * q + 2] + b.z, p.act);
            v[4 * q + 3] = activate(acc[t][4 * q + 3] + b.w, p.act);
        }
        if (VEC) {
#pragma unroll
            for (int q = 0; q < 4; q += 2) {
                const auto s0 = __builtin_amdgcn_permlane32_swap(mgn_pack2(v[4 * q], v[4 * q + 1]), mgn_pack2(v[4 * q + 4], v[4 * q + 5]), false, false);
                const auto s1 = __builtin_amdgcn_permlane32_swap(mgn_pack2(v[4 * q + 2], v[4 * q + 3]), mgn_pack2(v[4 * q + 6], v[4 * q + 7]), false, false);
                const int n = n0 + t * 32 + 8 * (q + hi);
                const u32x4 w = {(unsigned)s0[0], (unsigned)s1[0], (unsigned)s0[1], (unsigned)s1[1]};
                __builtin_amdgcn_raw_buffer_store_b128(w, rs, n < p.N ? (r * (int)p.ldo + n) * 2 : OOB, 0, 0);
            }
        } else if (m0 + r < p.M) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int n = n0 + t * 32 + 8 * q + 4 * hi + e;
                    if (n >= p.N) continue;
                    if (p.out32) ((float*)p.out)[(m0 + r) * p.ldo + n] = v[4 * q + e];
                    else ((uint16_t*)p.out)[(m0 + r) * p.ldo + n] = (uint16_t)mgn_f2h(v[4 * q + e]);
                }
        }
    }
}

// bytes from the scale of row r0 of the first block to the end of the last block's scales
__device__ __forceinline__ long scale_span(const StreamParams& p, long r0) { return (long)((p.K + BLK - 1) / BLK) * p.lds - r0; }

template <int KB, int WN, int SRC>
struct Stream {
    static constexpr int TH = WN == 8 ? 512 : 256;                  // threads
    static constexpr int BM = 128 / KB * (SRC == 0 ? 2 : 1) * (TH / 256);
    static constexpr int PITCH = KB * BLK, TILE = BM * PITCH, LDS = 2 * (TILE + KB * BM) + 256 * 4;   // two tiles, their scales, the block's bias
    static constexpr int LPU = SRC == 0 ? 8 : 16;                   // lanes per (row, block): 16 bytes of source each
    static constexpr int PASS = BM * KB * LPU / TH;                  // 16-byte loads per thread and tile
    static_assert(PASS == 8, "32 KB of source per 256 threads and tile");
    __device__ static int swz(int r) { return KB == 1 ? (r >> 1) & 7 : r & 15; }
};

template <int KB, int NT, int WN, int SRC, bool VEC>
__device__ __forceinline__ void q8_stream_body(const StreamParams& p) {
    using S = Stream<KB, WN, SRC>;
    extern __shared__ __attribute__((aligned(16))) unsigned char q8_sm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lr = lane & 31, hi = lane >> 5;
    const int n0 = (blockIdx.y * WN + (WN == 1 ? 0 : wave)) * NT * 32;

    // source: unit u = pass * (TH / LPU) + tid / LPU = (row u / KB, block u % KB).  All memory traffic of the loop goes through buffer
    // descriptors of the tile's rows: rows and columns that are not there read as zeros and are not written, without a branch.
    const int ul = tid % S::LPU, u0 = tid / S::LPU, ukb = u0 % KB, urow = u0 / KB;   // (TH / LPU is a multiple of KB)
    const int ucol = ukb * BLK + ul * (SRC == 0 ? 16 : 8);
    constexpr int RSTEP = S::TH / S::LPU / KB;                      // rows per pass
    constexpr int ES = SRC == 0 ? 1 : 2;                            // bytes per source element
    const int soff = ucol < (SRC == 0 ? p.ld : p.K) ? (urow * p.ld + ucol) * ES : OOB;
    const int srow = tid % (S::BM / 4) * 4, skb = tid / (S::BM / 4);   // the four scales this thread moves
    const int qoff = tid < KB * S::BM / 4 && skb * BLK < p.K ? skb * (int)p.lds + srow : OOB;   // (p.lds < 2^31; see rsS)
    u32x4 q[8];
    uint32_t qs = 0;
    auto rows_of = [&](int tile) { const long left = p.M - (long)tile * S::BM; return (int)(left < S::BM ? (left > 0 ? left : 0) : S::BM); };
    auto fetch = [&](int tile) {
        const long r0 = (long)tile * S::BM;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.src + r0 * p.ld * ES), 0, (uint32_t)(rows_of(tile) * p.ld * ES), 0x00020000);
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = __builtin_amdgcn_raw_buffer_load_b128(rs, soff + j * RSTEP * p.ld * ES, 0, 0);
        if (SRC == 0) {
            const __amdgpu_buffer_rsrc_t rsS = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.src_scales + r0), 0, (uint32_t)(tile < p.ntiles ? scale_span(p, r0) : 0), 0x00020000);
            qs = __builtin_amdgcn_raw_buffer_load_b32(rsS, r0 + srow < p.lds ? qoff : OOB, 0, 0);
        }
    };
    auto settle = [&](int tile, int buf) {                           // registers -> LDS tile `buf` [-> packed form in memory]
        unsigned char* st = q8_sm + buf * S::TILE;
        unsigned char* sc = q8_sm + 2 * S::TILE + buf * KB * S::BM;
        const __amdgpu_buffer_rsrc_t rs = SRC == 2 ? __builtin_amdgcn_make_buffer_rsrc(p.codes + (long)tile * S::BM * p.ldc, 0, blockIdx.y == 0 ? (uint32_t)(rows_of(tile) * p.ldc) : 0u, 0x00020000)
                                                   : __builtin_amdgcn_make_buffer_rsrc(p.codes, 0, 0, 0x00020000);
        const int coff = ucol < p.ldc ? urow * p.ldc + ucol : OOB;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = urow + j * RSTEP;
            if (SRC == 0) {
                *reinterpret_cast<u32x4*>(st + r * S::PITCH + (((ukb * 8 + ul) ^ S::swz(r)) << 4)) = q[j];
            } else {
                uint32_t s;
                const uint2 e = quantize8<16>(make_uint4(q[j][0], q[j][1], q[j][2], q[j][3]), s);
                *reinterpret_cast<uint2*>(st + r * S::PITCH + (((ukb * 8 + (ul >> 1)) ^ S::swz(r)) << 4) + (ul & 1) * 8) = e;
                if (ul == 0) sc[ukb * S::BM + r] = (unsigned char)s;
                if (SRC == 2) __builtin_amdgcn_raw_buffer_store_b64(u32x2{e.x, e.y}, rs, coff + j * RSTEP * p.ldc, 0, 0);
            }
        }
        if (SRC == 0 && tid < KB * S::BM / 4) *reinterpret_cast<uint32_t*>(sc + tid * 4) = qs;
    };

    int tile = blockIdx.x, buf = 0;
    if (tile >= p.ntiles) return;
    fetch(tile);

    // the wave's weights
    i32x8 w[NT][KB * 2];
    int ws[NT][KB];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int n = n0 + t * 32 + lr;
        const unsigned char* row = p.b + (long)(n < p.N ? n : 0) * p.ldb;
#pragma unroll
        for (int kk = 0; kk < KB * 2; ++kk) {
            int4 u[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int c = kk * 64 + hi * 32 + h * 16;
                u[h] = (n < p.N && c < p.ldb) ? *reinterpret_cast<const int4*>(row + c) : make_int4(0, 0, 0, 0);
            }
            w[t][kk] = i32x8{u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w};
        }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) ws[t][kb] = (n < p.N && kb * BLK < p.K) ? p.sb[(long)kb * p.ldb_s + n] : 0;
    }

    float* bias = reinterpret_cast<float*>(q8_sm + 2 * (S::TILE + KB * S::BM));
    if (tid < NT * WN * 32) {
        const int n = blockIdx.y * NT * WN * 32 + tid;
        bias[tid] = (p.bias && n < p.N) ? p.bias[n] : 0.f;
    }

    // (the weights have arrived before the loop: waited for at their first use inside it, every round would wait for the stores before it too)
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
    settle(tile, 0);
    for (;;) {
        fetch(tile + gridDim.x);          // (behind the last tile there are no rows: nothing is loaded, and the loop keeps one shape)
        __syncthreads();                  // this tile is in LDS; the tile before it, which settle() below overwrites, has been read
        const unsigned char* st = q8_sm + buf * S::TILE;
        const unsigned char* sc = q8_sm + 2 * S::TILE + buf * KB * S::BM;
        const long m0 = (long)tile * S::BM;
        if (SRC == 2) {
            const __amdgpu_buffer_rsrc_t rsS = __builtin_amdgcn_make_buffer_rsrc(p.scales + m0, 0, blockIdx.y == 0 ? (uint32_t)scale_span(p, m0) : 0u, 0x00020000);
            const uint32_t v = *reinterpret_cast<const uint32_t*>(sc + (tid < KB * S::BM / 4 ? tid * 4 : 0));
            __builtin_amdgcn_raw_buffer_store_b32(v, rsS, m0 + srow < p.lds ? qoff : OOB, 0, 0);
        }
        const __amdgpu_buffer_rsrc_t rsO = __builtin_amdgcn_make_buffer_rsrc((uint16_t*)p.out + m0 * p.ldo, 0, VEC ? (uint32_t)(rows_of(tile) * (int)p.ldo * 2) : 0u, 0x00020000);
#pragma unroll
        for (int gi = 0; gi < S::BM / 32; gi += WN == 1 ? 4 : 1) {
            const int g = gi + (WN == 1 ? wave : 0);
            if (WN == 1 && S::BM < 128 && g >= S::BM / 32) break;
            const int r = g * 32 + lr;
            const unsigned char* row = st + r * S::PITCH;
            const int sw = S::swz(r);
            f32x16 acc[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[t][e] = 0.f;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const int xs = sc[kb * S::BM + r];
#pragma unroll
                for (int kk = 2 * kb; kk < 2 * kb + 2; ++kk) {
                    const int4 u = *reinterpret_cast<const int4*>(row + (((kk * 4 + hi * 2) ^ sw) << 4)), v = *reinterpret_cast<const int4*>(row + (((kk * 4 + hi * 2 + 1) ^ sw) << 4));
                    const i32x8 x = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int t = 0; t < NT; ++t) acc[t] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[t][kk], x, acc[t], 0, 0, 0, ws[t][kb], 0, xs);
                }
            }
            stream_store<NT, VEC>(p, rsO, m0, r, n0, hi, bias + (WN == 1 ? 0 : wave) * NT * 32, acc);
        }
        tile += gridDim.x;
        if (tile >= p.ntiles) break;
        buf ^= 1;
        settle(tile, buf);                // (loads and the stores behind them lie in one piece of straight code: only the loads are waited for)
    }
}

#define Q8_STREAM(NAME, KB, NT, WN, VEC) \
    __global__ __launch_bounds__(WN == 8 ? 512 : 256, 2) void q8_stream_##NAME##_packed(StreamParams p) { q8_stream_body<KB, NT, WN, 0, VEC>(p); } \
    __global__ __launch_bounds__(WN == 8 ? 512 : 256, 2) void q8_stream_##NAME##_h16(StreamParams p) { q8_stream_body<KB, NT, WN, 1, VEC>(p); } \
    __global__ __launch_bounds__(WN == 8 ? 512 : 256, 2) void q8_stream_##NAME##_keep(StreamParams p) { q8_stream_body<KB, NT, WN, 2, VEC>(p); }
Q8_STREAM(1_any, 1, 1, 1, false) Q8_STREAM(2_any, 2, 1, 1, false) Q8_STREAM(4_any, 4, 1, 1, false)      // N <= 32: any N and result type
Q8_STREAM(1_32, 1, 1, 1, true) Q8_STREAM(2_32, 2, 1, 1, true) Q8_STREAM(4_32, 4, 1, 1, true)
Q8_STREAM(1_128, 1, 1, 4, true) Q8_STREAM(2_128, 2, 1, 4, true) Q8_STREAM(4_128, 4, 1, 4, true)
Q8_STREAM(1_256, 1, 2, 4, true) Q8_STREAM(2_256, 2, 2, 4, true) Q8_STREAM(4_256, 4, 1, 8, true)         // (<4, 2, 4>: 128 registers for the weights alone, spills)
#undef Q8_STREAM

// Few tiles: a block per 32 x 32 outputs, the blocks of k dealt to its four waves, each with LDS stages of its own (rows travel by LDS-DMA,
// the next block's while one is multiplied; no barrier), the four partial tiles added through LDS in wave order.  1 x 4096 x 4096: 5.7 us
// (16.8 MB of weights, 3.3 at the rate of a copy), 128 x 4096 x 4096 9.2.  Rows loaded straight into registers as the MFMA wants them, 16
// bytes of another row in every lane, cost the address unit a cycle a lane: 8.6 and 19 us.  More waves for k do not help (8: 7.6 and 20).
constexpr int SMALL_STAGE = 64 * BLK;     // 32 rows of A, 32 of B
__global__ __launch_bounds__(TPB) void q8_mm_small(MmParams p) {
    extern __shared__ __attribute__((aligned(16))) unsigned char q8_sm[];   // [stages][4 waves][SMALL_STAGE], later [4][32][33] floats
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 31, hi = lane >> 5;
    const int n0 = blockIdx.x * 32;
    const long m0 = (long)blockIdx.y * 32;
    const int rowsA = (int)(p.M - m0 < 32 ? p.M - m0 : 32), rowsB = p.N - n0 < 32 ? p.N - n0 : 32;
    const __amdgpu_buffer_rsrc_t rsA = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.a + m0 * p.ld), 0, (uint32_t)(rowsA * p.ld), 0x00020000);
    const __amdgpu_buffer_rsrc_t rsB = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.b + (long)n0 * p.ld), 0, (uint32_t)(rowsB * p.ld), 0x00020000);
    int off[4], col[2];                   // 16-byte chunk c of row r at c ^ ((r >> 1) & 7); a piece has 8 rows
#pragma unroll
    for (int q = 0; q < 4; ++q) off[q] = (q * 8 + (lane >> 3)) * p.ld;
#pragma unroll
    for (int q = 0; q < 2; ++q) col[q] = ((lane & 7) ^ ((q * 4 + (lane >> 4)) & 7)) << 4;
    // rows behind the last one lie behind the descriptor; columns behind the row's end are sent there
    auto issue = [&](int kb, unsigned char* st) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int c = kb * BLK + col[q & 1], at = c < p.ld ? off[q] + c : OOB;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsA, (lds_ptr)(st + q * 1024), 16, at, 0, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsB, (lds_ptr)(st + (4 + q) * 1024), 16, at, 0, 0, 0);
        }
    };
    // (rows that are not there take the first row's scale: their codes are zeros, and no select waits for a scale that is still on its way)
    const unsigned char *as = p.sa + m0 + (lr < rowsA ? lr : 0), *bs = p.sb + n0 + (lr < rowsB ? lr : 0);
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
    const int sw = (lr >> 1) & 7;
    auto multiply = [&](const unsigned char* __restrict__ st, int xs, int ws) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const int c0 = ((kk * 4 + hi * 2) ^ sw) << 4, c1 = ((kk * 4 + hi * 2 + 1) ^ sw) << 4;
            const int4 u = *reinterpret_cast<const int4*>(st + lr * BLK + c0), v = *reinterpret_cast<const int4*>(st + lr * BLK + c1);
            const int4 g = *reinterpret_cast<const int4*>(st + (32 + lr) * BLK + c0), h = *reinterpret_cast<const int4*>(st + (32 + lr) * BLK + c1);
            acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(i32x8{g.x, g.y, g.z, g.w, h.x, h.y, h.z, h.w}, i32x8{u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w},
                                                                  acc, 0, 0, 0, ws, 0, xs);
        }
    };
    unsigned char* const mine = q8_sm + wave * SMALL_STAGE;
    int at = 0, xs = 0, ws = 0;
    if (wave < p.nb) {
        xs = as[(long)wave * p.lda_s], ws = bs[(long)wave * p.ldb_s];
        issue(wave, mine);
    }
    for (int kb = wave; kb < p.nb; kb += 4) {
        const unsigned char* st = mine + at * 4 * SMALL_STAGE;
        int xn = 0, wn = 0;
        if (kb + 4 < p.nb) {
            at ^= 1;
            xn = as[(long)(kb + 4) * p.lda_s], wn = bs[(long)(kb + 4) * p.ldb_s];
            __builtin_amdgcn_sched_barrier(0);
            issue(kb + 4, mine + at * 4 * SMALL_STAGE);
            asm volatile("s_waitcnt vmcnt(10)" ::: "memory");   // (10: what was issued just now)
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        multiply(st, xs, ws);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // read: the stage may be loaded again
        xs = xn, ws = wn;
    }
    __syncthreads();
    float(*part)[32][33] = reinterpret_cast<float(*)[32][33]>(q8_sm);
#pragma unroll
    for (int e = 0; e < 16; ++e) part[wave][lr][8 * (e >> 2) + 4 * hi + (e & 3)] = acc[e];
    __syncthreads();
    const int r = threadIdx.x >> 3, n = (threadIdx.x & 7) * 4;
    if (m0 + r < p.M && n0 + n < p.N) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (part[0][r][n + e] + part[1][r][n + e]) + (part[2][r][n + e] + part[3][r][n + e]);
        mm_emit(p, m0 + r, n0 + n, v);
    }
}

// ------------------------------------------------------------------------------------------------------
// dW[n][k] = sum_m dy[m][n] x^[m][k], db[n] = sum_m dy[m][n]: dy in 16 bits, x^ from its codes.
//   A block computes a 128 x 128 tile over one of `splits` row ranges.  dy rows go to LDS by LDS-DMA (three stages), codes through
//   registers, where a value and its scale become the exact 16-bit x^ (one instruction for two); both tiles are read back with the
//   transposing LDS reads, since the summed index is the row.  Loads run two steps ahead (80 KB of LDS: two blocks a CU).
//   v_mfma_f32_32x32x16, fp32 accumulation; the splits' tiles are added by q8_wgrad_reduce in order.
//   262144 x 256 x 256: 54-59 us, 3.6 TB/s (201 MB, each byte read once: 39 us at the rate of a copy, 41 at the 4.9 TB/s that a pass of this
//   library which only reads reaches on 537 MB), and 9 us for the reduction of 128 partial results (34 MB).  Neither memory nor matrix cores
//   (37 % busy) are full; a quarter of the LDS cycles are conflicts.
//   db: the same dy fragments times a column of ones, in the blocks of the first k tile.
// ------------------------------------------------------------------------------------------------------
struct WgradParams8 {
    const uint16_t* dy;
    const unsigned char *codes, *scales;
    float* part;                          // [splits][N * K + N, padded to 4]
    int M, N, K, ldy, ldc;
    long lds;
    int rows_per_split, splits, ntn, ntk;
};
MGN_PLAN_RO(WgradParams8, MGN_RO(dy) MGN_RO(codes) MGN_RO(scales))

constexpr int WG_ROWS = 64;               // rows per step
constexpr int WG_TILE = WG_ROWS * 256;    // bytes of a [64][128] 16-bit tile
constexpr int WG_LDS = 5 * WG_TILE;       // dy x 3, x^ x 2

__device__ __forceinline__ uint32_t decode2(uint32_t c, float s, int word) {
#ifdef MGN_F16
    return word ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, s, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, s, false));
#else
    return word ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, s, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, s, false));
#endif
}

__global__ __launch_bounds__(TPB, 2) void q8_wgrad(WgradParams8 p) {
    extern __shared__ __attribute__((aligned(16))) unsigned char q8_sm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 1, wn = wave & 1;
    // the tiles of one row range share an XCD (its rows are then read from HBM once)
    const int tiles = p.ntn * p.ntk, id = (int)block_id(), local = id >> 3;
    const int z = (local / tiles) * 8 + (id & 7), t = local % tiles;
    if (z >= p.splits) return;
    const int tn = t % p.ntn, tk = t / p.ntn;
    const long mb = (long)z * p.rows_per_split;
    const int rows = (int)(p.M - mb < p.rows_per_split ? p.M - mb : p.rows_per_split);   // >= 1 by the host's choice of splits
    const int steps = (rows + WG_ROWS - 1) / WG_ROWS;
    const __amdgpu_buffer_rsrc_t rsY = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(p.dy + mb * p.ldy), 0, (uint32_t)(rows * p.ldy * 2), 0x00020000);
    auto swz = [](int r) { return (r & 3) << 2; };
    int yo[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int r = (wave + 4 * q) * 4 + (lane >> 4), ch = (lane & 15) ^ swz(r);
        yo[q] = tn * 128 + ch * 8 < p.ldy ? r * p.ldy * 2 + (tn * 128 + ch * 8) * 2 : OOB;
    }
    auto issue = [&](int ks, unsigned char* st) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int r = ks * WG_ROWS + (wave + 4 * q) * 4 + (lane >> 4);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsY, (lds_ptr)(st + (wave + 4 * q) * 1024), 16,
                                                     (r < rows && yo[q] != OOB) ? yo[q] + ks * WG_ROWS * p.ldy * 2 : OOB, 0, 0, 0);
        }
    };
    // codes: thread = (rows tid / 8 and 32 further, 16 columns); the two 16-byte halves of its x^ leave in an order that alternates with the row,
    // so that the 16 lanes of two neighbouring rows write every bank once
    const int cr = tid >> 3, cc = (tid & 7) * 16, kcol = tk * BLK + cc, odd = cr & 1;
    const __amdgpu_buffer_rsrc_t rsX = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.codes + mb * p.ldc), 0, (uint32_t)(rows * p.ldc), 0x00020000);
    const __amdgpu_buffer_rsrc_t rsC = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p.scales + (long)tk * p.lds + mb), 0, (uint32_t)rows, 0x00020000);
    const int xo = kcol < p.ldc ? cr * p.ldc + kcol : OOB;
    struct Fetched { u32x4 c[2]; uint32_t s[2]; };
    auto fetch = [&](int ks) {
        Fetched f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f.c[h] = __builtin_amdgcn_raw_buffer_load_b128(rsX, xo + (ks * WG_ROWS + 32 * h) * p.ldc, 0, 0);
            f.s[h] = __builtin_amdgcn_raw_buffer_load_b8(rsC, cr + ks * WG_ROWS + 32 * h, 0, 0);
        }
        return f;
    };
    auto spread = [&](const Fetched& f, unsigned char* __restrict__ tile) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            unsigned char* b = tile + (cr + 32 * h) * 256;
            const float s = pow2(f.s[h]);
            const u32x4 c = f.c[h];
            const uint32_t a0 = odd ? c[2] : c[0], a1 = odd ? c[3] : c[1], b0 = odd ? c[0] : c[2], b1 = odd ? c[1] : c[3];
            const int ch = (cc >> 3) + odd;
            *reinterpret_cast<uint4*>(b + ((ch ^ swz(cr)) << 4)) = make_uint4(decode2(a0, s, 0), decode2(a0, s, 1), decode2(a1, s, 0), decode2(a1, s, 1));
            *reinterpret_cast<uint4*>(b + (((ch ^ 1) ^ swz(cr)) << 4)) = make_uint4(decode2(b0, s, 0), decode2(b0, s, 1), decode2(b1, s, 0), decode2(b1, s, 1));
        }
    };
    // transposed fragments: lane group g = lane >> 4 reads rows 8 * (g >> 1) + (i >> 2) [+ 4], columns 16 * (g & 1) + 4 * (i & 3)
    const int g = lane >> 4, i4 = lane & 15, prow = 8 * (g >> 1) + (i4 >> 2);
    int fa[2], fb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int ca = wm * 64 + i * 32 + (g & 1) * 16 + 4 * (i4 & 3), cb = wn * 64 + i * 32 + (g & 1) * 16 + 4 * (i4 & 3);
        fa[i] = prow * 256 + (((ca >> 3) ^ swz(prow)) << 4) + (ca & 7) * 2;
        fb[i] = prow * 256 + (((cb >> 3) ^ swz(prow)) << 4) + (cb & 7) * 2;
    }
    typedef __attribute__((address_space(3))) s16x4* lp;
    auto frag = [&](const unsigned char* q) {
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q + 4 * 256));
        return __builtin_bit_cast(h16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    f32x16 acc[2][2], accb[2];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        acc[0][0][e] = acc[0][1][e] = acc[1][0][e] = acc[1][1][e] = 0.f;
        accb[0][e] = accb[1][e] = 0.f;
    }
    h16x8 ones;
#pragma unroll
    for (int e = 0; e < 8; ++e) ones[e] = (decltype(ones[0] + ones[0]))1.0f;
    const bool with_db = tk == 0 && wn == 0;

    // In flight at the top of step ks: the loads of steps ks and ks + 1, 4 LDS-DMA and 4 register loads each, in this order.
    // The 16 rows of the next MFMAs are read while the current ones run; `db` (with the ones column) is a type, so that no branch parts the step.
    // (restrict pointers, waits outside: see q8_mm_body)
    auto multiply = [&](auto db, int ks, const unsigned char* __restrict__ sa, const unsigned char* __restrict__ sb, unsigned char* __restrict__ next, Fetched& f) {
        h16x8 a[2][2], b[2][2];
        auto read = [&](int kk) {         // the swizzle depends on row bits 0..1: unchanged by + 16 rows
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[kk & 1][i] = frag(sa + fa[i] + kk * 16 * 256);
                b[kk & 1][i] = frag(sb + fb[i] + kk * 16 * 256);
            }
        };
        read(0);
        issue(ks + 2, next);              // (rows behind the range load nothing)
        f = fetch(ks + 2);
#pragma unroll
        for (int kk = 0; kk < WG_ROWS / 16; ++kk) {
            if (kk + 1 < WG_ROWS / 16) read(kk + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = MGN_MFMA_32x32x16(a[kk & 1][i], b[kk & 1][j], acc[i][j]);
            if constexpr (decltype(db)::value) {
                accb[0] = MGN_MFMA_32x32x16(a[kk & 1][0], ones, accb[0]);
                accb[1] = MGN_MFMA_32x32x16(a[kk & 1][1], ones, accb[1]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto run = [&](auto db) {
        auto step = [&](int ks, int a_buf, Fetched& f) {
            asm volatile("s_waitcnt vmcnt(8)" ::: "memory");   // step ks has landed
            unsigned char* xb = q8_sm + (3 + (ks & 1)) * WG_TILE;
            spread(f, xb);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();     // ... for everyone; step ks - 1 has been read
            multiply(db, ks, q8_sm + a_buf * WG_TILE, xb, q8_sm + (a_buf == 0 ? 2 : a_buf - 1) * WG_TILE, f);
        };
        issue(0, q8_sm);
        Fetched f0 = fetch(0);
        __builtin_amdgcn_sched_barrier(0);    // (in this order: the loop's waits count on it)
        issue(1, q8_sm + WG_TILE);
        __builtin_amdgcn_sched_barrier(0);
        Fetched f1 = fetch(1);
        __builtin_amdgcn_sched_barrier(0);
        int a_buf = 0;
        for (int ks = 0; ks < steps; ks += 2) {   // (an odd last step multiplies rows of zeros)
            step(ks, a_buf, f0);
            a_buf = a_buf == 2 ? 0 : a_buf + 1;
            step(ks + 1, a_buf, f1);
            a_buf = a_buf == 2 ? 0 : a_buf + 1;
        }
    };
    if (with_db) run(std::true_type{}); else run(std::false_type{});
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no LDS-DMA outlives the block
    const long wsize = ((long)p.N * p.K + p.N + 3) & ~3L;
    float* out = p.part + (long)z * wsize;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int n = tn * 128 + wm * 64 + i * 32 + (e & 3) + 8 * (e >> 2) + 4 * (lane >> 5);
            if (n >= p.N) continue;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int k = tk * BLK + wn * 64 + j * 32 + (lane & 31);
                if (k < p.K) out[(long)n * p.K + k] = acc[i][j][e];
            }
            if (with_db && (lane & 31) == 0) out[(long)p.N * p.K + n] = accb[i][e];
        }
}

// dw | db = the splits' partial results added in a fixed order: 16 waves take every 16th split of 256 neighbouring sums (1 KB a wave and
// split, up to 8 splits in flight), joined in wave order
__global__ __launch_bounds__(1024) void q8_wgrad_reduce(const float* __restrict__ part, int splits, long total, long nk, float* __restrict__ dw,
                                                        float* __restrict__ db) {
    __shared__ float4 sh[16][64];
    const int lane = threadIdx.x & 63, g = threadIdx.x >> 6;
    const long stride = (total + 3) & ~3L, i = (block_id() * 64 + lane) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < stride) {
        const float* src = part + i;
        int z = g;
        for (; z + 7 * 16 < splits; z += 8 * 16) {
            float4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const float4*>(src + (long)(z + 16 * k) * stride);
#pragma unroll
            for (int k = 0; k < 8; ++k) { s.x += v[k].x; s.y += v[k].y; s.z += v[k].z; s.w += v[k].w; }
        }
        for (; z < splits; z += 16) {
            const float4 v = *reinterpret_cast<const float4*>(src + (long)z * stride);
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
    }
    sh[g][lane] = s;
    __syncthreads();
    if (g != 0) return;
    for (int k = 1; k < 16; ++k) { const float4 v = sh[k][lane]; s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w; }
    const float r[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (i + e < nk) dw[i + e] = r[e];
        else if (db && i + e < total) db[i + e - nk] = r[e];
    }
}

// dy rows of N 16-bit values -> rows of ld (a multiple of 8) with zeros behind: what the 16-byte loads of the two gradients want
__global__ __launch_bounds__(TPB) void q8_pad_rows(const uint16_t* __restrict__ src, long M, int N, int ld, uint4* __restrict__ dst) {
    const int per = ld / 8;
    const long i = block_id() * TPB + threadIdx.x;
    if (i >= M * per) return;
    const long r = i / per;
    const int c = (int)(i - r * per) * 8;
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t lo = c + 2 * k < N ? src[r * N + c + 2 * k] : 0, hi = c + 2 * k + 1 < N ? src[r * N + c + 2 * k + 1] : 0;
        w[k] = lo | (hi << 16);
    }
    dst[i] = make_uint4(w[0], w[1], w[2], w[3]);
}

// ------------------------------------------------------------------------------------------------------
// block tail y = relu(norm(x) + shortcut) whose backward pass reads x^ instead of x.  Thread mapping of the four kernels: blockIdx.y = a
// block of 128 channels, LPB lanes (8 channels each) per row -- a thread's channels never change, so their coefficients stay in
// registers.  All are bound by HBM: 1048576 x 64 bf16, 134 MB a tensor: statistics 35 us (134 MB), forward 80 (478 MB, 6.0 TB/s), backward
// sums 63 (344 MB, 5.4 TB/s), dx 56 (336 MB, 6.0 TB/s); joining the partial sums 5 and 5 us, two launches of latency.
// The statistics read 134 MB at 3.9 TB/s with 512 row blocks, at 3.4 with 1024 or 2048; iabn.hip's statistics pass reads 134 MB at 4.0 and 537 MB
// at 4.9.
// ------------------------------------------------------------------------------------------------------
constexpr int TAIL_BLOCKS = 512;          // row blocks of the two reductions (= partial rows)

// column sums of two quantities over this block's rows -> part[blockIdx.x][C][2]; NL rows in flight per thread
template <int LPB>
__device__ __forceinline__ void tail_flush(const float (&a)[8], const float (&b)[8], int C, float* part) {
    __shared__ float sh[TPB / LPB][LPB * 16 + 1];
    const int l = threadIdx.x % LPB, ty = threadIdx.x / LPB;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        sh[ty][(l * 8 + k) * 2] = a[k];
        sh[ty][(l * 8 + k) * 2 + 1] = b[k];
    }
    __syncthreads();
    const int base = blockIdx.y * BLK * 2;
    for (int i = threadIdx.x; i < LPB * 16; i += TPB) {
        float s = 0.f;
        for (int y = 0; y < TPB / LPB; ++y) s += sh[y][i];
        if (base + i < C * 2) part[(long)blockIdx.x * C * 2 + base + i] = s;
    }
}

// sums of (x - shift) and their squares; shift = the mean of 4 TPB / LPB (64 .. 256) rows spread over the map, the same in every block.  The
// variance is a difference of two sums, off by some 2^-24 (mean - shift)^2: the mean of a sample is near the mean, also where one row alone (the
// first, say) would be an outlier, as in channels that are zero almost everywhere.
template <int LPB>
__global__ __launch_bounds__(TPB) void q8_tail_stats(const uint16_t* __restrict__ x, int M, int C, float* __restrict__ part, float* __restrict__ shift) {
    constexpr int RPB = TPB / LPB, NS = 4 * RPB;
    __shared__ float sample[RPB][LPB * 8 + 4];
    const int l = threadIdx.x % LPB, ty = threadIdx.x / LPB, c0 = blockIdx.y * BLK + l * 8;
    const bool on = c0 < C;
    float s[8], a[8], b[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) s[k] = a[k] = b[k] = 0.f;
    if (on) {
        uint4 q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = *reinterpret_cast<const uint4*>(x + (long)(ty + j * RPB) * M / NS * C + c0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float v[8];
            unpack8(q[j], v);
#pragma unroll
            for (int k = 0; k < 8; ++k) s[k] = fmaf(v[k], 1.f / NS, s[k]);   // (scaled before it is added: no overflow)
        }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) sample[ty][l * 8 + k] = s[k];
    __syncthreads();
    if (threadIdx.x < LPB * 8) {
        float m = 0.f;
        for (int y = 0; y < RPB; ++y) m += sample[y][threadIdx.x];
        sample[0][threadIdx.x] = m;       // (its column is this thread's alone)
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; ++k) s[k] = sample[0][l * 8 + k];
    const int stride = gridDim.x * (TPB / LPB);
    auto add = [&](const uint4& q) {
        float v[8];
        unpack8(q, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) { const float d = v[k] - s[k]; a[k] += d; b[k] = fmaf(d, d, b[k]); }
    };
    if (on) {
        long r = (long)blockIdx.x * (TPB / LPB) + threadIdx.x / LPB;
        for (; r + 7L * stride < M; r += 8L * stride) {
            uint4 q[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = *reinterpret_cast<const uint4*>(x + (r + (long)j * stride) * C + c0);
#pragma unroll
            for (int j = 0; j < 8; ++j) add(q[j]);
        }
        for (; r < M; r += stride) add(*reinterpret_cast<const uint4*>(x + r * C + c0));
        if (blockIdx.x == 0 && threadIdx.x < LPB) {
#pragma unroll
            for (int k = 0; k < 8; ++k) shift[c0 + k] = s[k];
        }
    }
    tail_flush<LPB>(a, b, C, part);
}

// y = relu(scale * x + offset + shortcut); codes and scales of x; the mask y > 0, one byte per 8 outputs.  8 rows per lane group.
// KEEP false (inference): y alone.
template <int LPB, bool KEEP>
__global__ __launch_bounds__(TPB) void q8_tail_fwd(const uint16_t* __restrict__ x, const uint16_t* __restrict__ shortcut, const float* __restrict__ scale,
                                                   const float* __restrict__ offset, int M, int C, int ldc, long lds, uint16_t* __restrict__ y,
                                                   unsigned char* __restrict__ codes, unsigned char* __restrict__ scales, unsigned char* __restrict__ bits) {
    const int l = threadIdx.x % LPB, c0 = blockIdx.y * BLK + l * 8;
    const long r0l = ((long)blockIdx.x * (TPB / LPB) + threadIdx.x / LPB) * RPG;
    if (r0l >= M) return;
    const int r0 = (int)r0l;
    const bool on = c0 < C;
    uint4 q[RPG], t[RPG];
#pragma unroll
    for (int j = 0; j < RPG; ++j) {
        const bool in = on && r0 + j < M;
        const long o = (long)(r0 + j) * C + c0;
        q[j] = in ? *reinterpret_cast<const uint4*>(x + o) : make_uint4(0, 0, 0, 0);
        t[j] = in ? *reinterpret_cast<const uint4*>(shortcut + o) : make_uint4(0, 0, 0, 0);
    }
    float sc[8], of[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        sc[k] = on ? scale[c0 + k] : 0.f;
        const float o = on ? offset[c0 + k] : 0.f;
        // (an infinity in a channel makes its mean, and this offset, infinite: the channel is NaN, not the zeros that the ReLU of -inf is)
        of[k] = (__float_as_uint(o) & 0x7f800000u) == 0x7f800000u ? __uint_as_float(0x7fc00000u) : o;
    }
    uint32_t sb[RPG];
#pragma unroll
    for (int j = 0; j < RPG; ++j) {
        float v[8], w[8];
        unpack8(q[j], v);
        unpack8(t[j], w);
        uint2 e = make_uint2(0, 0);
        sb[j] = 0;
        if (KEEP) e = quantize8<LPB>(q[j], sb[j]);
        if (r0 + j >= M) continue;
        const long o = (long)(r0 + j) * C + c0;
        if (KEEP && c0 < ldc) *reinterpret_cast<uint2*>(codes + (long)(r0 + j) * ldc + c0) = e;
        if (!on) continue;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float z = fmaf(v[k], sc[k], of[k]) + w[k];
            v[k] = z < 0.f ? 0.f : z;     // (NaN stays)
        }
        const uint4 r = pack8(v);
        *reinterpret_cast<uint4*>(y + o) = r;
        if (!KEEP) continue;
        const uint32_t u[4] = {r.x, r.y, r.z, r.w};
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) m |= (((u[k] & 0x7fffu) != 0u ? 1u : 0u) | ((u[k] & 0x7fff0000u) != 0u ? 2u : 0u)) << (2 * k);
        bits[o >> 3] = (unsigned char)m;
    }
    if (KEEP && l == 0)
        *reinterpret_cast<uint2*>(scales + blockIdx.y * lds + r0) =
            make_uint2(sb[0] | (sb[1] << 8) | (sb[2] << 16) | (sb[3] << 24), sb[4] | (sb[5] << 8) | (sb[6] << 16) | (sb[7] << 24));
}

__device__ __forceinline__ uint32_t mask2(uint32_t e) { return ((e & 1u) * 0xffffu) | (((e >> 1) & 1u) * 0xffff0000u); }

// dz = g * mask, written (the shortcut's gradient) and reduced: sum dz, sum dz * (x^ - mean)
template <int LPB>
__global__ __launch_bounds__(TPB) void q8_tail_bwd_reduce(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                          const uint16_t* __restrict__ g, const unsigned char* __restrict__ bits,
                                                          const float* __restrict__ mean, int M, int C, int ldc, long lds, uint16_t* __restrict__ dz,
                                                          float* __restrict__ part) {
    const int l = threadIdx.x % LPB, c0 = blockIdx.y * BLK + l * 8;
    const bool on = c0 < C;
    float mu[8], a[8], b[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) { mu[k] = on ? mean[c0 + k] : 0.f; a[k] = b[k] = 0.f; }
    const int stride = gridDim.x * (TPB / LPB);
    const unsigned char* srow = scales + blockIdx.y * lds;
    auto one = [&](long r, const uint2& c, uint32_t s, uint4 q, uint32_t e) {
        q.x &= mask2(e); q.y &= mask2(e >> 2); q.z &= mask2(e >> 4); q.w &= mask2(e >> 6);
        *reinterpret_cast<uint4*>(dz + r * C + c0) = q;
        float v[8], w[8];
        decode8(c, pow2(s), v);
        unpack8(q, w);
#pragma unroll
        for (int k = 0; k < 8; ++k) { a[k] += w[k]; b[k] = fmaf(w[k], v[k] - mu[k], b[k]); }
    };
    if (on) {
        long r = (long)blockIdx.x * (TPB / LPB) + threadIdx.x / LPB;
        for (; r + 3L * stride < M; r += 4L * stride) {
            uint2 c[4];
            uint4 q[4];
            uint32_t s[4], e[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const long rr = r + (long)j * stride;
                c[j] = *reinterpret_cast<const uint2*>(codes + rr * ldc + c0);
                q[j] = *reinterpret_cast<const uint4*>(g + rr * C + c0);
                s[j] = srow[rr];
                e[j] = bits[(rr * C + c0) >> 3];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) one(r + (long)j * stride, c[j], s[j], q[j], e[j]);
        }
        for (; r < M; r += stride)
            one(r, *reinterpret_cast<const uint2*>(codes + r * ldc + c0), srow[r], *reinterpret_cast<const uint4*>(g + r * C + c0), bits[(r * C + c0) >> 3]);
    }
    tail_flush<LPB>(a, b, C, part);
}

#ifndef MGN_F16
// partial sums -> sums[2][C] = {sum dz, sum dz * x_hat}, dwb[2][C] = {sign(weight) * sums[1], sums[0]}; fixed order, 64-bit
__global__ __launch_bounds__(TPB) void q8_tail_sums(const float* __restrict__ part, int rows, int C, const float* __restrict__ rstd,
                                                    const float* __restrict__ weight, float* __restrict__ sums, float* __restrict__ dwb) {
    __shared__ double sh[TPB / 8][8];
    const int c0 = blockIdx.x * 4, col = threadIdx.x & 7, rg = threadIdx.x >> 3;
    double s = 0.0;
    const float* p = part + (long)c0 * 2 + col;
    int r = rg;
    for (; r + 15 * (TPB / 8) < rows; r += 16 * (TPB / 8)) {   // (16 loads in flight: 512 rows 7.0 -> 4.8 us)
        float v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = p[(long)(r + k * (TPB / 8)) * C * 2];
#pragma unroll
        for (int k = 0; k < 16; ++k) s += (double)v[k];
    }
    for (; r < rows; r += TPB / 8) s += (double)p[(long)r * C * 2];
    sh[rg][col] = s;
    __syncthreads();
    if (threadIdx.x < 4) {
        double t1 = 0.0, t2 = 0.0;
        for (int k = 0; k < TPB / 8; ++k) { t1 += sh[k][2 * threadIdx.x]; t2 += sh[k][2 * threadIdx.x + 1]; }
        const int c = c0 + threadIdx.x;
        const float s1 = (float)t1, s2 = (float)(t2 * (double)rstd[c]), w = weight[c];
        sums[c] = s1;
        sums[C + c] = s2;
        dwb[c] = s2 * (float)((w > 0.f) - (w < 0.f));
        dwb[C + c] = s1;
    }
}
#endif

// dx = gain * rstd * (dz - sums[0] / n - x_hat * sums[1] / n),  x_hat = (x^ - mean) * rstd,  gain = |weight| + eps
template <int LPB>
__global__ __launch_bounds__(TPB) void q8_tail_bwd_apply(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                         const uint16_t* __restrict__ dz, const float* __restrict__ weight,
                                                         const float* __restrict__ mean, const float* __restrict__ rstd, const float* __restrict__ sums,
                                                         float inv_n, float eps, int M, int C, int ldc, long lds, uint16_t* __restrict__ dx) {
    const int l = threadIdx.x % LPB, c0 = blockIdx.y * BLK + l * 8;
    const long r0l = ((long)blockIdx.x * (TPB / LPB) + threadIdx.x / LPB) * RPG;
    if (r0l >= M || c0 >= C) return;
    const int r0 = (int)r0l;
    uint2 c[RPG];
    uint4 q[RPG];
    const uint2 sb = *reinterpret_cast<const uint2*>(scales + blockIdx.y * lds + r0);
#pragma unroll
    for (int j = 0; j < RPG; ++j) {
        const bool in = r0 + j < M;
        c[j] = in ? *reinterpret_cast<const uint2*>(codes + (long)(r0 + j) * ldc + c0) : make_uint2(0, 0);
        q[j] = in ? *reinterpret_cast<const uint4*>(dz + (long)(r0 + j) * C + c0) : make_uint4(0, 0, 0, 0);
    }
    float A[8], m1[8], B[8], mu[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const float rs = rstd[c0 + k];
        A[k] = (fabsf(weight[c0 + k]) + eps) * rs;
        m1[k] = sums[c0 + k] * inv_n;
        B[k] = rs * (sums[C + c0 + k] * inv_n);
        mu[k] = mean[c0 + k];
    }
#pragma unroll
    for (int j = 0; j < RPG; ++j) {
        if (r0 + j >= M) break;
        float v[8], w[8];
        decode8(c[j], pow2(((j < 4 ? sb.x : sb.y) >> (8 * (j & 3))) & 0xffu), v);
        unpack8(q[j], w);
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = A[k] * ((w[k] - m1[k]) - (v[k] - mu[k]) * B[k]);
        *reinterpret_cast<uint4*>(dx + (long)(r0 + j) * C + c0) = pack8(w);
    }
}

inline int nblocks(int C) { return (C + BLK - 1) / BLK; }
inline int code_ld(int C) { return (C + 15) & ~15; }
inline long scale_ld(long M) { return (M + 15) & ~15L; }
inline int lanes_for(int C) { return C > 64 ? 16 : (C > 32 ? 8 : 4); }
inline bool aligned(const void* p, int n) { return ((uintptr_t)p & (uintptr_t)(n - 1)) == 0; }
inline int done() { return hipGetLastError() == hipSuccess ? MGN_OK : MGN_ELAUNCH; }
constexpr long MAX_ROWS = 0x7fffff00L;    // rows are counted in 32 bits (padded to 16), offsets in 64
constexpr int MAX_COLS = 1 << 20;

// The streaming product's form for these sizes; false where another kernel is meant.  src_kind as SRC; `least` tiles for each block, or that
// other kernel; vec: 16-bit results in rows of 16-byte pieces.
struct StreamForm { int ki, shape, th, BM, groups, gx, ntiles; };
bool stream_form(long M, int K, int N, bool vec, int src_kind, int least, StreamForm* f) {
    if (K > 512 || scale_ld(M) * 4 > 0x7fffffffL || (!vec && N > 32)) return false;
    f->ki = K <= 128 ? 0 : (K <= 256 ? 1 : 2);
    const int KB = 1 << f->ki;
    f->shape = !vec ? 0 : (N <= 32 ? 1 : (N <= 128 ? 2 : 3));
    const int chans = f->shape <= 1 ? 32 : (f->shape == 2 ? 128 : 256);
    f->th = KB == 4 && f->shape == 3 ? 512 : 256;
    f->BM = 128 / KB * (src_kind == 0 ? 2 : 1) * (f->th / 256);
    f->groups = (N + chans - 1) / chans;
    f->ntiles = (int)((M + f->BM - 1) / f->BM);
    f->gx = (512 * 256 / f->th) / f->groups & ~7;   // two blocks a CU (one of 512 threads)
    if (f->gx < 8 || f->ntiles < least * f->gx) return false;
    f->gx = f->ntiles < f->gx ? f->ntiles : f->gx;
    return true;
}
bool stream_vec(int N, const void* out, int out32, long ldo) { return !out32 && N % 8 == 0 && ldo % 8 == 0 && ldo <= MAX_COLS && aligned(out, 16); }

// The streaming product; MGN_ENOTSUP where another kernel is meant.
int launch_stream(StreamParams p, int src_kind, int least, hipStream_t s) {
    StreamForm f;
    if (!stream_form(p.M, p.K, p.N, stream_vec(p.N, p.out, p.out32, p.ldo), src_kind, least, &f)) return MGN_ENOTSUP;
    p.ntiles = f.ntiles;
    const int ki = f.ki, shape = f.shape, KB = 1 << ki, lds = 2 * (f.BM * KB * BLK + KB * f.BM) + 1024;
    typedef void (*K)(StreamParams);
#define Q8_SRC(N) {q8_stream_##N##_packed, q8_stream_##N##_h16, q8_stream_##N##_keep}
    static const K table[3][4][3] = {{Q8_SRC(1_any), Q8_SRC(1_32), Q8_SRC(1_128), Q8_SRC(1_256)},
                                     {Q8_SRC(2_any), Q8_SRC(2_32), Q8_SRC(2_128), Q8_SRC(2_256)},
                                     {Q8_SRC(4_any), Q8_SRC(4_32), Q8_SRC(4_128), Q8_SRC(4_256)}};
#undef Q8_SRC
    K kernel = table[ki][shape][src_kind];
    if (lds > 65536) {
        int dev = 0;
        static bool ready[64][3][4][3] = {};
        if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return MGN_ELAUNCH;
        bool& r = ready[dev][ki][shape][src_kind];
        if (!r) {
            if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return MGN_ELAUNCH;
            r = true;
        }
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)f.gx, (unsigned)f.groups), dim3(f.th), lds, s, p);
    return done();
}

template <int BM, int BN, int LDS, int TH>
int launch_mm(void (*kernel)(MmParams), MmParams p, hipStream_t s) {
    p.mt = (int)(((long)p.M + BM - 1) / BM);
    p.nt = (p.N + BN - 1) / BN;
    const long blocks = ((long)p.mt * p.nt + 7) / 8 * 8;
    dim3 grid;
    if (blocks > 0x7fffffffL || !flat_grid(blocks, TH, &grid)) return MGN_EINVAL;
    if (LDS > 65536) {
        static bool ready[64] = {};
        int dev = 0;
        if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return MGN_ELAUNCH;
        if (!ready[dev]) {
            if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess) return MGN_ELAUNCH;
            ready[dev] = true;
        }
    }
    hipLaunchKernelGGL(kernel, grid, dim3(TH), LDS, s, p);
    return done();
}

}  // namespace

#define Q8_LANES(C, CALL) do { switch (lanes_for(C)) { case 16: { constexpr int LPB = 16; CALL; } break; case 8: { constexpr int LPB = 8; CALL; } break; default: { constexpr int LPB = 4; CALL; } } } while (0)

extern "C" {

#ifndef MGN_F16
int mgn_q8_bytes(long M, int C, size_t* codes, size_t* scales) {
    if (M < 0 || M > MAX_ROWS || C < 1 || C > MAX_COLS || !codes || !scales) return MGN_EINVAL;
    *codes = (size_t)M * code_ld(C);
    *scales = (size_t)nblocks(C) * scale_ld(M);
    return MGN_OK;
}
#endif

int MGN_SYM(mgn_q8_pack)(const void* x, int dtype, long M, int C, long sn, long sh, long sw, int H, int W, void* codes, void* scales, void* stream_) {
    if (M < 0 || M > MAX_ROWS || C < 1 || C > MAX_COLS || (dtype != 0 && dtype != 1) || sn < 0 || sh < 0 || sw < 0) return MGN_EINVAL;
    if (M == 0) return MGN_OK;
    if (!x || !codes || !scales || H < 1 || W < 1 || M % ((long)H * W) != 0 || !aligned(codes, 16) || !aligned(scales, 16) || !aligned(x, dtype ? 2 : 4)) return MGN_EINVAL;
    long images = M / ((long)H * W);
    if (W == 1) { W = H; H = 1; sw = sh; }                                  // (the stride of an axis of length one says nothing)
    if (W == 1 && images <= 0x7fffffffL) { W = (int)images; sw = sn; images = 1; }
    RowMap map = {sn, sh, sw, H, W, 0};
    map.flat = (H == 1 || sh == (long)W * sw) && (images == 1 || sn == (long)H * W * sw);
    const int nb = nblocks(C), ldc = code_ld(C), lpb = lanes_for(C);
    const long groups = (M + RPG - 1) / RPG * nb;
    dim3 grid;
    if (!flat_grid((groups * lpb + TPB - 1) / TPB, TPB, &grid)) return MGN_EINVAL;
    hipStream_t s = (hipStream_t)stream_;
#define Q8_PACK(T) Q8_LANES(C, (hipLaunchKernelGGL((q8_pack<T, LPB>), grid, dim3(TPB), 0, s, (const T*)x, map, (int)M, C, nb, ldc, \
                                                   scale_ld(M), (unsigned char*)codes, (unsigned char*)scales)))
    if (dtype) Q8_PACK(uint16_t); else Q8_PACK(float);
#undef Q8_PACK
    return done();
}

int MGN_SYM(mgn_q8_unpack)(const void* codes, const void* scales, long M, int C, void* y, int dtype, void* stream_) {
    if (M < 0 || M > MAX_ROWS || C < 1 || C > MAX_COLS || (dtype != 0 && dtype != 1)) return MGN_EINVAL;
    if (M == 0) return MGN_OK;
    if (!codes || !scales || !y || !aligned(codes, 16) || !aligned(scales, 16) || !aligned(y, dtype ? 2 : 4)) return MGN_EINVAL;
    const int nb = nblocks(C), ldc = code_ld(C), lpb = lanes_for(C);
    const long groups = (M + RPG - 1) / RPG * nb;
    dim3 grid;
    if (!flat_grid((groups * lpb + TPB - 1) / TPB, TPB, &grid)) return MGN_EINVAL;
    hipStream_t s = (hipStream_t)stream_;
#define Q8_UNPACK(T) Q8_LANES(C, (hipLaunchKernelGGL((q8_unpack<T, LPB>), grid, dim3(TPB), 0, s, (const unsigned char*)codes, \
                                                     (const unsigned char*)scales, (int)M, C, nb, ldc, scale_ld(M), (T*)y)))
    if (dtype) Q8_UNPACK(uint16_t); else Q8_UNPACK(float);
#undef Q8_UNPACK
    return done();
}

int MGN_SYM(mgn_q8_pack_weight)(const void* w, int dtype, long sr, long sc, int N, int K, void* codes, void* scales, void* codes_t, void* scales_t,
                                void* stream_) {
    if (N < 1 || K < 1 || N > MAX_COLS || K > MAX_COLS || (dtype != 0 && dtype != 1) || !w || sr < 0 || sc < 0 || !aligned(w, dtype ? 2 : 4)) return MGN_EINVAL;
    if ((!codes && !codes_t) || !codes != !scales || !codes_t != !scales_t || !aligned(codes, 16) || !aligned(codes_t, 16)) return MGN_EINVAL;
    const dim3 grid((unsigned)nblocks(N), (unsigned)nblocks(K));
    hipStream_t s = (hipStream_t)stream_;
    if (dtype) hipLaunchKernelGGL(q8_pack_tile<uint16_t>, grid, dim3(TILE_TPB), 0, s, (const uint16_t*)w, sr, sc, N, K, (unsigned char*)codes,
                                  (unsigned char*)scales, (unsigned char*)codes_t, (unsigned char*)scales_t);
    else hipLaunchKernelGGL(q8_pack_tile<float>, grid, dim3(TILE_TPB), 0, s, (const float*)w, sr, sc, N, K, (unsigned char*)codes, (unsigned char*)scales,
                            (unsigned char*)codes_t, (unsigned char*)scales_t);
    return done();
}

int MGN_SYM(mgn_q8_matmul)(const void* a, const void* a_scales, long M, const void* b, const void* b_scales, int N, int K, const float* bias, int act,
                           float slope, void* out, int out_f32, long ldo, void* stream_) {
    if (M < 0 || M > MAX_ROWS || N < 1 || N > MAX_COLS || K < 1 || K > MAX_COLS || !act_ok(act, slope) || ldo < N) return MGN_EINVAL;
    if (M == 0) return MGN_OK;
    if (!a || !a_scales || !b || !b_scales || !out || !aligned(a, 16) || !aligned(b, 16) || !aligned(a_scales, 16) || !aligned(b_scales, 16) ||
        !aligned(out, out_f32 ? 4 : 2)) return MGN_EINVAL;
    MmParams p = {(const unsigned char*)a, (const unsigned char*)a_scales, (const unsigned char*)b, (const unsigned char*)b_scales, bias, out,
                  (int)M, N, K, nblocks(K), code_ld(K), scale_ld(M), scale_ld(N), ldo, make_act(act, slope), out_f32, 0, 0};
    hipStream_t s = (hipStream_t)stream_;
    auto tiles = [&](int BM, int BN) { return ((M + BM - 1) / BM) * ((N + BN - 1) / BN); };
    // Up to some 1400 tiles of 32 x 32 the chip is better filled by those, k split over their waves, than by larger ones: 256 x 4096 x 4096
    // (1024 tiles) 15.2 us against 21.9 with 128 x 128, 459 x 2932 x 3872 (1380) 22.9 against 22.6, 1500^3 (2209) 16.3 against 12.8
    const long gy = (M + 31) / 32;
    if ((M <= 64 || tiles(32, 32) <= 1400) && gy <= 65535) {
        const int lds = p.nb > 4 ? 8 * SMALL_STAGE : 4 * SMALL_STAGE;   // (a wave with one block of k needs one stage)
        hipLaunchKernelGGL(q8_mm_small, dim3((unsigned)((N + 31) / 32), (unsigned)gy), dim3(TPB), lds, s, p);
        return done();
    }
    if (K <= 512) {
        // more than 128 channels: only with two tiles or more for each persistent block (16000 x 512 x 512, one tile a block: 13.5 us against
        // 10.9 with 128 x 128 tiles; 256000 x 512 x 512: 106 against 133)
        StreamParams q = {p.a, p.sa, nullptr, nullptr, p.b, p.sb, bias, out, (int)M, K, N, p.ld, p.ld, p.ld, 0, p.lda_s, p.ldb_s, ldo, make_act(act, slope), out_f32};
        const int rc = launch_stream(q, 0, N > 128 ? 2 : 0, s);
        if (rc != MGN_ENOTSUP) return rc;
    }
    if (N <= 32) return launch_mm<128, 32, MmTile<128, 32, 4, 1, 3>::LDS, 256>(q8_mm_128x32, p, s);
    // 256 blocks of 256 x 256 fill the chip, 512 of 128 x 128, the former 1.16 times as fast (8192^3: 421 us against 490): the better of the two
    // by the share of a whole number of rounds that is used
    auto used = [&](int B, long slots) { const long t = tiles(B, B); return (double)M * N / ((double)((t + slots - 1) / slots * slots) * B * B); };
    if (N > 128 && 1.16 * used(256, 256) >= used(128, 512)) return launch_mm<256, 256, Mm256::LDS, 512>(q8_mm_256x256, p, s);
    return launch_mm<128, 128, MmTile<128, 128, 2, 2, 2>::LDS, 256>(q8_mm_128x128, p, s);
}

// whether mgn_q8_pack_matmul packs on the way
static bool stream_packs(const void* x, long M, int K, long ldx, int N, const void* out, int out_f32, long ldo, int src_kind) {
    StreamForm f;
    return K % 8 == 0 && ldx % 8 == 0 && aligned(x, 16) && stream_form(M, K, N, stream_vec(N, out, out_f32, ldo), src_kind, 0, &f);
}

int MGN_SYM(mgn_q8_pack_matmul)(const void* x, long M, int K, long ldx, void* codes, void* scales, const void* b, const void* b_scales, int N,
                                const float* bias, int act, float slope, void* out, int out_f32, long ldo, void* stream_) {
    if (M < 0 || M > MAX_ROWS || N < 1 || N > MAX_COLS || K < 1 || K > MAX_COLS || !act_ok(act, slope) || ldo < N || ldx < K || ldx > MAX_COLS) return MGN_EINVAL;
    if (M == 0) return MGN_OK;
    if (!x || !b || !b_scales || !out || !codes != !scales || !aligned(codes, 16) || !aligned(scales, 16) || !aligned(b, 16) || !aligned(x, 2) ||
        !aligned(out, out_f32 ? 4 : 2)) return MGN_EINVAL;
    if (!stream_packs(x, M, K, ldx, N, out, out_f32, ldo, codes ? 2 : 1)) return MGN_ENOTSUP;
    StreamParams p = {(const unsigned char*)x, nullptr, (unsigned char*)codes, (unsigned char*)scales, (const unsigned char*)b, (const unsigned char*)b_scales, bias, out,
                      (int)M, K, N, (int)ldx, code_ld(K), code_ld(K), 0, scale_ld(M), scale_ld(N), ldo, make_act(act, slope), out_f32};
    return launch_stream(p, codes ? 2 : 1, 0, (hipStream_t)stream_);
}

#ifndef MGN_F16
static size_t wgrad_floats(int N, int K) { return ((size_t)N * K + N + 3) & ~(size_t)3; }
// Row ranges: the power of two that minimises (steps a CU goes through) + (writing and reading the partial results), with the step at
// 0.5 us and the traffic at 5 TB/s, both as measured, among those whose ranges a 32-bit buffer descriptor reaches (offsets run up to four
// steps past the range); 0 if none does.  262144 x 256 x 256: 128; 16384 x 256 x 512: 32.
static long wgrad_rows(long M, int splits) { return ((M + splits - 1) / splits + WG_ROWS - 1) / WG_ROWS * WG_ROWS; }
static bool wgrad_reach(long rows, long ldy, int K) { return (rows + 4 * WG_ROWS) * (ldy * 2 > code_ld(K) ? ldy * 2 : code_ld(K)) <= 0x7fffffffL; }
static int wgrad_splits(long M, int N, int K) {
    const double tiles = (double)nblocks(N) * nblocks(K), bytes = 8.0 * (double)wgrad_floats(N, K);
    double best = 1e300;
    int z = 0;
    for (int c = 1; c <= 512 && (c == 1 || (long)c * WG_ROWS <= M * 2); c *= 2) {
        if (!wgrad_reach(wgrad_rows(M, c), (N + 7) & ~7, K)) continue;
        const double steps = (double)((M + (long)c * WG_ROWS - 1) / ((long)c * WG_ROWS)), rounds = (double)((long)((tiles * c + 511) / 512));
        const double t = steps * rounds * 0.5 + c * bytes / 5e6;
        if (t < best) { best = t; z = c; }
    }
    return z;
}
int mgn_q8_wgrad_workspace_bytes(long M, int N, int K, size_t* bytes) {
    if (M < 1 || M > MAX_ROWS || N < 1 || K < 1 || N > 65536 || K > 65536 || !bytes) return MGN_EINVAL;
    const int splits = wgrad_splits(M, N, K);
    if (splits == 0) return MGN_EINVAL;
    *bytes = sizeof(float) * (size_t)splits * wgrad_floats(N, K);
    return MGN_OK;
}
#endif

int MGN_SYM(mgn_q8_wgrad)(const void* dy, long ldy, long M, int N, const void* codes, const void* scales, int K, float* dw, float* db, void* ws,
                          size_t ws_bytes, void* stream_) {
    size_t need = 0;
    const int rc = mgn_q8_wgrad_workspace_bytes(M, N, K, &need);
    if (rc != MGN_OK) return rc;
    if (!dy || !codes || !scales || !dw || !ws || !aligned(dy, 16) || !aligned(codes, 16) || ldy < N || ldy % 8 != 0 || ldy > 65536) return MGN_EINVAL;
    if (ws_bytes < need) return MGN_ENOSPC;
    const int zmax = (int)(need / (sizeof(float) * (((size_t)N * K + N + 3) & ~(size_t)3)));
    const long rows = ((M + zmax - 1) / zmax + WG_ROWS - 1) / WG_ROWS * WG_ROWS;   // whole steps
    if ((rows + 4 * WG_ROWS) * (ldy * 2 > code_ld(K) ? ldy * 2 : code_ld(K)) > 0x7fffffffL) return MGN_EINVAL;   // (a row pitch beyond wgrad_splits' own)
    WgradParams8 p = {(const uint16_t*)dy, (const unsigned char*)codes, (const unsigned char*)scales, (float*)ws, (int)M, N, K, (int)ldy, code_ld(K),
                      scale_ld(M), (int)rows, (int)((M + rows - 1) / rows), nblocks(N), nblocks(K)};
    const long blocks = (long)((p.splits + 7) / 8) * 8 * p.ntn * p.ntk;
    const long nk = (long)N * K, total = nk + N;
    dim3 grid, rgrid;
    if (blocks > 0x7fffffffL || !flat_grid(blocks, TPB, &grid) || !flat_grid((total + 255) / 256, 1024, &rgrid)) return MGN_EINVAL;
    hipStream_t s = (hipStream_t)stream_;
    static bool ready[64] = {};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return MGN_ELAUNCH;
    if (!ready[dev]) {
        if (hipFuncSetAttribute(reinterpret_cast<const void*>(q8_wgrad), hipFuncAttributeMaxDynamicSharedMemorySize, WG_LDS) != hipSuccess) return MGN_ELAUNCH;
        ready[dev] = true;
    }
    hipLaunchKernelGGL(q8_wgrad, grid, dim3(TPB), WG_LDS, s, p);
    hipLaunchKernelGGL(q8_wgrad_reduce, rgrid, dim3(1024), 0, s, (const float*)ws, p.splits, total, nk, dw, db);
    return done();
}

/* ---- the trained 1x1 convolution in two calls ---- */
// [transposed weights][weights][packed x], offsets, every piece a multiple of 16 bytes: what the data gradient reads comes first, what only the
// weight gradient reads comes last
struct ConvBuffer { size_t tcodes, tscales, wcodes, wscales, codes, scales, total; };
static ConvBuffer conv_buffer(long M, int C, int N) {
    ConvBuffer b;
    b.tcodes = 0;
    b.tscales = b.tcodes + (size_t)C * code_ld(N);
    b.wcodes = b.tscales + (size_t)nblocks(N) * scale_ld(C);
    b.wscales = b.wcodes + (size_t)N * code_ld(C);
    b.codes = b.wscales + (size_t)nblocks(C) * scale_ld(N);
    b.scales = b.codes + (size_t)M * code_ld(C);
    b.total = b.scales + (size_t)nblocks(C) * scale_ld(M);
    return b;
}
static bool conv_shape(long M, int C, int N) { return M >= 0 && M <= MAX_ROWS && C >= 1 && C <= 65536 && N >= 1 && N <= 65536; }
static int pad8(int n) { return (n + 7) & ~7; }
// what the backward call needs: [dy padded][dy packed, if the data gradient's product does not pack it on the way][partial weight gradients]
struct ConvScratch { size_t pad, codes, scales, part, total; };
static ConvScratch conv_scratch(long M, int N, bool pack, size_t part_bytes) {
    ConvScratch b;
    b.pad = 0;
    b.codes = N % 8 ? (size_t)M * pad8(N) * 2 : 0;
    b.scales = b.codes + (pack ? (size_t)M * code_ld(N) : 0);
    b.part = b.scales + (pack ? (size_t)nblocks(N) * scale_ld(M) : 0);
    b.total = b.part + part_bytes;
    return b;
}
// dy and dx are 16-byte aligned rows (`dy`: the padded rows are in the scratch memory, as well aligned)
static bool conv_packs_dy(long M, int C, int N, const void* dx) { return !stream_packs(nullptr, M, pad8(N), pad8(N), C, dx, 0, C, 1); }

#ifndef MGN_F16
int mgn_q8_conv1x1_bytes(long M, int C, int N, size_t* buffer, size_t* scratch) {
    if (!conv_shape(M, C, N) || !buffer || !scratch) return MGN_EINVAL;
    *buffer = conv_buffer(M, C, N).total;
    size_t part = 0;
    if (M > 0) { const int rc = mgn_q8_wgrad_workspace_bytes(M, N, C, &part); if (rc != MGN_OK) return rc; }
    *scratch = conv_scratch(M, N, true, part).total;
    return MGN_OK;
}
int mgn_q8_conv1x1_bwd_bytes(long M, int C, int N, int want_dx, int want_dw, size_t* scratch) {
    if (!conv_shape(M, C, N) || !scratch) return MGN_EINVAL;
    size_t part = 0;
    if (M > 0 && want_dw) { const int rc = mgn_q8_wgrad_workspace_bytes(M, N, C, &part); if (rc != MGN_OK) return rc; }
    *scratch = M > 0 ? conv_scratch(M, N, want_dx && conv_packs_dy(M, C, N, nullptr), part).total : 0;
    return MGN_OK;
}
#endif

// rows of C 16-bit values one behind the other
static bool conv_flat(long M, int C, long sn, long sh, long sw, int H, int W) {
    const long images = H < 1 || W < 1 ? 0 : M / ((long)H * W);
    return (W == 1 || sw == C) && (H == 1 || sh == (long)W * C) && (images == 1 || sn == (long)H * W * C);
}
// x goes into the product without a packed form in memory
static bool conv_unkept(const void* x, long M, int C, long sn, long sh, long sw, int H, int W, int N, const void* y, int keep) {
    return M == 0 || (!keep && conv_flat(M, C, sn, sh, sw, H, W) && stream_packs(x, M, C, C, N, y, 0, N, 1));
}

#ifndef MGN_F16
int mgn_q8_conv1x1_fwd_bytes(const void* x, long M, int C, long sn, long sh, long sw, int H, int W, int N, const void* y, int keep, size_t* buffer,
                             size_t* kept) {
    if (!conv_shape(M, C, N) || !buffer || !kept) return MGN_EINVAL;
    const ConvBuffer b = conv_buffer(M, C, N);
    *buffer = conv_unkept(x, M, C, sn, sh, sw, H, W, N, y, keep) ? b.codes : b.total;
    *kept = keep ? b.total : b.wcodes;
    return MGN_OK;
}
#endif

int MGN_SYM(mgn_q8_conv1x1_fwd)(const void* x, long M, int C, long sn, long sh, long sw, int H, int W, const void* w, int w_dtype, long w_sr, long w_sc,
                                int N, const float* bias, int relu, void* y, int keep, void* buffer, size_t buffer_bytes, void* stream_) {
    if (!conv_shape(M, C, N) || !w || !buffer || !aligned(buffer, 16)) return MGN_EINVAL;
    if (M > 0 && (!x || !y || H < 1 || W < 1 || M % ((long)H * W) != 0 || sn < 0 || sh < 0 || sw < 0 || !aligned(x, 2) || !aligned(y, 2))) return MGN_EINVAL;
    const ConvBuffer b = conv_buffer(M, C, N);
    if (buffer_bytes < (conv_unkept(x, M, C, sn, sh, sw, H, W, N, y, keep) ? b.codes : b.total)) return MGN_ENOSPC;
    unsigned char* p = (unsigned char*)buffer;
    int rc = MGN_SYM(mgn_q8_pack_weight)(w, w_dtype, w_sr, w_sc, N, C, p + b.wcodes, p + b.wscales, p + b.tcodes, p + b.tscales, stream_);
    if (rc != MGN_OK || M == 0) return rc;
    rc = MGN_ENOTSUP;
    if (conv_flat(M, C, sn, sh, sw, H, W)) rc = MGN_SYM(mgn_q8_pack_matmul)(x, M, C, C, keep ? p + b.codes : nullptr, keep ? p + b.scales : nullptr, p + b.wcodes, p + b.wscales, N, bias,
                                               relu ? 1 : 0, 0.f, y, 0, N, stream_);
    if (rc != MGN_ENOTSUP) return rc;
    rc = MGN_SYM(mgn_q8_pack)(x, 1, M, C, sn, sh, sw, H, W, p + b.codes, p + b.scales, stream_);
    if (rc != MGN_OK) return rc;
    return MGN_SYM(mgn_q8_matmul)(p + b.codes, p + b.scales, M, p + b.wcodes, p + b.wscales, N, C, bias, relu ? 1 : 0, 0.f, y, 0, N, stream_);
}

int MGN_SYM(mgn_q8_conv1x1_bwd)(const void* dy, long M, int C, int N, const void* buffer, void* dx, float* dw, float* db, void* scratch,
                                size_t scratch_bytes, void* stream_) {
    if (!conv_shape(M, C, N)) return MGN_EINVAL;
    size_t part = 0;
    int rc = dw ? mgn_q8_wgrad_workspace_bytes(M, N, C, &part) : MGN_OK;
    if (rc != MGN_OK) return rc;
    if (M < 1 || !dy || !buffer || (!dx && !dw) || (db && !dw) || !aligned(dy, 16) || !aligned(buffer, 16) || !aligned(scratch, 16)) return MGN_EINVAL;
    const ConvBuffer b = conv_buffer(M, C, N);
    const ConvScratch t = conv_scratch(M, N, dx && conv_packs_dy(M, C, N, dx), part);
    if (!scratch && t.total) return MGN_EINVAL;
    if (scratch_bytes < t.total) return MGN_ENOSPC;
    const unsigned char* p = (const unsigned char*)buffer;
    unsigned char* s = (unsigned char*)scratch;
    const int ldy = pad8(N);
    if (N % 8) {
        dim3 grid;
        if (!flat_grid((M * (ldy / 8) + TPB - 1) / TPB, TPB, &grid)) return MGN_EINVAL;
        hipLaunchKernelGGL(q8_pad_rows, grid, dim3(TPB), 0, (hipStream_t)stream_, (const uint16_t*)dy, M, N, ldy, (uint4*)(s + t.pad));
        dy = s + t.pad;
    }
    if (dx) {   // (K = N padded: the columns behind N are zeros on both sides)
        rc = MGN_SYM(mgn_q8_pack_matmul)(dy, M, ldy, ldy, nullptr, nullptr, p + b.tcodes, p + b.tscales, C, nullptr, 0, 0.f, dx, 0, C, stream_);
        if (rc == MGN_ENOTSUP) {
            rc = MGN_SYM(mgn_q8_pack)(dy, 1, M, N, ldy, 0, 0, 1, 1, s + t.codes, s + t.scales, stream_);
            if (rc == MGN_OK) rc = MGN_SYM(mgn_q8_matmul)(s + t.codes, s + t.scales, M, p + b.tcodes, p + b.tscales, C, N, nullptr, 0, 0.f, dx, 0, C, stream_);
        }
        if (rc != MGN_OK) return rc;
    }
    if (dw) return MGN_SYM(mgn_q8_wgrad)(dy, ldy, M, N, p + b.codes, p + b.scales, C, dw, db, s + t.part, part, stream_);
    return MGN_OK;
}

/* ---- block tail ---- */
static int tail_shape(long M, int C) { return (M < 1 || M > MAX_ROWS || C < 8 || C % 8 != 0 || C > 8192) ? MGN_EINVAL : MGN_OK; }
static unsigned tail_rows(long M, int C) {   // row blocks of the reductions: 16 rows a thread before there are more blocks than fill the chip
    const int rpb = TPB / lanes_for(C);
    const long b = (M + (long)rpb * 16 - 1) / ((long)rpb * 16);
    return (unsigned)(b < 1 ? 1 : (b > TAIL_BLOCKS ? TAIL_BLOCKS : b));
}
static unsigned tail_grid(long M, int C) {
    const int rows = TPB / lanes_for(C) * RPG;
    return (unsigned)((M + rows - 1) / rows);
}

#ifndef MGN_F16
int mgn_q8_tail_partial_rows(long M, int C, int* rows) {
    if (tail_shape(M, C) != MGN_OK || !rows) return MGN_EINVAL;
    *rows = (int)tail_rows(M, C);
    return MGN_OK;
}
#endif

int MGN_SYM(mgn_q8_tail_stats)(const void* x, long M, int C, float* partials, float* shift, void* stream_) {
    if (tail_shape(M, C) != MGN_OK || !x || !partials || !shift || !aligned(x, 16)) return MGN_EINVAL;
    const dim3 grid(tail_rows(M, C), (unsigned)nblocks(C));
    Q8_LANES(C, (hipLaunchKernelGGL(q8_tail_stats<LPB>, grid, dim3(TPB), 0, (hipStream_t)stream_, (const uint16_t*)x, (int)M, C, partials, shift)));
    return done();
}

int MGN_SYM(mgn_q8_tail_fwd)(const void* x, const void* shortcut, const float* scale, const float* offset, long M, int C, void* y, void* codes,
                             void* scales, void* relu_bits, void* stream_) {
    if (tail_shape(M, C) != MGN_OK || !x || !shortcut || !scale || !offset || !y || !codes != !scales || !codes != !relu_bits || !aligned(x, 16) ||
        !aligned(shortcut, 16) || !aligned(y, 16) || !aligned(codes, 16) || !aligned(scales, 16)) return MGN_EINVAL;
    const dim3 grid(tail_grid(M, C), (unsigned)nblocks(C));
#define Q8_TAIL(K) Q8_LANES(C, (hipLaunchKernelGGL((q8_tail_fwd<LPB, K>), grid, dim3(TPB), 0, (hipStream_t)stream_, (const uint16_t*)x, \
        (const uint16_t*)shortcut, scale, offset, (int)M, C, code_ld(C), scale_ld(M), (uint16_t*)y, (unsigned char*)codes, (unsigned char*)scales, \
        (unsigned char*)relu_bits)))
    if (codes) Q8_TAIL(true); else Q8_TAIL(false);
#undef Q8_TAIL
    return done();
}

int MGN_SYM(mgn_q8_tail_bwd_reduce)(const void* codes, const void* scales, const void* g, const void* relu_bits, const float* mean, const float* rstd,
                                    const float* weight, long M, int C, void* dz, float* partials, float* sums, float* dwb, void* stream_) {
    if (tail_shape(M, C) != MGN_OK || !codes || !scales || !g || !relu_bits || !mean || !rstd || !weight || !dz || !partials || !sums || !dwb ||
        !aligned(codes, 16) || !aligned(g, 16) || !aligned(dz, 16)) return MGN_EINVAL;
    const dim3 grid(tail_rows(M, C), (unsigned)nblocks(C));
    hipStream_t s = (hipStream_t)stream_;
    Q8_LANES(C, (hipLaunchKernelGGL(q8_tail_bwd_reduce<LPB>, grid, dim3(TPB), 0, s, (const unsigned char*)codes, (const unsigned char*)scales,
                                    (const uint16_t*)g, (const unsigned char*)relu_bits, mean, (int)M, C, code_ld(C), scale_ld(M), (uint16_t*)dz, partials)));
    return mgn_q8_tail_sums(partials, (int)grid.x, C, rstd, weight, sums, dwb, stream_);
}

#ifndef MGN_F16
int mgn_q8_tail_sums(const float* partials, int rows, int C, const float* rstd, const float* weight, float* sums, float* dwb, void* stream_) {
    if (!partials || rows < 1 || C < 8 || C % 8 != 0 || !rstd || !weight || !sums || !dwb) return MGN_EINVAL;
    hipLaunchKernelGGL(q8_tail_sums, dim3((unsigned)(C / 4)), dim3(TPB), 0, (hipStream_t)stream_, partials, rows, C, rstd, weight, sums, dwb);
    return done();
}
#endif

int MGN_SYM(mgn_q8_tail_bwd_apply)(const void* codes, const void* scales, const void* dz, const float* weight, const float* mean, const float* rstd,
                                   const float* sums, float total_count, float eps, long M, int C, void* dx, void* stream_) {
    if (tail_shape(M, C) != MGN_OK || !codes || !scales || !dz || !weight || !mean || !rstd || !sums || !dx || !(total_count > 0.f) ||
        !aligned(codes, 16) || !aligned(scales, 16) || !aligned(dz, 16) || !aligned(dx, 16)) return MGN_EINVAL;
    const dim3 grid(tail_grid(M, C), (unsigned)nblocks(C));
    Q8_LANES(C, (hipLaunchKernelGGL(q8_tail_bwd_apply<LPB>, grid, dim3(TPB), 0, (hipStream_t)stream_, (const unsigned char*)codes,
                                    (const unsigned char*)scales, (const uint16_t*)dz, weight, mean, rstd, sums, 1.f / total_count, eps, (int)M, C,
                                    code_ld(C), scale_ld(M), (uint16_t*)dx)));
    return done();
}

#ifndef MGN_F16
int mgn_q8_tail_workspace_bytes(long M, int C, size_t* bytes) {
    if (tail_shape(M, C) != MGN_OK || !bytes) return MGN_EINVAL;
    *bytes = sizeof(float) * ((size_t)tail_rows(M, C) * C * 2 + C);
    return MGN_OK;
}
#endif

int MGN_SYM(mgn_q8_tail_train_fwd)(const void* x, const void* shortcut, long M, int C, const float* weight, const float* bias, float eps, float momentum,
                                   float* running_mean, float* running_var, float* coef, void* y, void* codes, void* scales, void* relu_bits, void* ws,
                                   size_t ws_bytes, void* stream_) {
    size_t need = 0;
    int rc = mgn_q8_tail_workspace_bytes(M, C, &need);
    if (rc != MGN_OK) return rc;
    if (!ws || !coef) return MGN_EINVAL;
    if (ws_bytes < need) return MGN_ENOSPC;
    const int rows = (int)tail_rows(M, C);
    float *part = (float*)ws, *shift = part + (size_t)rows * C * 2;
    rc = MGN_SYM(mgn_q8_tail_stats)(x, M, C, part, shift, stream_);
    if (rc == MGN_OK) rc = mgn_iabn_coeffs_from_partials(part, rows, C, M, shift, weight, bias, eps, momentum, running_mean, running_var, coef, nullptr, stream_);
    if (rc == MGN_OK) rc = MGN_SYM(mgn_q8_tail_fwd)(x, shortcut, coef, coef + C, M, C, y, codes, scales, relu_bits, stream_);
    return rc;
}

int MGN_SYM(mgn_q8_tail_train_bwd)(const void* codes, const void* scales, const void* g, const void* relu_bits, const float* coef, const float* weight,
                                   float eps, long M, int C, void* dz, void* dx, float* sums_dwb, void* ws, size_t ws_bytes, void* stream_) {
    size_t need = 0;
    int rc = mgn_q8_tail_workspace_bytes(M, C, &need);
    if (rc != MGN_OK) return rc;
    if (!ws || !coef || !sums_dwb) return MGN_EINVAL;
    if (ws_bytes < need) return MGN_ENOSPC;
    rc = MGN_SYM(mgn_q8_tail_bwd_reduce)(codes, scales, g, relu_bits, coef + 2 * (size_t)C, coef + 3 * (size_t)C, weight, M, C, dz, (float*)ws, sums_dwb,
                                         sums_dwb + 2 * (size_t)C, stream_);
    if (rc == MGN_OK && dx) rc = MGN_SYM(mgn_q8_tail_bwd_apply)(codes, scales, dz, weight, coef + 2 * (size_t)C, coef + 3 * (size_t)C, sums_dwb, (float)M, eps, M, C,
                                                                dx, stream_);
    return rc;
}

}  // extern "C"
