// paged_chunk.hpp - attention of requests with many new tokens (more than 16 query
// rows per KV head, or more than 8 beside larger ones) over a paged q4_0 pool.
//
// A workgroup takes 128 (or 64) query rows of one request and KV head (GQA packed: row
// r is token r / G, head kvh * G + r % G) and a range of its keys, 32 at a time. Its 8
// wavefronts split the work by kind as in the contiguous prefill kernel: four score
// wavefronts hold Q' (hi and lo) of 32 rows each and make the logits and P of tile t,
// four value wavefronts hold O of the same rows and add P V of tile t - 1.
//   S^T = sum over q4_0 blocks b of d_k[b] (Kc_b . Q'h_b + Kc_b . Q'l_b): exact codes as
//   fp16 on v_mfma_f32_32x32x16_f16 (64 rows: 16x16x32), Q' = q8_0(Q) * scale * log2(e) as
//   an fp16 hi + lo pair, the scaling by d_k in fp32; softmax base 2 with a reference
//   maximum that moves only when a logit passes it by kSlack; O += (P d_v) V with P d_v as
//   an fp16 hi + lo pair and exact codes.
// The 32x32 tiles leave the vector unit more of their time than 16x16 ones (two wavefronts
// with 8 fmas for every two 16x16x32: 21.4 ns a pair, for one 32x32x16 18.2), a lane holds one
// row, and LDS serves them without conflicts. Cycles are 8% fewer; how much of that is time is
// up to the card's power: 2040 tokens behind 16000 shared keys 1163 -> 1129 us on one card, as
// long as before on another, 2048 behind 30001 2290 -> 2170 and 2264.
//
// There is no pre-pass: the contiguous kernel expands K and V into 2112 bytes per key
// in its workspace, which for a batch would have to hold every request's keys. Here
// the value wavefronts bring the q4_0 rows themselves into LDS (288 bytes per key and
// head; a 16-key group lies on one page, so its id is one scalar load and its rows a
// scalar base plus constant offsets), which are expanded there for all 128 rows, K by the
// score and V by the value wavefronts between their MFMAs (K by the value wavefronts too:
// 2200 us where this is 2170):
//   iteration t: rows of K tile t + 2 and V tile t + 1 are on their way; K tile t + 1
//   and V tile t are expanded; P V of tile t - 1.
// K codes leave a dword of nibbles by shifts and masks alone: the 8 values of a chunk
// are its dims in the order 0 2 16 18 1 3 17 19, and Q' is laid out in the same order.
// V needs the codes of 8 keys side by side: 16-bit reads of 8 rows, packed in pairs.
//
// d_v enters as d_v 2^E with E, one for a pair of blocks, from the largest |d_v| of the
// keys so far (in [1/2, 1) there; O is rescaled when it falls), and P as P 2^kEp, so that
// A = P d_v stays below 2^14 and the parts that count stay clear of fp16's subnormals for
// V of any size.
//
// Bound: the issue of instructions by one wavefront of each kind a SIMD: vector 0.56 of the
// cycles, matrix 0.43, both at once 0.23, LDS at work in 0.40. Exact products take two MFMAs for
// each useful one; without any the tile still takes 0.64 of its time. 2048 tokens behind 30001, 16
// heads on 2 KV heads: 2.17 ms, 480 TFLOP/s, 2.2 us a tile of 128 x 32. A workgroup's start and
// end are 11 us that nothing overlaps (LDS holds one a CU): Q 2.7, its quantization 2.6,
// the last tile 1.9, the result 3 to 4 (turned in LDS into whole rows it took 5).
#pragma once
#include <type_traits>

#include "paged_work.hpp"

namespace sqa {
namespace paged {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

constexpr int kPK = kChunkKeys;          // keys per tile
constexpr int kScoreWaves = 4;
constexpr int kValueWaves = 4;
constexpr int kThreads = 64 * (kScoreWaves + kValueWaves);
constexpr int kMaxRG = 2;                // 16-row groups per score wave: 1 or 2 (kRG in the kernel)
constexpr int rows_per_wg(int rg) { return kScoreWaves * rg * 16; }
constexpr int kWideRow = 520;            // K stage: Kc (rows of 512 bytes, or of 520), Dk
constexpr int kOffDk = kPK * kWideRow;
constexpr int kKStage = kOffDk + 8 * kPK * 2;
constexpr int kOffDv = kHeadDim * kPK * 2;  // V stage: Vc, Dv
constexpr int kVStage = kOffDv + 8 * kPK * 2;
constexpr int kRawTile = kPK * kHeadRowBytes;  // q4_0 rows of a tile
// LDS map: 2 K stages | 2 V stages | 2 P buffers | 2 rescale buffers | 2 sets of exponents | raw K, V tiles, 2 each
constexpr int kLdsV = 2 * kKStage;
constexpr int kLdsP = kLdsV + 2 * kVStage;        // [4 waves][kRG][2 halves][64 lanes][16 B]
constexpr int kPBuf = kScoreWaves * kMaxRG * 2 * 1024;
constexpr int kLdsA = kLdsP + 2 * kPBuf;          // [4 waves][kRG][16 rows] f32
constexpr int kABuf = kScoreWaves * kMaxRG * 16 * 4;
constexpr int kLdsE = kLdsA + 2 * kABuf;          // [2][4] exponents of the V scales, one per pair of blocks
constexpr int kLdsF = kLdsE + 32;               // [2][4] whether a maximum of the wave's rows has moved
constexpr int kLdsRaw = kLdsF + 32;               // [K, V][2][32 rows][144 B]
constexpr int kLdsBytes = kLdsRaw + 4 * kRawTile + 16;
static_assert(kLdsBytes <= 160 * 1024, "LDS budget");
static_assert(kLdsRaw % 16 == 0 && kKStage % 16 == 0 && kVStage % 16 == 0, "alignment of the stages");
constexpr int kSlack = 8;  // log2 of the largest P the lazy rescale admits
constexpr int kEp = kPBits;  // P travels as P 2^kEp (at most 2^14)
constexpr int kMaxE = 24;  // of the V scales: makes the smallest fp16 one

// max(x, x of lane ^ 16) and max(x, x of lane ^ 32) with gfx950's row swaps (no
// LDS round trip): each swap returns the two halves of a lane pair's values.
__device__ __forceinline__ float xmax16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xmax32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// sa[i] += c[i] * (dk of lane i of every 16 lanes), i = 4 K .. 4 K + 3: the multiplication reads the
// other lane's register (the compiler makes a move of its own of that; every lane reading all its
// scales from LDS, 16 reads of 16 bytes a tile instead of one, took 3% longer). These lines are
// no instructions to the compiler that read c, a matrix instruction's result: K = 0 has one of the
// compiler's own before them, and its waits. s_nop: dk may have been written just before.
template <int K>
__device__ __forceinline__ void add_scaled(float (&sa)[16], float c0, float c1, float c2, float c3, float dk) {
    if constexpr (K == 0) {
        sa[0] = fmaf(__int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(dk), 0x150, 0xf, 0xf, true)), c0, sa[0]);
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_nop 1\n\t"
                     "v_fmac_f32_dpp %0, %3, %4 row_newbcast:1 row_mask:0xf bank_mask:0xf\n\t"
                     "v_fmac_f32_dpp %1, %3, %5 row_newbcast:2 row_mask:0xf bank_mask:0xf\n\t"
                     "v_fmac_f32_dpp %2, %3, %6 row_newbcast:3 row_mask:0xf bank_mask:0xf"
                     : "+v"(sa[1]), "+v"(sa[2]), "+v"(sa[3]) : "v"(dk), "v"(c1), "v"(c2), "v"(c3));
    } else {
        asm volatile("s_nop 1\n\t"
                     "v_fmac_f32_dpp %0, %4, %5 row_newbcast:%9 row_mask:0xf bank_mask:0xf\n\t"
                     "v_fmac_f32_dpp %1, %4, %6 row_newbcast:%10 row_mask:0xf bank_mask:0xf\n\t"
                     "v_fmac_f32_dpp %2, %4, %7 row_newbcast:%11 row_mask:0xf bank_mask:0xf\n\t"
                     "v_fmac_f32_dpp %3, %4, %8 row_newbcast:%12 row_mask:0xf bank_mask:0xf"
                     : "+v"(sa[4 * K]), "+v"(sa[4 * K + 1]), "+v"(sa[4 * K + 2]), "+v"(sa[4 * K + 3])
                     : "v"(dk), "v"(c0), "v"(c1), "v"(c2), "v"(c3), "n"(4 * K), "n"(4 * K + 1), "n"(4 * K + 2), "n"(4 * K + 3));
    }
    __builtin_amdgcn_sched_barrier(0);
}

// LDS row of key k (0..31) of a tile, such that the logits that a lane holds after S^T are those of
// the keys of its operands in P V: 8g .. 8g + 7 (16x16 tiles), 8g .. and 16 + 8g .. (32x32).
template <bool kWide>
__device__ __forceinline__ int key_row(int k) {
    return kWide ? (k & 19) | ((k & 4) << 1) | ((k & 8) >> 1) : 16 * ((k >> 2) & 1) + 4 * (k >> 3) + (k & 3);
}
// V's chunk c of dim d is at c ^ v_swap(d)
template <bool kWide>
__device__ __forceinline__ int v_swap(int d) { return kWide ? ((d >> 1) & 2) | ((d >> 4) & 1) : (d >> 1) & 3; }

// Codes n of the low (bits 0-3, 16-19) or high nibbles (4-7, 20-23) of x as the packed
// fp16 pair n - 8: 0x6400 | n is exactly 1024 + n and 0x6400 | 16 n is 1024 + 16 n; minus
// 1032, or times 1/16 minus 72, is exact.
// `magic` is 0x64006400 in a vector register: with the mask in a scalar one, and and or
// are one instruction (two constants in scalar registers would make them two).
__device__ __forceinline__ uint32_t codes_lo(uint32_t x, uint32_t magic) {
    const uint32_t y = (x & 0x000F000Fu) | magic;
    half2v v;
    __builtin_memcpy(&v, &y, 4);
    v = v + half2v{(_Float16)-1032.0f, (_Float16)-1032.0f};
    uint32_t r;
    __builtin_memcpy(&r, &v, 4);
    return r;
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t x, uint32_t magic) {
    const uint32_t y = (x & 0x00F000F0u) | magic;
    half2v v;
    __builtin_memcpy(&v, &y, 4);
    v = __builtin_elementwise_fma(v, half2v{(_Float16)0.0625f, (_Float16)0.0625f}, half2v{(_Float16)-72.0f, (_Float16)-72.0f});
    uint32_t r;
    __builtin_memcpy(&r, &v, 4);
    return r;
}

// Two 8-byte LDS reads into one MFMA operand. volatile keeps them two single
// ds_read_b64 straight into the operand's registers: merged into ds_read2 pairs
// they would bring halves of different operands and need register moves.
__device__ __forceinline__ half8 lds_half8(const uint8_t *base, int off_lo, int off_hi) {
    typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
    typedef const volatile __attribute__((address_space(3))) u32x2 lds_u32x2;
    const u32x2 a = *(lds_u32x2 *)(base + off_lo);
    const u32x2 b = *(lds_u32x2 *)(base + off_hi);
    const uint4 u = make_uint4(a.x, a.y, b.x, b.y);
    half8 h;
    __builtin_memcpy(&h, &u, 16);
    return h;
}


// The expansion of a tile, K by the 256 lanes of the score and V by those of the value wavefronts,
// in parts that they place between their MFMAs. Stores are 8 bytes, the halves of a 16-byte chunk
// at addresses that differ in bit 3 (which first is a matter of the row: no selects).
//   K: lane takes block b of key k: k & 3, b & 3, k >> 4, b >> 2 from the lane's bits 0-1,
//      2-3, 4, 5, the middle bits of k from the wavefront. Row r = key_row(k) of the
//      stage, chunk 4b + m (dims 32b + 4m + {0, 2, 16, 18, 1, 3, 17, 19}) at
//      (4b + m) ^ (r & 7), halves swapped when r & 8.
//      32x32: k & 3, bit 3 of k, b & 3, b >> 2 from bits 0-1, 2, 3-4, 5, the others from the
//      wavefront; rows of 520 bytes, chunk 4b + m at its place.
//   V: lane takes bytes 4m + 2i, 4m + 2i + 1 of block b's codes for the keys 8c .. 8c + 7
//      (c, i, m from the lane's bits 0-1, 2, 3-4, b = 2w + bit 5) and stores those keys'
//      chunk of the bytes' 4 dims, chunk c of dim d at c ^ v_swap(d), halves
//      swapped when d & 8; odd m the second byte first.
//   V scales: lane takes key lane & 31 of block 2w + (lane >> 5).
// With these maps the 32 lanes that LDS serves at a time store to 32 different pairs of
// banks (lanes over whole rows of K and over all blocks of V met in 16 of them 16 deep:
// 3260 LDS cycles a tile, 56% of them conflicts; now 1800, 27%, of the reads of raw rows).
template <bool kWide>
struct Expand {
    int k_raw, k_sh, k_to, dk_raw, dk_to;   // LDS offsets in the first of two buffers
    int v_raw, v_to, v_odd, dv_raw, dv_to, dv_key;
    uint32_t x[4], k[5], d, dk, magic;
    __device__ __forceinline__ void init(int w, int lane) {
        const int key = kWide ? 16 * (w >> 1) + 8 * ((lane >> 2) & 1) + 4 * (w & 1) + (lane & 3) : 16 * ((lane >> 4) & 1) + 4 * w + (lane & 3);
        const int kb = 4 * (lane >> 5) + ((lane >> (kWide ? 3 : 2)) & 3), r = key_row<kWide>(key);
        dk_raw = kLdsRaw + kHeadRowBytes * key + 18 * kb;
        k_raw = kLdsRaw + kHeadRowBytes * key + ((18 * kb + 2) & ~3);  // the codes start 2 bytes off a dword for even blocks
        k_sh = kb & 1 ? 0 : 16;
        k_to = kWide ? r * kWideRow + 64 * kb : r * 512 + 16 * ((4 * kb) ^ (r & 7)) + (r & 8);
        dk_to = kOffDk + (kWide ? key * 8 + kb : kb * kPK + r) * 2;
        const int c = lane & 3, i = (lane >> 2) & 1, m = (lane >> 3) & 3, b = 2 * w + (lane >> 5);
        v_raw = kLdsRaw + 2 * kRawTile + kHeadRowBytes * 8 * c + 18 * b + 2 + 4 * m + 2 * i;
        const int dim = 32 * b + 4 * m + 2 * i;
        v_to = kLdsV + 64 * dim + 16 * (c ^ v_swap<kWide>(dim)) + (dim & 8);
        v_odd = m & 1;
        dv_key = lane & 31;
        dv_raw = kLdsRaw + 2 * kRawTile + kHeadRowBytes * dv_key + 18 * b;
        dv_to = kLdsV + kOffDv + 64 * b + 2 * dv_key;
        magic = 0x64006400u;
        asm volatile("" : "+v"(magic));
    }
    // reads of V tile t
    __device__ __forceinline__ void read_v(const uint8_t *smem, int t) {
        const uint8_t *src = smem + v_raw + (t & 1) * kRawTile;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            x[j] = (uint32_t)*reinterpret_cast<const uint16_t *>(src + kHeadRowBytes * 2 * j) |
                   ((uint32_t)*reinterpret_cast<const uint16_t *>(src + kHeadRowBytes * (2 * j + 1)) << 16);
        d = *reinterpret_cast<const uint16_t *>(smem + dv_raw + (t & 1) * kRawTile);
    }
    // reads of K tile t
    __device__ __forceinline__ void read_k(const uint8_t *smem, int t) {
        const uint32_t *src = reinterpret_cast<const uint32_t *>(smem + k_raw + (t & 1) * kRawTile);
#pragma unroll
        for (int m = 0; m < 5; ++m) k[m] = src[m];
        dk = *reinterpret_cast<const uint16_t *>(smem + dk_raw + (t & 1) * kRawTile);
    }
    // byte j of the lane's two (odd m: the other one), both nibbles
    __device__ __forceinline__ void store_v(uint8_t *smem, int t, int j) {
        const int byte = v_odd ^ j, to = v_to + (t & 1) * kVStage + 64 * byte;
        uint32_t y[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) y[q] = x[q] >> (8 * byte);
        *reinterpret_cast<uint2 *>(smem + to) = make_uint2(codes_lo(y[0], magic), codes_lo(y[1], magic));
        *reinterpret_cast<uint2 *>(smem + (to ^ 8)) = make_uint2(codes_lo(y[2], magic), codes_lo(y[3], magic));
        const int hi = (kWide ? to ^ 16 : to) + 1024;  // dims 16 further
        *reinterpret_cast<uint2 *>(smem + hi) = make_uint2(codes_hi(y[0], magic), codes_hi(y[1], magic));
        *reinterpret_cast<uint2 *>(smem + (hi ^ 8)) = make_uint2(codes_hi(y[2], magic), codes_hi(y[3], magic));
    }
    // chunk m of the lane's block
    __device__ __forceinline__ void store_k(uint8_t *smem, int t, int m) {
        const int at = k_to + (t & 1) * kKStage, to = kWide ? at + 16 * m : at ^ (16 * m);
        const uint32_t y = __builtin_amdgcn_alignbit(k[m + 1], k[m], (uint32_t)k_sh), z = y >> 8;
        if (m == 0) *reinterpret_cast<uint16_t *>(smem + dk_to + (t & 1) * kKStage) = (uint16_t)dk;
        *reinterpret_cast<uint2 *>(smem + to) = make_uint2(codes_lo(y, magic), codes_hi(y, magic));
        *reinterpret_cast<uint2 *>(smem + (kWide ? to + 8 : to ^ 8)) = make_uint2(codes_lo(z, magic), codes_hi(z, magic));
    }
    // V scales of tile t as d_v 2^e (two blocks of this wavefront), 0 for keys at or past
    // `left`, on pages that are not there, and for NaN or Inf (bytes that are no q4_0):
    // their P is 0, and 0 * NaN would not be. Returns e: at most the one given, and such
    // that the largest is below 1.
    __device__ __forceinline__ int scales_v(uint8_t *smem, int t, int left, bool has_a, bool has_b, int e) {
        const bool ok = dv_key < left && (dv_key < 16 ? has_a : has_b) && (d & 0x7C00u) != 0x7C00u;
        d = ok ? d : 0u;
        // fp16 bits of 2^-e, the smallest scale that would reach 1 (e in [-17, 24])
        const uint32_t over = e <= 14 ? (uint32_t)(15 - e) << 10 : 1u << (24 - e);
        if (e == kMaxE || __any((d & 0x7fffu) >= over)) {
            const int mx = wave_max((int)(d & 0x7fffu));
            if (mx != 0) {
                const int ex = mx >> 10;
                const int lg = ex ? ex - 15 : (31 - __builtin_clz(mx)) - 24;  // floor(log2 max |d_v|)
                e = min(e, -1 - lg);
            }
        }
        const uint16_t bits = (uint16_t)d;
        _Float16 h;
        __builtin_memcpy(&h, &bits, 2);
        *reinterpret_cast<_Float16 *>(smem + dv_to + (t & 1) * kVStage) = (_Float16)__builtin_amdgcn_ldexpf((float)h, e);
        return e;
    }
};

// Q' of a row as B operands: the lane's 8 dims of every block (in the order of the K
// chunks), q8_0 with ggml's x86 rounding (d = amax / 127 over the block, codes =
// rint(x * 127 / amax)), times fp16(d) * scale * log2(e) in fp32, as fp16 hi and
// lo = fp16(Q' - hi). The loads of a row are one batch (block by block they were 16
// memory latencies at the start of every workgroup).
template <bool kWide>
struct QRow {
    static constexpr int kC = kWide ? 2 : 1;  // chunks of 8 dims of a block that a lane holds: g, or g and 2 + g
    float4a v[16 * kC];
    __device__ __forceinline__ void load(const Call &p, int64_t row, int h, int g) {
        const float *q = reinterpret_cast<const float *>(p.q + row * p.q_nb1 + (int64_t)h * p.q_nb2) + 4 * g;
#pragma unroll
        for (int b = 0; b < 8 * kC; ++b)
#pragma unroll
            for (int k = 0; k < 2; ++k) v[2 * b + k] = *reinterpret_cast<const float4a *>(q + 32 * (b / kC) + 8 * (b % kC) + 16 * k);
    }
    __device__ __forceinline__ void quantize(float qscale, bool ok, half8 (&hi)[8 * kC], half8 (&lo)[8 * kC]) const {
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            float amax = 0.0f;
#pragma unroll
            for (int k = 2 * kC * b; k < 2 * kC * (b + 1); ++k)
                amax = fmaxf(fmaxf(fmaxf(amax, fabsf(v[k].x)), fmaxf(fabsf(v[k].y), fabsf(v[k].z))), fabsf(v[k].w));
            amax = xmax32(kWide ? amax : xmax16(amax));
            const float d = amax / 127.f;
            const float id = amax != 0.0f ? 127.f / amax : 0.0f;
            const float qd = ok ? (float)(_Float16)d * qscale : 0.0f;
#pragma unroll
            for (int c = kC * b; c < kC * (b + 1); ++c) {
                const float4a u = v[2 * c], w = v[2 * c + 1];
                const float x[8] = {u.x, u.z, w.x, w.z, u.y, u.w, w.y, w.w};
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    // y opaque: left visible, the compiler may round code * qd to fp16 twice
                    // (once from the fp32 product for hi, once from the exact product for the
                    // hi it subtracts), and a hi + lo off by one fp16 ulp of hi
                    y[j] = rintf(x[j] * id) * qd;
                    asm volatile("" : "+v"(y[j]));
                    hi[c][j] = (_Float16)y[j];
                }
                uint32_t hw[4];
                __builtin_memcpy(hw, &hi[c], 16);
#pragma unroll
                for (int j = 0; j < 8; ++j) {  // the exact residual, hi read from its packed half
                    float r;
                    if (j & 1)
                        asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "=v"(r) : "v"(y[j]), "v"(hw[j >> 1]));
                    else
                        asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,0] op_sel_hi:[0,0,1]" : "=v"(r) : "v"(y[j]), "v"(hw[j >> 1]));
                    lo[c][j] = (_Float16)r;
                }
            }
        }
    }
};

// ---------------------------------------------------------------- work split

template <class C>
__device__ __forceinline__ Item many_item(const C &c, int lin, int qb) {
    Item it{};
    const Work w = *reinterpret_cast<const Work *>(c.work);
    it = reinterpret_cast<const Item *>(c.work + kListAt)[min(lin, kListed - 1)];  // beside it, used if there is a list
    const int len = uniform(w.len), items = uniform(w.items);
    const int id = uniform(w.even) ? id_of_workgroup(lin, items) : lin < items ? lin : -1;
    if (id < 0 || uniform(w.listed)) {
        if (id < 0) it.b = -1;
        return it;
    }
    // the last request whose first item is at most id: 64 at a time
    const int *first = c.work + kFirstAt, *slot = first + entries(c) + 1, lane = threadIdx.x & 63;
    int lo = 0, hi = entries(c);
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) / 64, at = lo + lane * step;
        const uint64_t below = __ballot(at < hi && first[min(at, entries(c))] <= id);
        const int l = 63 - __builtin_clzll(below);  // lane 0 is always below
        lo = uniform(lo + l * step);
        hi = uniform(min(hi, lo + step));
    }
    it.b = lo;
    it.rq = uniform_request(c, lo);
    int kt;
    it.tiles = uniform(chunk_tiles(c, it.rq, qb, &kt));
    it.splits = uniform(div_ceil(kt, len));
    const int k = id - uniform(first[lo]), q = uniform(div_floor(k, it.tiles));
    it.tile = k - q * it.tiles;
    it.kvh = uniform(div_floor(q, it.splits));
    it.split = q - it.kvh * it.splits;
    split_range(kt, it.splits, it.split, &it.t0, &it.t1);
    it.slot = slot[lo];
    return it;
}

// kRG = 2: 128 query rows a workgroup; 1: 64 rows. OPT: the logits are capped or biased. C: Call,
// or Parts, where a tile's tokens may be members of a group.
template <int kRG, bool OPT, class C>
__global__ __launch_bounds__(kThreads, 1) void paged_many_kernel(C p) {
    constexpr bool kPart = kIsParts<C>;
    constexpr bool kWide = kRG == 2;
    constexpr int kN = 16 * kRG;          // rows of a wave, a lane's column of the matrix tiles
    constexpr int kV = 8 * kRG;           // keys of its row that a lane holds, 8 g .. 8 g + 7 (+ 16)
    constexpr int kT = kHeadDim / kN;     // matrix tiles of O
    constexpr int kR = kWide ? 16 : 4;    // rows of O that a lane holds
    typedef float Tile __attribute__((ext_vector_type(kWide ? 16 : 4)));
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63, g = lane / kN, n = lane % kN;
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem;

    const int qb = uniform(group_of(p, rows_per_wg(kRG)));  // tokens of a query tile
    Item it = many_item(p, (int)blockIdx.x, qb);
    if (uniform(it.b) < 0) return;
    for (int *x : {&it.b, &it.kvh, &it.tile, &it.tiles, &it.split, &it.splits, &it.t0, &it.t1, &it.slot}) *x = uniform(*x);
    const Request rq{uniform(it.rq.q0), uniform(it.rq.n), uniform(it.rq.kv), uniform(it.rq.pos0), uniform(it.rq.prefix)};
    const int q_base = it.tile * qb;        // its first token in the request
    const int q_top = min(q_base + qb, rq.n);
    const bool shared = is_group(p, it.b);
    const bool whole = !shared && it.splits == 1;  // of the keys: the result goes out from here
    const int slot = it.slot + (it.kvh * it.splits + it.split) * it.tiles + it.tile;
    int own_row = 0;
    if (it.split == 0 && it.kvh == 0 && tid < q_top - q_base && (own_row = row_of_token(p, rq, shared, q_base + tid)) >= 0) {
        int4 *where = p.where;
        if constexpr (kPart) where = shared ? p.g_where : where;
        where[own_row] =
            whole ? make_int4(0, 0, 0, kPart ? kWhole : kDone) : make_int4(it.slot + it.tile, it.splits, tid * p.G, 4 * it.tiles + kMany);
    }

    // Key range: the split, cut at the last key any token of the tile sees.
    const int k_begin = it.t0 * kPK;
    const int k_end = min(it.t1 * kPK, sees(rq, q_top - 1));
    const int n_tiles = uniform(k_end > k_begin ? (k_end - k_begin + kPK - 1) / kPK : 0);
    if (n_tiles == 0 && !whole) {
        // a split past the tile's last visible key leaves its O unwritten: the
        // merge takes no partial whose m is -inf
        if (tid < rows_per_wg(kRG)) {
            float *ml = p.ml_c + ((int64_t)slot * rows_per_wg(kRG) + tid) * 2;
            store_through(ml, -INFINITY);
            store_through(ml + 1, 0.0f);
        }
        return;
    }
    const int kvh = it.kvh;
    const int see_all = sees(rq, q_base);  // keys that every token of the tile sees
    const TableRow table = table_row(p, it.b);
    const int last_group = max(rq.kv - 1, 0) & ~15;
    // 16-key group gi of tile t; one behind the last key stands for the last one
    // Tiles in order, with a bias the last first: the logits grow towards the token, and
    // every tile in order would move the maximum.
    const bool back = OPT && p.bias != 0.0f;
    auto tile_at = [&](int t) { return back ? n_tiles - 1 - t : t; };
    auto group_key = [&](int t, int gi) {
        return __builtin_amdgcn_readfirstlane(min(k_begin + tile_at(t) * kPK + 16 * gi, last_group));
    };
    auto id_of = [&](int t, int gi) { return t < n_tiles ? page_id(table, group_key(t, gi) >> p.lp) : 0; };
    auto there = [&](int id) { return (uint32_t)id < (uint32_t)p.n_pages; };

    const float lim_top = (float)(kSlack + kEp);  // the lazy test's bound on s'
    const int nh = (n >> 3) & 1;

    // The two kinds of wave run separate code with the same barrier count:
    // one before the loop, n_tiles + 1 in it, then two for the hand-over of m and l.
    if (wave < kScoreWaves) {
        const int w = wave;
        float *ml = reinterpret_cast<float *>(smem + kLdsP) + w * (kN * 2);  // [row][m, l]
        // Q' hi and lo of row r = kN w + n (position q_base + r / G, head kvh*G + r % G) as B
        // operands: chunk g of every block, or chunks g and 2 + g
        half8 bqh[8 * kRG], bql[8 * kRG];
        const int r = kN * w + n, i_tok = group_of(p, r), h = kvh * p.G + r - i_tok * p.G;
        const bool ok = q_base + i_tok < q_top;
        const int my_see = ok ? sees(rq, q_base + i_tok) : 0;
        int my_pos = rq.pos0 + q_base + i_tok;
        const float my_slope = OPT && p.bias != 0.0f ? slope2(p, h) : 0.0f;
        // The logits are accumulated relative to the row's P reference mref =
        // (m_run, or 0 before the first visible key) - ep: s' = s - mref, so that
        // P = 2^s' needs no subtraction, and the lazy-maximum test s > m_run +
        // ks reads s' > lim_s (ks + ep, or -inf before the first visible key).
        // Both change only when the maximum moves.
        float m_run = -INFINITY, l_part = 0.0f, mref = -(float)kEp, lim_s = -INFINITY;
        {
            const int row = ok ? row_of_token(p, rq, shared, q_base + i_tok) : kPart ? 0 : rq.q0;
            if constexpr (kPart && OPT)
                if (shared) my_pos = ok ? p.m_pos[rq.q0 + q_base + i_tok] : 0;
            QRow<kWide> q;
            q.load(p, kPart ? max(row, 0) : row, h, g);
            __builtin_amdgcn_sched_barrier(0);  // the loads stay together
            // raw rows of the first tile: the value waves expand them while Q is quantized
            if (n_tiles > 0) asm volatile("s_barrier" ::: "memory");
            q.quantize(p.qscale, ok, bqh, bql);
        }
        // 16x16: K operand of key row 16kg + n, chunk (4b + g) ^ (n & 7), halves swapped when n & 8;
        // the XOR touches bit 2 of 4b + g, so even and odd b use two bases and b >> 1 adds 128 bytes.
        // 32x32: row n, chunks 4b + g and 4b + 2 + g, one base.
        int k_off[2][2];  // [b & 1][half]
#pragma unroll
        for (int bp = 0; bp < 2; ++bp)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
                k_off[bp][hf] = kWide ? n * kWideRow + 16 * g : n * 512 + 16 * ((4 * bp + g) ^ (n & 7)) + 8 * (hf ^ nh);
        const int p_off = w * (kRG * 2048) + 16 * lane;  // P slots [w][8 keys][hi, lo][lane]
        const int dk_off = kOffDk + 16 * (16 * ((lane >> 3) & 1) + 8 * g + (lane & 7));
        Expand<kWide> ex;
        ex.init(w, lane);

        int ida = id_of(0, 0), idb = id_of(0, 1);  // pages of the tile's two groups
        for (int t = 0; t <= n_tiles && n_tiles > 0; ++t) {
            // the value waves wait for their DMAs before this barrier, which makes them
            // visible and retires the buffers the new ones overwrite
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (t == n_tiles) break;
            const int kt = k_begin + tile_at(t) * kPK;
            const bool has_a = there(ida), has_b = there(idb);
            ida = id_of(t + 1, 0);
            idb = id_of(t + 1, 1);
            // this tile's per-lane K bases, opaque to the compiler: every K read
            // is then one of them plus an immediate offset (hoisting all 64
            // base + offset sums out of the loop would need 64 more registers)
            int kb[2][2];
#pragma unroll
            for (int bp = 0; bp < (kWide ? 1 : 2); ++bp)
#pragma unroll
                for (int hf = 0; hf < (kWide ? 1 : 2); ++hf) {
                    kb[bp][hf] = (t & 1) * kKStage + k_off[bp][hf];
                    asm volatile("" : "+v"(kb[bp][hf]));
                }
            // ---- S^T: the logits of the lane's keys in s --------------------------------
            // K of a step is on its way while the one before multiplies (read at its start, every step
            // waited for LDS: 2% more). The d_k scaling of a step runs while the next one's MFMAs execute;
            // the scheduling barriers keep the compiler from pulling it back next to the MFMAs it reads (it
            // did, leaving 4-12 instructions between an MFMA and its consumer).
            const float start = OPT && p.cap2 != 0.0f ? 0.0f : -mref;
            float s[kV];  // base-2 logits
            if constexpr (kWide) {
                // a step is a block: two chunks, hi and lo, on one sum
                float sa[16];
                Tile cp;
#pragma unroll
                for (int i = 0; i < 16; ++i) sa[i] = start;
                // d_k of all blocks, the lane's key that of value lane & 15: the sums take it from there
                half8 an[2], dkh;
                float dk[8];
                auto load = [&](int b) {
#pragma unroll
                    for (int m = 0; m < 2; ++m)
                        an[m] = lds_half8(smem, kb[0][0] + 64 * b + 32 * m, kb[0][0] + 64 * b + 32 * m + 8);
                };
                load(0);
                dkh = *reinterpret_cast<const half8 *>(smem + (t & 1) * kKStage + dk_off);
#pragma unroll
                for (int b = 0; b <= 8; ++b) {
                    Tile c = 0.0f;
                    half8 a0, a1;
                    if (b < 8) {
                        a0 = an[0], a1 = an[1];
                        if (b < 7) load(b + 1);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    // between two MFMAs four of the sums of the block before
                    auto step = [&](auto k_) {
                        constexpr int k = decltype(k_)::value;
                        if (b < 8) c = __builtin_amdgcn_mfma_f32_32x32x16_f16(k < 2 ? a0 : a1, (k & 1 ? bql : bqh)[2 * b + (k >> 1)], c, 0, 0, 0);
                        __builtin_amdgcn_sched_barrier(0);
                        if (b > 0) add_scaled<k>(sa, cp[4 * k], cp[4 * k + 1], cp[4 * k + 2], cp[4 * k + 3], dk[b - 1]);
                    };
                    step(std::integral_constant<int, 0>{});
                    step(std::integral_constant<int, 1>{});
                    step(std::integral_constant<int, 2>{});
                    step(std::integral_constant<int, 3>{});
                    if (b == 0) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            dk[i] = (float)dkh[i];
                            asm volatile("" : "+v"(dk[i]));
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    cp = c;
                    // the expansion of the next K tile goes between the MFMAs (the value waves do the first)
                    if (b == 0) ex.read_k(smem, t + 1);
                    if (b >= 4 && b < 8) ex.store_k(smem, t + 1, b - 4);
                }
#pragma unroll
                for (int jj = 0; jj < kV; ++jj) s[jj] = sa[jj];
            } else {
                // step j is (block j >> 1, key group j & 1): sa[kg][i] of key 8g + 4kg + i
                Tile sa[2];
                sa[0] = sa[1] = start;
                // d_k of the lane's four C rows 16kg + 4g + i, block b: 8 bytes at Dk[b][16kg + 4g]
                const uint8_t *dkb = smem + (t & 1) * kKStage + kOffDk + 8 * g;
                Tile cp;
                uint2 dkp, dkn;
                half8 akn;
                auto load = [&](int j) {
                    const int b = j >> 1, kg = j & 1, o = kg * 8192 + 128 * (b >> 1);
                    akn = lds_half8(smem, kb[b & 1][0] + o, kb[b & 1][1] + o);
                    dkn = *reinterpret_cast<const uint2 *>(dkb + 64 * b + 32 * kg);
                };
                load(0);
#pragma unroll
                for (int j = 0; j <= 16; ++j) {
                    Tile cn;
                    uint2 dkj;
                    if (j < 16) {
                        const int b = j >> 1;
                        const half8 ak = akn;
                        dkj = dkn;
                        if (j < 15) load(j + 1);
                        __builtin_amdgcn_sched_barrier(0);
                        cn = __builtin_amdgcn_mfma_f32_16x16x32_f16(ak, bqh[b], Tile(0.0f), 0, 0, 0);
                        cn = __builtin_amdgcn_mfma_f32_16x16x32_f16(ak, bql[b], cn, 0, 0, 0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    if (j > 0) {
                        const int kg = (j - 1) & 1;
                        _Float16 dk[4];
                        __builtin_memcpy(dk, &dkp, 8);
#pragma unroll
                        for (int i = 0; i < 4; ++i) sa[kg][i] = fmaf(cp[i], (float)dk[i], sa[kg][i]);
                    }
                    if (j < 16) dkp = dkj, cp = cn;
                    if (j == 0) ex.read_k(smem, t + 1);
                    if (j >= 8 && j < 16 && j % 2 == 0) ex.store_k(smem, t + 1, (j - 8) / 2);
                }
#pragma unroll
                for (int jj = 0; jj < kV; ++jj) s[jj] = sa[jj >> 2][jj & 3];
            }
            if (OPT || kWide) {
                // the scaled sums before what follows (the compiler moved some behind the cap, and
                // kept 64 products alive till there)
#pragma unroll
                for (int jj = 0; jj < kV; ++jj) asm volatile("" : "+v"(s[jj]));
                __builtin_amdgcn_sched_barrier(0);
            }
            if (OPT) {
#pragma unroll
                for (int u = 0; u < kRG; ++u) {  // eight by eight: all at once need more registers than there are
                    float (&x)[8] = *reinterpret_cast<float (*)[8]>(s + 8 * u);
                    if (p.cap2 != 0.0f) cap_logits(x, p.cap2, p.cap_inv, -mref);
                    if (p.bias != 0.0f) {
                        const float far = (float)(my_pos - (kt + 16 * u + 8 * g));
#pragma unroll
                        for (int jj = 0; jj < 8; ++jj) x[jj] = fmaf(-my_slope, fabsf(far - (float)jj), x[jj]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            // ---- causal limit, prefix, last key, pages that are not there: whatever the
            // logit is, NaN of garbage bytes too
            if (kt + kPK > see_all || !has_a || !has_b) {
#pragma unroll
                for (int u = 0; u < kRG; ++u) {
                    const bool has = (kWide ? u == 0 : g < 2) ? has_a : has_b;
                    const int see = has ? min(my_see, k_end) - (kt + 16 * u + 8 * g) : 0;
#pragma unroll
                    for (int jj = 0; jj < 8; ++jj) s[8 * u + jj] = jj < see ? s[8 * u + jj] : -INFINITY;
                }
            }
            // ---- online softmax (base 2); P and the rescale factors to LDS -----------
            uint8_t *pb = smem + kLdsP + (t & 1) * kPBuf + p_off;
            float *ab = reinterpret_cast<float *>(smem + kLdsA + (t & 1) * kABuf) + w * kN;
            // lazy maximum: the reference moves only when a logit passes it by more
            // than ks, so P <= 2^ks and most tiles need no rescale of O
            float alpha = 1.0f;
            int moved = 0;
            bool over = false;
#pragma unroll
            for (int jj = 0; jj < kV; ++jj) over |= s[jj] > lim_s;
            if (__any(over)) {
                float mt = s[0];
#pragma unroll
                for (int jj = 1; jj < kV; ++jj) mt = fmaxf(mt, s[jj]);
                if (!kWide) mt = xmax16(mt);
                mt = xmax32(mt);
                const float m_new = fmaxf(m_run, mt + mref);
                alpha = m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - m_new);
                l_part *= alpha;
                moved = 1;
                m_run = m_new;
                // onto the new reference: s - mref_new = s' + (mref - mref_new)
                const float mref_new = (m_new == -INFINITY ? 0.0f : m_new) - (float)kEp;
                const float d = mref - mref_new;
#pragma unroll
                for (int jj = 0; jj < kV; ++jj) s[jj] += d;
                mref = mref_new;
                lim_s = m_new == -INFINITY ? -INFINITY : lim_top;
            }
#pragma unroll
            for (int u = 0; u < kRG; ++u) {
                float pf[8], psum = 0.0f;
#pragma unroll
                for (int jj = 0; jj < 8; ++jj) {
                    pf[jj] = __builtin_amdgcn_exp2f(s[8 * u + jj]);
                    psum += pf[jj];
                }
                l_part += psum;
                // P as an fp16 hi + lo pair (22 bits): the value waves form P d_v from it
                half8 ph, pl;
#pragma unroll
                for (int jj = 0; jj < 8; ++jj) ph[jj] = (_Float16)pf[jj];
                // the exact residual p - hi, with hi read from its packed fp16 half by
                // v_fma_mix (no conversion of hi back to fp32)
                uint32_t hw[4];
                __builtin_memcpy(hw, &ph, 16);
#pragma unroll
                for (int jj = 0; jj < 8; ++jj) {
                    float x;
                    if (jj & 1)
                        asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "=v"(x) : "v"(pf[jj]), "v"(hw[jj >> 1]));
                    else
                        asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,0] op_sel_hi:[0,0,1]" : "=v"(x) : "v"(pf[jj]), "v"(hw[jj >> 1]));
                    pl[jj] = (_Float16)x;
                }
                *reinterpret_cast<half8 *>(pb + u * 2048) = ph;
                *reinterpret_cast<half8 *>(pb + u * 2048 + 1024) = pl;
            }
            if (g == 0) ab[n] = alpha;
            if (lane == 0) *reinterpret_cast<int *>(smem + kLdsF + 16 * (t & 1) + 4 * w) = moved;
        }
        // ---- hand m and l of the rows to the value waves ----------------------------
        __syncthreads();
        if (n_tiles > 0) {
            if (!kWide) l_part += __shfl_xor(l_part, 16);
            l_part += __shfl_xor(l_part, 32);
            if (g == 0) {
                ml[2 * n] = m_run;
                ml[2 * n + 1] = l_part;
            }
        }
        __syncthreads();
        return;
    }

    // ---- value waves: O[row kN w + 8 (k >> 2) + 4g + (k & 3)][dim kN T + n] in acc[T][k] ----------
    const int w = wave - kScoreWaves;
    const float *ml = reinterpret_cast<const float *>(smem + kLdsP) + w * (kN * 2);  // [row][m, l]
    // V operand of dim kN T + n, keys 8g..8g+7: chunk g ^ v_swap, halves swapped when n & 8; of keys
    // 16 + 8g..: chunk 2 + g
    int v_off[kRG][2];
#pragma unroll
    for (int u = 0; u < kRG; ++u)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) v_off[u][hf] = 64 * n + 16 * ((2 * u + g) ^ v_swap<kWide>(n)) + 8 * (hf ^ nh);
    const int p_off = w * (kRG * 2048) + 16 * lane;
    // DMA: wave w moves 16 rows of a tile, group w & 1, of K (w < 2) or V. They lie on
    // one page: 9 x 16 bytes a row as two instructions of 64 lanes and one of 16.
    uint32_t off[3];
#pragma unroll
    for (int r = 0; r < 3; ++r) {
        const int s = 64 * r + lane;
        off[r] = (uint32_t)(s / 9) * (uint32_t)p.row_bytes + (uint32_t)(kvh * kHeadRowBytes + 16 * (s % 9));
    }
    const uint8_t *pool = w < 2 ? p.k : p.v;
    const int64_t page_bytes = w < 2 ? p.k_page : p.v_page;
    auto issue = [&](int t, int id) {
        const int key = group_key(t, w & 1);
        const uint8_t *from = pool + (int64_t)(there(id) ? id : 0) * page_bytes + (int64_t)(key & (p.page - 1)) * p.row_bytes;
        const uint32_t to = lds0 + (uint32_t)(kLdsRaw + (2 * (w >> 1) + (t & 1)) * kRawTile + (w & 1) * (kRawTile / 2));
        // rows behind the last key re-read the end of its row
        const uint32_t lim = (uint32_t)(min(rq.kv - key, 16) * p.row_bytes - 16);
        dma16(min(off[0], lim), from, to);
        dma16(min(off[1], lim), from, to + 1024);
        if (lane < 16) dma16(min(off[2], lim), from, to + 2048);
    };
    // ids of the groups of tiles t, t + 1, t + 2
    int a0 = id_of(0, 0), b0 = id_of(0, 1), a1 = id_of(1, 0), b1 = id_of(1, 1), a2 = id_of(2, 0), b2 = id_of(2, 1);
    auto mine = [&](int a, int b) { return w & 1 ? b : a; };
    Expand<kWide> ex;
    ex.init(w, lane);
    int e_own = kMaxE;                            // of this wavefront's pair of blocks, up to the tile expanded last
    int4 e_acc = make_int4(kMaxE, kMaxE, kMaxE, kMaxE);  // of O's pairs
    auto scales = [&](int t, int a, int b) {
        e_own = ex.scales_v(smem, t, k_end - (k_begin + tile_at(t) * kPK), there(a), there(b), e_own);
        if (lane == 0) *reinterpret_cast<int *>(smem + kLdsE + 16 * (t & 1) + 4 * w) = e_own;
    };
    if (n_tiles > 0) {
        issue(0, mine(a0, b0));
        if (w < 2 && n_tiles > 1) issue(1, mine(a1, b1));
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        ex.read_k(smem, 0);
#pragma unroll
        for (int m = 0; m < 4; ++m) ex.store_k(smem, 0, m);
        ex.read_v(smem, 0);
        scales(0, a0, b0);
        ex.store_v(smem, 0, 0);
        ex.store_v(smem, 0, 1);
    }
    Tile acc[kT];
#pragma unroll
    for (int T = 0; T < kT; ++T) acc[T] = 0.0f;
    // (behind the last tile the expansion works on bytes that are there, into stages that
    // nobody reads any more)
    for (int t = 0; t <= n_tiles && n_tiles > 0; ++t) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int a3 = id_of(t + 3, 0), b3 = id_of(t + 3, 1);
        if (w < 2) {
            if (t + 2 < n_tiles) issue(t + 2, mine(a2, b2));
        } else {
            if (t + 1 < n_tiles) issue(t + 1, mine(a1, b1));
        }
        const int x0 = a0, y0 = b0;
        a0 = a1, b0 = b1, a1 = a2, b1 = b2, a2 = a3, b2 = b3;
        if (t == 0) continue;
        const int tp = t - 1;
        const uint8_t *vs = smem + kLdsV + (tp & 1) * kVStage;
        // this tile's per-lane V bases, opaque to the compiler (see the K reads)
        int vb[kRG][2];
#pragma unroll
        for (int u = 0; u < kRG; ++u)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                vb[u][hf] = kLdsV + (tp & 1) * kVStage + v_off[u][hf];
                asm volatile("" : "+v"(vb[u][hf]));
            }
        const uint8_t *pb = smem + kLdsP + (tp & 1) * kPBuf + p_off;
        const float *ab = reinterpret_cast<const float *>(smem + kLdsA + (tp & 1) * kABuf) + w * kN + 4 * g;
        // O onto the exponents of this tile's V scales where a larger one has come
        int4 e_t = *reinterpret_cast<const int4 *>(smem + kLdsE + 16 * (tp & 1));
        e_t.x = __builtin_amdgcn_readfirstlane(e_t.x), e_t.y = __builtin_amdgcn_readfirstlane(e_t.y);
        e_t.z = __builtin_amdgcn_readfirstlane(e_t.z), e_t.w = __builtin_amdgcn_readfirstlane(e_t.w);
        half8 ph[kRG], pl[kRG];  // of the lane's row n
        const int resc = __builtin_amdgcn_readfirstlane(*reinterpret_cast<const int *>(smem + kLdsF + 16 * (tp & 1) + 4 * w));
#pragma unroll
        for (int u = 0; u < kRG; ++u) {
            ph[u] = *reinterpret_cast<const half8 *>(pb + u * 2048);
            pl[u] = *reinterpret_cast<const half8 *>(pb + u * 2048 + 1024);
        }
        if (resc) {  // rare with the lazy maximum: O = alpha O, alpha of rows 8q + 4g .. + 3
#pragma unroll
            for (int q = 0; q < kR / 4; ++q) {
                const floatx4 a4 = *reinterpret_cast<const floatx4 *>(ab + 8 * q);
#pragma unroll
                for (int T = 0; T < kT; ++T)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[T][4 * q + i] *= a4[i];
            }
        }
        if ((e_t.x ^ e_acc.x) | (e_t.y ^ e_acc.y) | (e_t.z ^ e_acc.z) | (e_t.w ^ e_acc.w)) {
            const int from[4] = {e_acc.x, e_acc.y, e_acc.z, e_acc.w}, to[4] = {e_t.x, e_t.y, e_t.z, e_t.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float f = __builtin_amdgcn_ldexpf(1.0f, to[q] - from[q]);
#pragma unroll
                for (int T = kT / 4 * q; T < kT / 4 * (q + 1); ++T) acc[T] *= f;
            }
            e_acc = e_t;
        }
        // d_v and V of block b + 1 are read while block b computes: the LDS latency stays
        // off the MFMA chain. Between the blocks, parts of the next tiles' expansion.
        half8 dvn[kRG], bvn[2];
        auto load = [&](int b) {
#pragma unroll
            for (int u = 0; u < kRG; ++u) dvn[u] = *reinterpret_cast<const half8 *>(vs + kOffDv + 64 * b + 32 * u + 16 * g);
#pragma unroll
            for (int k = 0; k < 2; ++k) {  // the block's 32 dims for 16 keys each, or two times 16 dims
                const int u = kWide ? k : 0, o = 2048 * b + (kWide ? 0 : 1024 * k);
                bvn[k] = lds_half8(smem, vb[u][0] + o, vb[u][1] + o);
            }
        };
        load(0);
        ex.read_v(smem, t);
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const half8 bv[2] = {bvn[0], bvn[1]};
            half8 dv[kRG];
#pragma unroll
            for (int u = 0; u < kRG; ++u) dv[u] = dvn[u];
            if (b < 7) load(b + 1);
            // A = P 2^ep d_v as an fp16 hi + lo pair (22 bits): the products with the
            // exact V codes are then exact in fp32, so a row that a few keys
            // dominate carries no fp16 rounding of P d_v into its output. Ph d_v has
            // at most 22 significant bits, so its residual after rounding to fp16
            // (at most 11 bits) is exact in one fma; Pl d_v is 2^-11 of it and
            // rounds once.
            half8 ah[kRG], al[kRG];
#pragma unroll
            for (int u = 0; u < kRG; ++u) {
                ah[u] = ph[u] * dv[u];
                const half8 x = __builtin_elementwise_fma(ph[u], dv[u], -ah[u]);
                al[u] = __builtin_elementwise_fma(pl[u], dv[u], x);
            }
            if constexpr (kWide) {
                acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[0], bv[0], acc[b], 0, 0, 0);
                acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[1], bv[1], acc[b], 0, 0, 0);
                acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[0], bv[0], acc[b], 0, 0, 0);
                acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[1], bv[1], acc[b], 0, 0, 0);
            } else {
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) acc[2 * b + hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah[0], bv[hf], acc[2 * b + hf], 0, 0, 0);
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) acc[2 * b + hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(al[0], bv[hf], acc[2 * b + hf], 0, 0, 0);
            }
            if (b == 1) scales(t, x0, y0);
            if (b == 2) ex.store_v(smem, t, 0);
            if (b == 3) ex.store_v(smem, t, 1);
        }
    }
    __syncthreads();  // m and l of the rows ...
    __syncthreads();  // ... are in LDS
    const int e_out[4] = {-e_acc.x, -e_acc.y, -e_acc.z, -e_acc.w};
    // the lane's rows, one after the other; the gate of the next one is on its way while a row goes out
    auto row_at = [&](int k) { return 8 * (k >> 2) + 4 * g + (k & 3); };
    auto token_of = [&](int k, int *h) {
        const int r = kN * w + row_at(k), tok = group_of(p, r);
        *h = kvh * p.G + r - tok * p.G;
        return q_base + tok;
    };
    float *dst = p.dst;
    if constexpr (kPart) dst = p.whole;
    float gv[2][kT];
    auto load_gate = [&](int k, float (&x)[kT]) {
        int h;
        const int tok = token_of(k, &h);
        if (tok < q_top) {
            const float *from = reinterpret_cast<const float *>(p.gate + (int64_t)(rq.q0 + tok) * p.gate_nb2 + h * p.gate_nb1) + n;
#pragma unroll
            for (int T = 0; T < kT; ++T) x[T] = from[kN * T];
        }
    };
    if (!kPart && whole && p.gate) load_gate(0, gv[0]);
#pragma unroll
    for (int k = 0; k < kR; ++k) {
        if (!kPart && whole && p.gate && k + 1 < kR) load_gate(k + 1, gv[(k + 1) & 1]);
        int h;
        const int tok = token_of(k, &h);
        if (tok >= q_top) continue;
        const float mrow = n_tiles > 0 ? ml[2 * row_at(k)] : -INFINITY;
        const float lrow = n_tiles > 0 ? ml[2 * row_at(k) + 1] : 0.0f;
        if (whole) {
            const float inv = lrow == 0.0f ? 0.0f : 1.0f / lrow;
            float *to = dst + ((int64_t)(rq.q0 + tok) * p.H + h) * kHeadDim + n;
            float o[kT];
#pragma unroll
            for (int T = 0; T < kT; ++T) o[T] = __builtin_amdgcn_ldexpf(acc[T][k], e_out[T / (kT / 4)]) * inv;
            if (!kPart && p.gate) {
#pragma unroll
                for (int T = 0; T < kT; ++T) o[T] = gate_by(o[T], gv[k & 1][T]);
            }
            if constexpr (kPart)
                if (n == 0) {
                    float *ml_to = p.stats + ((int64_t)(rq.q0 + tok) * p.H + h) * 2;
                    store_through(ml_to, lrow != lrow ? lrow : mrow);
                    store_through(ml_to + 1, lrow);
                }
#pragma unroll
            for (int T = 0; T < kT; ++T) store_through(to + kN * T, o[T]);
        } else {
            const int64_t at = (int64_t)slot * rows_per_wg(kRG) + kN * w + row_at(k);
#pragma unroll
            for (int T = 0; T < kT; ++T)
                store_through(p.acc_c + at * kHeadDim + kN * T + n, __builtin_amdgcn_ldexpf(acc[T][k], e_out[T / (kT / 4)]));
            if (n == 0) {
                // (acc and l of every split carry the same 2^kEp, which cancels in the merge; a
                // row of NaN has seen keys, though none of them moved its maximum)
                store_through(p.ml_c + at * 2, lrow != lrow ? lrow : mrow);
                store_through(p.ml_c + at * 2 + 1, lrow);
            }
        }
    }
}
inline hipError_t raise_chunk_lds(const void *kernel) {
    return hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsBytes);
}

}  // namespace
}  // namespace paged
}  // namespace sqa
