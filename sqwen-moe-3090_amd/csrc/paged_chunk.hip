// paged_chunk.hip - attention of requests with many new tokens (more than 16 query
// rows per KV head, or more than 8 beside larger ones) over a paged q4_0 pool.
//
// A workgroup takes 128 (or 64) query rows of one request and KV head (GQA packed: row
// r is token r / G, head kvh * G + r % G) and a range of its keys, 32 at a time. Its 8
// wavefronts split the work by kind as in the contiguous prefill kernel: four score
// wavefronts hold Q' (hi and lo) of 32 rows each and make the logits and P of tile t,
// four value wavefronts hold O of the same rows and add P V of tile t - 1.
//   S^T = sum over q4_0 blocks b of d_k[b] (Kc_b . Q'h_b + Kc_b . Q'l_b): exact codes as
//   fp16 on v_mfma_f32_16x16x32_f16, Q' = q8_0(Q) * scale * log2(e) as an fp16 hi + lo
//   pair, the scaling by d_k in fp32; softmax base 2 with a reference maximum that
//   moves only when a logit passes it by kSlack; O += (P d_v) V with P d_v as an fp16
//   hi + lo pair and exact codes.
//
// There is no pre-pass: the contiguous kernel expands K and V into 2112 bytes per key
// in its workspace, which for a batch would have to hold every request's keys. Here
// the value wavefronts bring the q4_0 rows themselves into LDS (288 bytes per key and
// head; a 16-key group lies on one page, so its id is one scalar load and its rows a
// scalar base plus constant offsets) and expand them there for all 128 rows:
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
// Bound: the issue of vector (0.53 of the cycles) and matrix instructions (0.38), which add
// up; exact products take two MFMAs for each useful one. 2048 tokens behind 30001, 16 heads
// on 2 KV heads: 2.30 ms, 453 TFLOP/s, 2.4 us a tile of 128 x 32. A workgroup's start and
// end are 11 us that nothing overlaps (LDS holds one a CU): Q 2.7, its quantization 2.6,
// the last tile 1.9, the result 3 to 4 (turned in LDS into whole rows it took 5).
#include <mutex>

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
constexpr int kOffDk = kPK * 512;        // K stage: Kc, Dk
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
constexpr int kLdsRaw = kLdsE + 32;               // [K, V][2][32 rows][144 B]
constexpr int kLdsBytes = kLdsRaw + 4 * kRawTile + 16;
static_assert(kLdsBytes <= 160 * 1024, "LDS budget");
static_assert(kLdsRaw % 16 == 0 && kKStage % 16 == 0 && kVStage % 16 == 0, "alignment of the stages");
constexpr int kSlack = 8;  // log2 of the largest P the lazy rescale admits
constexpr int kEp = 6;     // P travels as P 2^kEp (at most 2^14)
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

// LDS/record row of key k (0..31) of a tile: the inverse of sigma.
__device__ __forceinline__ int key_row(int k) { return 16 * ((k >> 2) & 1) + 4 * (k >> 3) + (k & 3); }


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


// The expansion of a tile by the 256 value lanes, in 9 parts that the wavefronts place
// between the MFMAs of P V. Stores are 8 bytes, the halves of a 16-byte chunk at
// addresses that differ in bit 3 (which first is a matter of the row: no selects).
//   K: lane takes block b of key k: k & 3, b & 3, k >> 4, b >> 2 from the lane's bits 0-1,
//      2-3, 4, 5, the middle bits of k from the wavefront. Row r = key_row(k) of the
//      stage, chunk 4b + m (dims 32b + 4m + {0, 2, 16, 18, 1, 3, 17, 19}) at
//      (4b + m) ^ (r & 7), halves swapped when r & 8.
//   V: lane takes bytes 4m + 2i, 4m + 2i + 1 of block b's codes for the keys 8c .. 8c + 7
//      (c, i, m from the lane's bits 0-1, 2, 3-4, b = 2w + bit 5) and stores those keys'
//      chunk of the bytes' 4 dims, chunk c of dim d at c ^ ((d >> 1) & 3), halves
//      swapped when d & 8; odd m the second byte first.
//   V scales: lane takes key lane & 31 of block 2w + (lane >> 5).
// With these maps the 32 lanes that LDS serves at a time store to 32 different pairs of
// banks (lanes over whole rows of K and over all blocks of V met in 16 of them 16 deep:
// 3260 LDS cycles a tile, 56% of them conflicts).
struct Expand {
    int k_raw, k_sh, k_to, dk_raw, dk_to;   // LDS offsets in the first of two buffers
    int v_raw, v_to, v_odd, dv_raw, dv_to, dv_key;
    uint32_t x[4], k[5], d, dk, magic;
    __device__ __forceinline__ void init(int w, int lane) {
        const int key = 16 * ((lane >> 4) & 1) + 4 * w + (lane & 3), kb = 4 * (lane >> 5) + ((lane >> 2) & 3), r = key_row(key);
        dk_raw = kLdsRaw + kHeadRowBytes * key + 18 * kb;
        k_raw = kLdsRaw + kHeadRowBytes * key + ((18 * kb + 2) & ~3);  // the codes start 2 bytes off a dword for even blocks
        k_sh = kb & 1 ? 0 : 16;
        k_to = r * 512 + 16 * ((4 * kb) ^ (r & 7)) + (r & 8);
        dk_to = kOffDk + (kb * kPK + r) * 2;
        const int c = lane & 3, i = (lane >> 2) & 1, m = (lane >> 3) & 3, b = 2 * w + (lane >> 5);
        v_raw = kLdsRaw + 2 * kRawTile + kHeadRowBytes * 8 * c + 18 * b + 2 + 4 * m + 2 * i;
        const int dim = 32 * b + 4 * m + 2 * i;
        v_to = kLdsV + 64 * dim + 16 * (c ^ ((dim >> 1) & 3)) + (dim & 8);
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
        *reinterpret_cast<uint2 *>(smem + to + 1024) = make_uint2(codes_hi(y[0], magic), codes_hi(y[1], magic));
        *reinterpret_cast<uint2 *>(smem + (to ^ 8) + 1024) = make_uint2(codes_hi(y[2], magic), codes_hi(y[3], magic));
    }
    // chunk m of the lane's block
    __device__ __forceinline__ void store_k(uint8_t *smem, int t, int m) {
        const int to = (k_to + (t & 1) * kKStage) ^ (16 * m);
        const uint32_t y = __builtin_amdgcn_alignbit(k[m + 1], k[m], (uint32_t)k_sh), z = y >> 8;
        if (m == 0) *reinterpret_cast<uint16_t *>(smem + dk_to + (t & 1) * kKStage) = (uint16_t)dk;
        *reinterpret_cast<uint2 *>(smem + to) = make_uint2(codes_lo(y, magic), codes_hi(y, magic));
        *reinterpret_cast<uint2 *>(smem + (to ^ 8)) = make_uint2(codes_lo(z, magic), codes_hi(z, magic));
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
struct QRow {
    float4a v[16];
    __device__ __forceinline__ void load(const Call &p, int64_t row, int h, int g) {
        const float *q = reinterpret_cast<const float *>(p.q + row * p.q_nb1 + (int64_t)h * p.q_nb2) + 4 * g;
#pragma unroll
        for (int b = 0; b < 16; ++b) v[b] = *reinterpret_cast<const float4a *>(q + 16 * b);
    }
    __device__ __forceinline__ void quantize(float qscale, bool ok, half8 (&hi)[8], half8 (&lo)[8]) const {
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const float4a a = v[2 * b], c = v[2 * b + 1];
            const float x[8] = {a.x, a.z, c.x, c.z, a.y, a.w, c.y, c.w};
            float amax = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[j]));
            amax = xmax32(xmax16(amax));
            const float d = amax / 127.f;
            const float id = amax != 0.0f ? 127.f / amax : 0.0f;
            const float qd = ok ? (float)(_Float16)d * qscale : 0.0f;
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                // y opaque: left visible, the compiler may round code * qd to fp16 twice
                // (once from the fp32 product for hi, once from the exact product for the
                // hi it subtracts), and a hi + lo off by one fp16 ulp of hi
                y[j] = rintf(x[j] * id) * qd;
                asm volatile("" : "+v"(y[j]));
                hi[b][j] = (_Float16)y[j];
            }
            uint32_t hw[4];
            __builtin_memcpy(hw, &hi[b], 16);
#pragma unroll
            for (int j = 0; j < 8; ++j) {  // the exact residual, hi read from its packed half
                float r;
                if (j & 1)
                    asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "=v"(r) : "v"(y[j]), "v"(hw[j >> 1]));
                else
                    asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,0] op_sel_hi:[0,0,1]" : "=v"(r) : "v"(y[j]), "v"(hw[j >> 1]));
                lo[b][j] = (_Float16)r;
            }
        }
    }
};

// ---------------------------------------------------------------- work split

__device__ __forceinline__ Item many_item(const Call &c, int lin, int qb) {
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
    const int *first = c.work + kFirstAt, *slot = first + c.B + 1, lane = threadIdx.x & 63;
    int lo = 0, hi = c.B;
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) / 64, at = lo + lane * step;
        const uint64_t below = __ballot(at < hi && first[min(at, c.B)] <= id);
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

// kRG = 2: 128 query rows a workgroup; 1: 64 rows. OPT: the logits are capped or biased.
template <int kRG, bool OPT>
__global__ __launch_bounds__(kThreads, 1) void paged_many_kernel(Call p) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63, g = lane >> 4, n = lane & 15;
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem;

    const int qb = uniform(group_of(p, rows_per_wg(kRG)));  // tokens of a query tile
    Item it = many_item(p, (int)blockIdx.x, qb);
    if (uniform(it.b) < 0) return;
    for (int *x : {&it.b, &it.kvh, &it.tile, &it.tiles, &it.split, &it.splits, &it.t0, &it.t1, &it.slot}) *x = uniform(*x);
    const Request rq{uniform(it.rq.q0), uniform(it.rq.n), uniform(it.rq.kv), uniform(it.rq.pos0), uniform(it.rq.prefix)};
    const int q_base = it.tile * qb;        // its first token in the request
    const int q_top = min(q_base + qb, rq.n);
    const bool whole = it.splits == 1;      // of the keys: the result goes out from here
    const int slot = it.slot + (it.kvh * it.splits + it.split) * it.tiles + it.tile;
    if (it.split == 0 && it.kvh == 0 && tid < q_top - q_base)
        p.where[rq.q0 + q_base + tid] =
            whole ? make_int4(0, 0, 0, kDone) : make_int4(it.slot + it.tile, it.splits, tid * p.G, 4 * it.tiles + kMany);

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
        float *ml = reinterpret_cast<float *>(smem + kLdsP) + w * (kRG * 32);  // [rg][row][m, l]
        // Q' hi and lo of rows r = 16 kRG w + 16rg + n (position q_base + r / G, head
        // kvh*G + r % G) as B operands, dims 32b + 8g..+7
        half8 bqh[kRG][8], bql[kRG][8];
        int my_see[kRG], my_pos[kRG];
        QRow qrow[kRG];
        bool row_ok[kRG];
        float my_slope[kRG];
        float m_run[kRG], l_part[kRG];
        // The logits are accumulated relative to the row's P reference mref =
        // (m_run, or 0 before the first visible key) - ep: s' = s - mref, so that
        // P = 2^s' needs no subtraction, and the lazy-maximum test s > m_run +
        // ks reads s' > lim_s (ks + ep, or -inf before the first visible key).
        // Both change only when the maximum moves.
        float mref[kRG], lim_s[kRG];
#pragma unroll
        for (int rg = 0; rg < kRG; ++rg) {
            const int r = 16 * kRG * w + 16 * rg + n;
            const int i = group_of(p, r), h = kvh * p.G + r - i * p.G;
            const bool ok = q_base + i < q_top;
            my_see[rg] = ok ? sees(rq, q_base + i) : 0;
            my_pos[rg] = rq.pos0 + q_base + i;
            my_slope[rg] = OPT && p.bias != 0.0f ? slope2(p, h) : 0.0f;
            qrow[rg].load(p, ok ? rq.q0 + q_base + i : rq.q0, h, g);
            row_ok[rg] = ok;
            m_run[rg] = -INFINITY;
            l_part[rg] = 0.0f;
            mref[rg] = -(float)kEp;
            lim_s[rg] = -INFINITY;
        }
        __builtin_amdgcn_sched_barrier(0);  // the loads stay together
        // raw rows of the first tile: the value waves expand them while Q is quantized
        if (n_tiles > 0) asm volatile("s_barrier" ::: "memory");
#pragma unroll
        for (int rg = 0; rg < kRG; ++rg) qrow[rg].quantize(p.qscale, row_ok[rg], bqh[rg], bql[rg]);
        // K operand of key row 16kg + n, dims 32b + 8g..+7: chunk (4b + g) ^ (n & 7),
        // halves swapped when n & 8; the XOR touches bit 2 of 4b + g, so even and odd
        // b use two bases and b >> 1 adds 128 bytes.
        int k_off[2][2];  // [b & 1][half]
#pragma unroll
        for (int bp = 0; bp < 2; ++bp)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) k_off[bp][hf] = n * 512 + 16 * ((4 * bp + g) ^ (n & 7)) + 8 * (hf ^ nh);
        const int p_off = w * (kRG * 2048) + 16 * lane;  // P slots [w][rg][half][lane]

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
            // this tile's four per-lane K bases, opaque to the compiler: every K read
            // is then one of them plus an immediate offset (hoisting all 64
            // base + offset sums out of the loop would need 64 more registers)
            int kb[2][2];
#pragma unroll
            for (int bp = 0; bp < 2; ++bp)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    kb[bp][hf] = (t & 1) * kKStage + k_off[bp][hf];
                    asm volatile("" : "+v"(kb[bp][hf]));
                }
            // ---- S^T: sa[rg][kg][i] = S[key kt + 8g + 4kg + i][row n of group rg] ----
            floatx4 sa[kRG][2];
#pragma unroll
            for (int rg = 0; rg < kRG; ++rg) sa[rg][0] = sa[rg][1] = OPT && p.cap2 != 0.0f ? 0.0f : -mref[rg];
            // d_k of the lane's four C rows 16kg + 4g + i, block b: 8 bytes at
            // Dk[b][16kg + 4g]
            const uint8_t *dkb = smem + (t & 1) * kKStage + kOffDk + 8 * g;
            // Software-pipelined by one step: step j = (block j >> 1, key group j & 1)
            // issues its MFMAs, then the d_k scaling of step j - 1 runs while they
            // execute. The scheduling barrier keeps the compiler from pulling the
            // scaling back next to the MFMAs it reads (it did, leaving 4-12
            // instructions between an MFMA and its consumer). The sum into sa keeps
            // the block order of the plain loop.
            floatx4 cp[kRG];
            uint2 dkp;
#pragma unroll
            for (int j = 0; j <= 16; ++j) {
                floatx4 cn[kRG];
                uint2 dkn;
                if (j < 16) {
                    const int b = j >> 1, kg = j & 1;
                    const int o = kg * 8192 + 128 * (b >> 1);
                    const half8 ak = lds_half8(smem, kb[b & 1][0] + o, kb[b & 1][1] + o);
                    dkn = *reinterpret_cast<const uint2 *>(dkb + 64 * b + 32 * kg);
#pragma unroll
                    for (int rg = 0; rg < kRG; ++rg) {
                        const floatx4 c = __builtin_amdgcn_mfma_f32_16x16x32_f16(ak, bqh[rg][b],
                                                                                 floatx4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                        cn[rg] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ak, bql[rg][b], c, 0, 0, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                if (j > 0) {
                    const int kg = (j - 1) & 1;
                    _Float16 dk[4];
                    __builtin_memcpy(dk, &dkp, 8);
#pragma unroll
                    for (int rg = 0; rg < kRG; ++rg)
#pragma unroll
                        for (int i = 0; i < 4; ++i) sa[rg][kg][i] = fmaf(cp[rg][i], (float)dk[i], sa[rg][kg][i]);
                }
                if (j < 16) {
                    dkp = dkn;
#pragma unroll
                    for (int rg = 0; rg < kRG; ++rg) cp[rg] = cn[rg];
                }
            }
            float s[kRG][8];  // keys 8g + jj, base-2 logits
#pragma unroll
            for (int rg = 0; rg < kRG; ++rg)
#pragma unroll
                for (int jj = 0; jj < 8; ++jj) s[rg][jj] = sa[rg][jj >> 2][jj & 3];
            if (OPT) {
                // one row group after the other (both at once need more registers than there
                // are), and the scaled sums before (the compiler moved those of the second
                // group behind the first one's cap, and kept 64 products alive till there)
#pragma unroll
                for (int rg = 0; rg < kRG; ++rg)
#pragma unroll
                    for (int jj = 0; jj < 8; ++jj) asm volatile("" : "+v"(s[rg][jj]));
#pragma unroll
                for (int rg = 0; rg < kRG; ++rg) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (p.cap2 != 0.0f) cap_logits(s[rg], p.cap2, p.cap_inv, -mref[rg]);
                    if (p.bias != 0.0f) {
                        const float far = (float)(my_pos[rg] - (kt + 8 * g));
#pragma unroll
                        for (int jj = 0; jj < 8; ++jj) s[rg][jj] = fmaf(-my_slope[rg], fabsf(far - (float)jj), s[rg][jj]);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            // ---- causal limit, prefix, last key, pages that are not there: whatever the
            // logit is, NaN of garbage bytes too
            if (kt + kPK > see_all || !has_a || !has_b) {
                const bool has = g < 2 ? has_a : has_b;  // lanes' keys 8g..8g+7
#pragma unroll
                for (int rg = 0; rg < kRG; ++rg) {
                    const int see = has ? min(my_see[rg], k_end) - (kt + 8 * g) : 0;
#pragma unroll
                    for (int jj = 0; jj < 8; ++jj) s[rg][jj] = jj < see ? s[rg][jj] : -INFINITY;
                }
            }
            // ---- online softmax (base 2); P and the rescale factors to LDS -----------
            uint8_t *pb = smem + kLdsP + (t & 1) * kPBuf + p_off;
            float *ab = reinterpret_cast<float *>(smem + kLdsA + (t & 1) * kABuf) + w * (kRG * 16);
#pragma unroll
            for (int rg = 0; rg < kRG; ++rg) {
                // lazy maximum: the reference moves only when a logit passes it by more
                // than ks, so P <= 2^ks and most tiles need no rescale of O
                float alpha = 1.0f;
                bool over = false;
#pragma unroll
                for (int jj = 0; jj < 8; ++jj) over |= s[rg][jj] > lim_s[rg];
                if (__any(over)) {
                    float mt = fmaxf(fmaxf(fmaxf(s[rg][0], s[rg][1]), fmaxf(s[rg][2], s[rg][3])),
                                     fmaxf(fmaxf(s[rg][4], s[rg][5]), fmaxf(s[rg][6], s[rg][7])));
                    mt = xmax16(mt);
                    mt = xmax32(mt);
                    const float m_new = fmaxf(m_run[rg], mt + mref[rg]);
                    alpha = m_run[rg] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[rg] - m_new);
                    l_part[rg] *= alpha;
                    m_run[rg] = m_new;
                    // onto the new reference: s - mref_new = s' + (mref - mref_new)
                    const float mref_new = (m_new == -INFINITY ? 0.0f : m_new) - (float)kEp;
                    const float d = mref[rg] - mref_new;
#pragma unroll
                    for (int jj = 0; jj < 8; ++jj) s[rg][jj] += d;
                    mref[rg] = mref_new;
                    lim_s[rg] = m_new == -INFINITY ? -INFINITY : lim_top;
                }
                float pf[8], psum = 0.0f;
#pragma unroll
                for (int jj = 0; jj < 8; ++jj) {
                    pf[jj] = __builtin_amdgcn_exp2f(s[rg][jj]);
                    psum += pf[jj];
                }
                l_part[rg] += psum;
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
                    float r;
                    if (jj & 1)
                        asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "=v"(r) : "v"(pf[jj]), "v"(hw[jj >> 1]));
                    else
                        asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,0] op_sel_hi:[0,0,1]" : "=v"(r) : "v"(pf[jj]), "v"(hw[jj >> 1]));
                    pl[jj] = (_Float16)r;
                }
                *reinterpret_cast<half8 *>(pb + rg * 2048) = ph;
                *reinterpret_cast<half8 *>(pb + rg * 2048 + 1024) = pl;
                if (g == 0) ab[rg * 16 + n] = alpha;
            }
        }
        // ---- hand m and l of the rows to the value waves ----------------------------
        __syncthreads();
        if (n_tiles > 0) {
#pragma unroll
            for (int rg = 0; rg < kRG; ++rg) {
                float lp = l_part[rg];
                lp += __shfl_xor(lp, 16);
                lp += __shfl_xor(lp, 32);
                if (g == 0) {
                    ml[rg * 32 + 2 * n] = m_run[rg];
                    ml[rg * 32 + 2 * n + 1] = lp;
                }
            }
        }
        __syncthreads();
        return;
    }

    // ---- value waves: O[row 16 kRG w + 16rg + 4g + i][dim 16T + n] ----------------
    const int w = wave - kScoreWaves;
    const float *ml = reinterpret_cast<const float *>(smem + kLdsP) + w * (kRG * 32);  // [rg][row][m, l]
    // V operand of dim 16T + n, keys 8g..8g+7: chunk g ^ ((n >> 1) & 3), halves swapped when n & 8.
    const int v_off0 = 64 * n + 16 * (g ^ ((n >> 1) & 3)) + 8 * nh;
    const int v_off1 = v_off0 ^ 8;
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
    Expand ex;
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
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            ex.read_k(smem, k);
#pragma unroll
            for (int m = 0; m < 4; ++m) ex.store_k(smem, k, m);
        }
        ex.read_v(smem, 0);
        scales(0, a0, b0);
        ex.store_v(smem, 0, 0);
        ex.store_v(smem, 0, 1);
    }
    floatx4 acc[kRG][16];
#pragma unroll
    for (int rg = 0; rg < kRG; ++rg)
#pragma unroll
        for (int T = 0; T < 16; ++T) acc[rg][T] = floatx4{0.f, 0.f, 0.f, 0.f};
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
        // this tile's two per-lane V bases, opaque to the compiler (see the K reads)
        int vb0 = kLdsV + (tp & 1) * kVStage + v_off0, vb1 = kLdsV + (tp & 1) * kVStage + v_off1;
        asm volatile("" : "+v"(vb0), "+v"(vb1));
        const uint8_t *pb = smem + kLdsP + (tp & 1) * kPBuf + p_off;
        const float *ab = reinterpret_cast<const float *>(smem + kLdsA + (tp & 1) * kABuf) + w * (kRG * 16);
        // O onto the exponents of this tile's V scales where a larger one has come
        int4 e_t = *reinterpret_cast<const int4 *>(smem + kLdsE + 16 * (tp & 1));
        e_t.x = __builtin_amdgcn_readfirstlane(e_t.x), e_t.y = __builtin_amdgcn_readfirstlane(e_t.y);
        e_t.z = __builtin_amdgcn_readfirstlane(e_t.z), e_t.w = __builtin_amdgcn_readfirstlane(e_t.w);
        half8 ph[kRG], pl[kRG];
        bool resc = false;
#pragma unroll
        for (int rg = 0; rg < kRG; ++rg) {
            // rescale factors of rows 4g..4g+3: exactly 1 unless a maximum moved
            const floatx4 a4 = *reinterpret_cast<const floatx4 *>(ab + rg * 16 + 4 * g);
            resc |= (a4[0] != 1.0f) | (a4[1] != 1.0f) | (a4[2] != 1.0f) | (a4[3] != 1.0f);
            ph[rg] = *reinterpret_cast<const half8 *>(pb + rg * 2048);
            pl[rg] = *reinterpret_cast<const half8 *>(pb + rg * 2048 + 1024);
        }
        if (__any(resc)) {  // rare with the lazy maximum: O = alpha O
#pragma unroll
            for (int rg = 0; rg < kRG; ++rg) {
                const floatx4 a4 = *reinterpret_cast<const floatx4 *>(ab + rg * 16 + 4 * g);
#pragma unroll
                for (int T = 0; T < 16; ++T) acc[rg][T] *= a4;
            }
        }
        if ((e_t.x ^ e_acc.x) | (e_t.y ^ e_acc.y) | (e_t.z ^ e_acc.z) | (e_t.w ^ e_acc.w)) {
            const int from[4] = {e_acc.x, e_acc.y, e_acc.z, e_acc.w}, to[4] = {e_t.x, e_t.y, e_t.z, e_t.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float f = __builtin_amdgcn_ldexpf(1.0f, to[q] - from[q]);
#pragma unroll
                for (int rg = 0; rg < kRG; ++rg)
#pragma unroll
                    for (int T = 4 * q; T < 4 * q + 4; ++T) acc[rg][T] *= f;
            }
            e_acc = e_t;
        }
        // d_v and V of block b + 1 are read while block b computes: the LDS latency stays
        // off the MFMA chain. Between the blocks, parts of the next tiles' expansion.
        uint4 dvn = *reinterpret_cast<const uint4 *>(vs + kOffDv + 16 * g);
        half8 bvn[2];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) bvn[hf] = lds_half8(smem, vb0 + 1024 * hf, vb1 + 1024 * hf);
        ex.read_v(smem, t);
        ex.read_k(smem, t + 1);
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const half8 bv[2] = {bvn[0], bvn[1]};
            const uint4 dvr = dvn;
            if (b < 7) {
                dvn = *reinterpret_cast<const uint4 *>(vs + kOffDv + 64 * (b + 1) + 16 * g);
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
                    bvn[hf] = lds_half8(smem, vb0 + 1024 * (2 * b + 2 + hf), vb1 + 1024 * (2 * b + 2 + hf));
            }
            half8 dvb;
            __builtin_memcpy(&dvb, &dvr, 16);
            // A = P 2^ep d_v as an fp16 hi + lo pair (22 bits): the products with the
            // exact V codes are then exact in fp32, so a row that a few keys
            // dominate carries no fp16 rounding of P d_v into its output. Ph d_v has
            // at most 22 significant bits, so its residual after rounding to fp16
            // (at most 11 bits) is exact in one fma; Pl d_v is 2^-11 of it and
            // rounds once.
            half8 ah[kRG], al[kRG];
#pragma unroll
            for (int rg = 0; rg < kRG; ++rg) {
                ah[rg] = ph[rg] * dvb;
                const half8 r = __builtin_elementwise_fma(ph[rg], dvb, -ah[rg]);
                al[rg] = __builtin_elementwise_fma(pl[rg], dvb, r);
            }
#pragma unroll
            for (int rg = 0; rg < kRG; ++rg)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
                    acc[rg][2 * b + hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah[rg], bv[hf], acc[rg][2 * b + hf], 0, 0, 0);
#pragma unroll
            for (int rg = 0; rg < kRG; ++rg)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
                    acc[rg][2 * b + hf] = __builtin_amdgcn_mfma_f32_16x16x32_f16(al[rg], bv[hf], acc[rg][2 * b + hf], 0, 0, 0);
            if (b == 1) scales(t, x0, y0);
            if (b == 2) ex.store_v(smem, t, 0);
            if (b == 3) ex.store_v(smem, t, 1);
            if (b >= 4) ex.store_k(smem, t + 1, b - 4);
        }
    }
    __syncthreads();  // m and l of the rows ...
    __syncthreads();  // ... are in LDS
    const int e_out[4] = {-e_acc.x, -e_acc.y, -e_acc.z, -e_acc.w};
    // rows 16 kRG w + 16 rg + 4g + i, one after the other; the gate of the next one is on
    // its way while a row goes out
    auto token_of = [&](int k, int *h) {  // k = 4 rg + i
        const int r = 16 * kRG * w + 16 * (k >> 2) + 4 * g + (k & 3), tok = group_of(p, r);
        *h = kvh * p.G + r - tok * p.G;
        return q_base + tok;
    };
    float gv[2][16];
    auto load_gate = [&](int k, float (&x)[16]) {
        int h;
        const int tok = token_of(k, &h);
        if (tok < q_top) {
            const float *from = reinterpret_cast<const float *>(p.gate + (int64_t)(rq.q0 + tok) * p.gate_nb2 + h * p.gate_nb1) + n;
#pragma unroll
            for (int T = 0; T < 16; ++T) x[T] = from[16 * T];
        }
    };
    if (whole && p.gate) load_gate(0, gv[0]);
#pragma unroll
    for (int k = 0; k < 4 * kRG; ++k) {
        const int rg = k >> 2, i = k & 3, r = 16 * kRG * w + 16 * rg + 4 * g + i;
        if (whole && p.gate && k + 1 < 4 * kRG) load_gate(k + 1, gv[(k + 1) & 1]);
        int h;
        const int tok = token_of(k, &h);
        if (tok >= q_top) continue;
        const float mrow = n_tiles > 0 ? ml[rg * 32 + 2 * (4 * g + i)] : -INFINITY;
        const float lrow = n_tiles > 0 ? ml[rg * 32 + 2 * (4 * g + i) + 1] : 0.0f;
        if (whole) {
            const float inv = lrow == 0.0f ? 0.0f : 1.0f / lrow;
            float *to = p.dst + ((int64_t)(rq.q0 + tok) * p.H + h) * kHeadDim + n;
            float o[16];
#pragma unroll
            for (int T = 0; T < 16; ++T) o[T] = __builtin_amdgcn_ldexpf(acc[rg][T][i], e_out[T >> 2]) * inv;
            if (p.gate) {
#pragma unroll
                for (int T = 0; T < 16; ++T) o[T] = gate_by(o[T], gv[k & 1][T]);
            }
#pragma unroll
            for (int T = 0; T < 16; ++T) store_through(to + 16 * T, o[T]);
        } else {
            const int64_t at = (int64_t)slot * rows_per_wg(kRG) + r;
#pragma unroll
            for (int T = 0; T < 16; ++T)
                store_through(p.acc_c + at * kHeadDim + 16 * T + n, __builtin_amdgcn_ldexpf(acc[rg][T][i], e_out[T >> 2]));
            if (n == 0) {
                // (acc and l of every split carry the same 2^kEp, which cancels in the merge; a
                // row of NaN has seen keys, though none of them moved its maximum)
                store_through(p.ml_c + at * 2, lrow != lrow ? lrow : mrow);
                store_through(p.ml_c + at * 2 + 1, lrow);
            }
        }
    }
}

}  // namespace

int launch_many(const Call &c, hipStream_t s) {
    const bool opt = c.cap2 != 0.0f || c.bias != 0.0f;
    static std::once_flag once;  // the LDS limit is raised once per process
    static hipError_t err = hipSuccess;
    std::call_once(once, [] {
        for (const void *f : {(const void *)paged_many_kernel<1, false>, (const void *)paged_many_kernel<1, true>,
                              (const void *)paged_many_kernel<2, false>, (const void *)paged_many_kernel<2, true>})
            if (err == hipSuccess) err = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsBytes);
    });
    if (err != hipSuccess) return hip_status(err, "paged_attn LDS attribute");
    const dim3 grid((unsigned)c.grid_c);
    const int prof = profile_start("paged_chunk", s);
    if (c.rows_c == 64 && opt) paged_many_kernel<1, true><<<grid, dim3(kThreads), kLdsBytes, s>>>(c);
    else if (c.rows_c == 64) paged_many_kernel<1, false><<<grid, dim3(kThreads), kLdsBytes, s>>>(c);
    else if (opt) paged_many_kernel<2, true><<<grid, dim3(kThreads), kLdsBytes, s>>>(c);
    else paged_many_kernel<2, false><<<grid, dim3(kThreads), kLdsBytes, s>>>(c);
    profile_stop(prof, s);
    return hip_status(hipGetLastError(), "paged_attn launch");
}

}  // namespace paged
}  // namespace sqa
