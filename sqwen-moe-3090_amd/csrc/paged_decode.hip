// paged_decode.hip - attention of requests with few new tokens (up to 16 query rows
// per KV head) over a paged q4_0 pool: decode steps and verification of drafts.
//
// Work split
//   The (request, 64-key tile) pairs of the call are cut into pieces of about equal
//   length inside a request, as many as workgroups are resident together (two per
//   CU), or one per CU where that leaves a piece fewer than four tiles. Lengths are
//   known on the GPU only: every wavefront takes the sums over the batch for itself,
//   64 requests at a time, and finds its piece (few_piece), so no launch stands before
//   the work. Up to 64 requests are in its lanes, without a barrier; more go into LDS
//   once, by all wavefronts, between two barriers.
//   The KV heads of a piece run on one XCD, whose L2 serves the lines that the heads
//   share in a row of Hkv x 144 bytes.
//
// A workgroup (8 wavefronts): four score wavefronts (16-key quarter w of every tile)
// compute the logits and softmax weights P of tile t, four value wavefronts (64-dim
// slice v) accumulate P V of tile t - 1; P crosses through LDS, one barrier a tile.
// Memory: value wavefront w moves the 16 keys of quarter w HBM -> LDS with
// global_load_lds_dwordx4. A page holds 16 keys or a multiple, so the quarter lies on
// one page: its id is one scalar load, read a tile ahead, and every address is a
// scalar base plus the lane's constant offset - as in a contiguous cache. (Instructions
// that run over all 64 keys, 9 a tensor instead of 12, need a page per lane.) K goes
// into a ring of 3 stages two tiles ahead, V one tile ahead.
// Arithmetic as in the contiguous decode kernel: Q rounded to q8_0, exact integer
// block dots on v_mfma_i32_16x16x64_i8 (block-diagonal B operand: 8 rows x 2 blocks),
// d_k d_q in fp32; softmax base 2 in fp32 with a reference maximum that moves only
// when a logit passes it by kSlack; A = P d_v 2^E as an fp16 hi + lo pair, B = the
// codes, v_mfma_f32_16x16x32_f16, exact products, fp32 sums. E follows the largest
// |d_v| seen. A key that no row sees (behind the last, behind the causal limit, on a
// page that is not there) contributes exactly 0 whatever its bytes.
// Bound: the issue of its vector, LDS and matrix instructions (two workgroups a CU make
// 1.2 tiles of 18 KB a us, 5.7 TB/s on the chip) and about 8 us at a launch's start
// and end: 16 requests of 100000 to 131071 keys 231 us, 4.6 TB/s (a copy: 4.98).
#include <mutex>

#define SQA_PLAN_CHUNKS
#include "paged_work.hpp"

namespace sqa {
namespace paged {
namespace {

typedef int int32x4 __attribute__((ext_vector_type(4)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

constexpr int kScoreWaves = 4;
constexpr int kValueWaves = 4;
constexpr int kWaves = kScoreWaves + kValueWaves;
constexpr int kThreads = 64 * kWaves;
constexpr int kTileKeys = 64;
constexpr int kKStages = 3;
constexpr int kVStages = 3;
constexpr int kSlotsPerRow = 9;                       // the head row's 9 chunks
constexpr int kLdsRow = 16 * kSlotsPerRow;            // 144
constexpr int kTensorBytes = kTileKeys * kLdsRow;     // 9216
constexpr int kPRow = 136;                            // fp16 P row: 64 keys hi, 64 keys lo, 8 pad
// LDS map
constexpr int kOffV = kKStages * kTensorBytes;
constexpr int kOffDk = kOffV + kVStages * kTensorBytes;          // per score wave [8 blocks][16 keys] fp16
constexpr int kOffDv = kOffDk + kScoreWaves * 256;             // per value wave [2 blocks][2 halves][4][8] fp16
constexpr int kOffP = kOffDv + kValueWaves * 256;              // [2 tiles][16 rows][kPRow] fp16 hi|lo
constexpr int kOffM = kOffP + 2 * 16 * kPRow * 2;              // [2 tiles][4 waves][16 rows] f32
constexpr int kOffFlag = kOffM + 2 * 4 * 16 * 4;               // [2 tiles][4 waves] u32
constexpr int kOffL = kOffFlag + 2 * 4 * 4;                    // [4 waves][16 rows] f32
constexpr int kLdsBytes = kOffL + 4 * 16 * 4;
constexpr float kSlack = 8.0f;  // log2 of the largest P the lazy rescale admits
// P is stored as P 2^-kPShift (<= 2^(kSlack - kPShift) = 2^14) and l summed from the
// same values; with |d_v 2^E| < 2, A = P d_v 2^E stays below 2^15. (The range goes to P:
// at P 2^-4 its lo part lay so deep in fp16's subnormals that the output was 1.4e-6 off
// for 4096 keys, now 2e-7.)
constexpr float kPShift = -6.0f;
// Largest d_v exponent E of the value wavefronts (d_v enters A as d_v 2^E): V
// scales below 2^-20 lose low bits of A; 2^E stays two fp16 powers of two.
constexpr int kMaxDvExp = 18;
static_assert(kMaxRequests * 4 <= kLdsBytes, "tiles of every request");
static_assert(2 * kLdsBytes <= 160 * 1024, "two workgroups per CU");
static_assert((512 + 6 * 2600 + 8) * 4 <= kLdsBytes && (512 + kMaxRequests + 8) * 4 <= kLdsBytes, "the plan's LDS");
static_assert(4 * 2 * 64 * 32 <= (kVStages - 1) * kTensorBytes, "Q operands must fit in V stages 1..2");

typedef const __attribute__((address_space(3))) uint32_t lds_u32;  // LDS dword from a raw LDS address

__device__ __forceinline__ uint32_t lds32(const uint8_t *p) { return *reinterpret_cast<const uint32_t *>(p); }
__device__ __forceinline__ uint32_t lds16(const uint8_t *p) { return *reinterpret_cast<const uint16_t *>(p); }

// Exchanges with lane ^ 16 and lane ^ 32 through gfx950's row swaps (VALU, no
// LDS round trip): a swap of x with itself returns x and the partner's x in the
// two halves of its result, in an order that depends on the lane.
__device__ __forceinline__ float xmax16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xmax32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xsum16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float xsum32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ int xsum16(int x) {
    const auto r = __builtin_amdgcn_permlane16_swap((uint32_t)x, (uint32_t)x, false, false);
    return (int)(r[0] + r[1]);
}
__device__ __forceinline__ uint32_t or16(uint32_t x) {  // x | x of lane ^ 16
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return r[0] | r[1];
}
__device__ __forceinline__ uint32_t or32(uint32_t x) {  // x | x of lane ^ 32
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return r[0] | r[1];
}
// x of lane ^ 32: lanes 0-31 find it in the swapped source, lanes 32-63 in the
// swapped destination
__device__ __forceinline__ int xother32(int x) {
    const auto r = __builtin_amdgcn_permlane32_swap((uint32_t)x, (uint32_t)x, false, false);
    return (int)((threadIdx.x & 32) ? r[0] : r[1]);
}

// a * b - c in packed fp16, the negation as an operand modifier (written as
// -c in C, the backend lowers the negation of the first pair as three VALU)
__device__ __forceinline__ half8 fma_minus(half8 a, half8 b, half8 c) {
    uint32_t x[4], y[4], z[4], r[4];
    __builtin_memcpy(x, &a, 16);
    __builtin_memcpy(y, &b, 16);
    __builtin_memcpy(z, &c, 16);
#pragma unroll
    for (int m = 0; m < 4; ++m)
        asm("v_pk_fma_f16 %0, %1, %2, %3 neg_lo:[0,0,1] neg_hi:[0,0,1]" : "=v"(r[m]) : "v"(x[m]), "v"(y[m]), "v"(z[m]));
    half8 o;
    __builtin_memcpy(&o, r, 16);
    return o;
}

__device__ __forceinline__ float exp2_or_zero(float a, float b) {  // 2^(a-b), 0 when a = -inf
    return a == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(a - b);
}


// A piece of the call: tiles [t0, t1) of request b, split `split` of its n, which start
// at piece `first`. b < 0: no such piece.
struct Piece {
    int b, split, n, first, t0, t1;
    Request rq;
};

constexpr int kLengths = 8;

// Tiles of request b, r; 0: none of this kernel's.
__device__ __forceinline__ int tiles_of(const Call &c, int b, const Request &r, int most) {
    return b >= c.B || r.n == 0 || r.n * c.G > most ? 0 : max((r.kv + kTileKeys - 1) / kTileKeys, 1);
}

// Piece length: from total / P up to nearly twice that, the shortest whose pieces number
// at most P, the workgroups that run together: by bisection of up to 256 requests, of more
// the shortest of 8 lengths. (Up to 64 in lanes the steps cost nothing; 128 requests of 2000
// to 8000 keys 102.5 us with bisection and 105.3 with 8 lengths, 200 183.5 and 184.5, 300
// 273.2 and 263.3, 1000 of 500 to 2000 316.9 and 264.1.) Where no length does (as many
// requests as that) total / P, and the rest follows as others end. Up to 64 requests are in
// a wavefront's lanes, more in LDS (read again from memory for each of the sums, 1000
// requests of up to 500 keys took 181 us instead of 140; 16 a lane, the code for it cost
// every call 1.3 us).
__device__ __forceinline__ Piece few_piece(const Call &c, int *lds, int piece, int most) {
    const int lane = threadIdx.x & 63;
    const bool small = c.B <= 64;
    const Request mine = request(c, min(lane, c.B - 1));
    const int own = tiles_of(c, lane, mine, most);
    if (!small) {
        for (int b = threadIdx.x; b < c.B; b += kThreads) lds[b] = tiles_of(c, b, request(c, b), most);
        __syncthreads();
    }
    auto tiles = [&](int b0) { return small ? own : b0 + lane < c.B ? lds[b0 + lane] : 0; };
    int total = 0, longest = 0, active = 0;
    for (int b0 = 0; b0 < c.B; b0 += 64) {
        const int t = tiles(b0);
        total += min(t, 1 << 18);  // 2^12 requests: below 2^31
        longest = max(longest, t);
        active += t > 0;
    }
    total = wave_sum(total);
    longest = wave_max(longest);
    active = wave_sum(active);
    int P = (int64_t)total * c.Hkv >= 8 * c.cus ? c.all_pieces : c.few_pieces;
    P = max(min(P, c.room - active), 1);
    // (at or a little above total / P)
    const int share = (int)ceilf((float)total * __builtin_amdgcn_rcpf((float)P) * 0.999999f);
    // (no request has more than 2^25 tiles; lengths of up to 15 times this have to fit an int)
    const int base = min(max(max(share, (longest + kMostSplits - 1) / kMostSplits), 1), 1 << 25);
    int len = 0;
    if (c.B <= 256) {
        int lo = base, hi = 2 * base;  // the first length that will do, if it is below hi
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            int k = 0;
            for (int b0 = 0; b0 < c.B; b0 += 64) k += div_ceil(tiles(b0), mid);
            if (wave_sum(k) <= P) hi = mid;
            else lo = mid + 1;
        }
        len = lo < 2 * base ? lo : 0;
    }
    int n[kLengths] = {};
    for (int b0 = 0; b0 < c.B && len == 0; b0 += 64) {
        const int t = tiles(b0);
#pragma unroll
        for (int j = 0; j < kLengths; ++j) {
            const int len = (base * (kLengths + j) + kLengths - 1) / kLengths;
            n[j] += div_ceil(t, len);
        }
    }
#pragma unroll
    for (int j = 0; j < kLengths; ++j)
        if (len == 0 && wave_sum(n[j]) <= P) len = (base * (kLengths + j) + kLengths - 1) / kLengths;
    if (len == 0) len = wave_sum(n[0]) <= c.room ? base : 1 << 25;  // 2^25 tiles: every request whole
    Piece pc{-1, 0, 1, 0, 0, 0, {}};
    int first = 0;
    for (int b0 = 0; b0 < c.B && first <= piece; b0 += 64) {
        const int t = tiles(b0);
        const int k = div_ceil(t, len);
        const int upto = first + wave_scan(k);
        const uint64_t hit = __ballot(piece >= upto - k && piece < upto);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            pc.b = b0 + l;
            pc.n = __builtin_amdgcn_readlane(k, l);
            pc.first = __builtin_amdgcn_readlane(upto - k, l);
            pc.split = piece - pc.first;
            const int tiles = __builtin_amdgcn_readlane(t, l);
            const int q = div_floor(tiles, pc.n), rest = tiles - q * pc.n;  // the first `rest` splits are one longer
            pc.t0 = pc.split * q + min(pc.split, rest);
            pc.t1 = pc.t0 + q + (pc.split < rest);
            const int *from[5] = {&mine.q0, &mine.n, &mine.kv, &mine.pos0, &mine.prefix};
            int *to[5] = {&pc.rq.q0, &pc.rq.n, &pc.rq.kv, &pc.rq.pos0, &pc.rq.prefix};
#pragma unroll
            for (int i = 0; i < 5; ++i) *to[i] = __builtin_amdgcn_readlane(*from[i], l);
        }
        first = __builtin_amdgcn_readlane(upto, 63);
    }
    // (divisions run on the vector unit: back into scalar registers)
    for (int *x : {&pc.b, &pc.split, &pc.n, &pc.first, &pc.t0, &pc.t1}) *x = __builtin_amdgcn_readfirstlane(*x);
    if (pc.b >= 64) pc.rq = uniform_request(c, pc.b);
    if (!small) __syncthreads();  // lds is free again
    return pc;
}

// A call whose max_q says that every request is one of few rows: the tokens of others
// have no partials.
__device__ __forceinline__ void skip_large(const Call &c) {
    for (int b = threadIdx.x; b < c.B; b += kThreads) {
        const Request r = request(c, b);
        if (r.n * c.G > c.most_d)
            for (int i = 0; i < r.n; ++i) c.where[r.q0 + i] = make_int4(0, 0, 0, kDone);
    }
}

// Chunk rotation of an LDS row: K rows 8-15 of every 16-row group start one
// slot later, V rows two slots later per 8-row group (mod kSlotsPerRow).
__device__ __forceinline__ int k_rot(int row) { return (row >> 3) & 1; }
__device__ __forceinline__ int v_rot(int row) { return 2 * ((row >> 3) & 3); }

// Source offset of this lane in a wavefront's s-th group of 16 bytes: slot s % 9 of row
// s / 9 (of its 16, which start at row0 of the tile), chunk (slot - rot) mod 9 of the
// head's 144 bytes.
template <bool V>
__device__ __forceinline__ uint32_t slot_offset(int row0, int s, int kvh, uint32_t row_bytes) {
    const int row = s / kSlotsPerRow;
    const int slot = s - row * kSlotsPerRow;
    int c = slot - (V ? v_rot(row0 + row) : k_rot(row0 + row));
    c = c < 0 ? c + kSlotsPerRow : c;
    return (uint32_t)row * row_bytes + (uint32_t)(kvh * kHeadRowBytes + c * 16);
}
// LDS byte of head-row byte c (0..143) of row `row` inside a tile stage
template <bool V>
__device__ __forceinline__ int lds_byte(int row, int c) {
    int slot = (c >> 4) + (V ? v_rot(row) : k_rot(row));
    slot = slot >= kSlotsPerRow ? slot - kSlotsPerRow : slot;
    return row * kLdsRow + slot * 16 + (c & 15);
}

// TWO = false: requests of up to 8 query rows per KV head (one block-diagonal B set).
// TWO = true : up to 16 rows (rows 0-7 and 8-15 as two B sets, one A operand).
// OPT: the logits are capped or biased. PLAN: a last workgroup plans the many-row kernel.
// (128 registers a lane; TWO with OPT and PLAN keeps one more in scratch, the others none.)
template <bool TWO, bool OPT, bool PLAN>
__global__ __launch_bounds__(kThreads, 4) void paged_few_kernel(Call p) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // wave-uniform, in an SGPR
    const int lane = tid & 63;
    const int g = lane >> 4;
    const int n = lane & 15;
    const bool score = wave < kScoreWaves;
    const int wq = wave & 3;  // score: 16-key quarter of every tile; value: 64-dim slice
    // LDS byte address of smem, computed once: the cast carries a null check the
    // compiler would otherwise repeat at every use
    uint32_t lds0 = (uint32_t)(uintptr_t)smem;
    asm volatile("" : "+s"(lds0));
    constexpr int kRowMask = TWO ? 15 : 7;  // rows 8-15 mirror rows 0-7 when only 8 exist

    if (PLAN && blockIdx.z == gridDim.z - 1) {
        if (blockIdx.x == 0 && blockIdx.y == 0) plan_chunks(p, reinterpret_cast<int *>(smem));
        return;
    }
    // ---------------- piece and KV head of this workgroup ---------------------
    // Workgroups go round-robin to the 8 XCDs, x (of 8) first, then the KV heads (y), then
    // z: the heads of piece 8z + x share an XCD (and its L2).
    const int kvh = (int)blockIdx.y;
    const int piece = (int)(8 * blockIdx.z + blockIdx.x);
    const Piece pc = few_piece(p, reinterpret_cast<int *>(smem), piece, p.most_d);
    if (!PLAN && blockIdx.x + blockIdx.y + blockIdx.z == 0) skip_large(p);
    // The workspace has slots for `room` pieces. Requests whose ranges of q_start overlap may be
    // more than there are tokens, which room counts on, and the grid is a multiple of 8 of them.
    if (pc.b < 0 || piece >= p.room) return;
    const Request rq = pc.rq;
    const int rows = rq.n * p.G;
    const int slot = (pc.first + pc.split) * p.Hkv + kvh;
    if (pc.split == 0 && kvh == 0 && tid < rq.n)
        p.where[rq.q0 + tid] = make_int4(pc.first * p.Hkv, pc.n, tid * p.G, p.Hkv * 4 + kFew);
    const int k0 = pc.t0 * kTileKeys;
    const int k1 = min(pc.t1 * kTileKeys, rq.kv);
    const int n_tiles = uniform(k1 > k0 ? (k1 - k0 + kTileKeys - 1) / kTileKeys : 0);
    const TableRow table = table_row(p, pc.b);
    // page of 16-key group g16 of tile t; a group behind the last key stands for the last one
    const int last_key = max(rq.kv - 1, 0);
    // Tiles in order, with a bias the last first: the logits grow towards the token, and
    // every tile in order would move the maximum (12 requests of 10501 keys: 30 us
    // instead of 25).
    const bool back = OPT && p.bias != 0.0f;
    auto tile_at = [&](int t) { return back ? n_tiles - 1 - t : t; };
    auto group_key = [&](int t, int g16) {
        return __builtin_amdgcn_readfirstlane(min(k0 + tile_at(t) * kTileKeys + 16 * g16, last_key & ~15));
    };

    // Of two workgroups on a CU the first one gets ahead (1.30 us a tile against 1.82) and
    // leaves the CU to the other, at 1.2, for the last quarter of the time. The second one's
    // wavefronts go first in three tiles of four: 16 requests of 120000 keys 246 -> 243 us,
    // 12 of 10500 with two tokens 32.2 -> 31.0.
    const bool second = (int)(blockIdx.x + 8 * (blockIdx.y + gridDim.y * blockIdx.z)) >= p.cus;
    auto take_turns = [&](int t) {
        if (((t & 3) == 3) != second) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
    };

    uint8_t *qs_lds = smem + kOffV + kTensorBytes;  // Q operands (V stages 1-2, free until V(1) is issued)
    // Per-tile exchange areas
    _Float16 *pbuf = reinterpret_cast<_Float16 *>(smem + kOffP);
    float *mbuf = reinterpret_cast<float *>(smem + kOffM);
    uint32_t *fbuf = reinterpret_cast<uint32_t *>(smem + kOffFlag);
    float *lbuf = reinterpret_cast<float *>(smem + kOffL);
    
    if (score) {
        // ============ score wavefronts: QK and softmax weights =================
        // Q -> q8_0 block-diagonal B operands. Column n of C: row r = (n & 7)
        // [+ 8 for the second set], block 2*pair + (n >> 3). Lane (g, n) supplies
        // k = 16g..16g+15, i.e. values 16*(g&1).. of the column's block when
        // (g >> 1) == (n >> 3), zeros otherwise. The four wavefronts each load
        // their block pair (pair = wq) of the Q rows straight from global memory
        // at entry, quantise it and exchange the operands through LDS.
        constexpr int kSets = TWO ? 2 : 1;
        constexpr int kOpndBytes = 32;  // per lane: 16 code bytes, d_q, -8*sum(q8)
        int32x4 bq[kSets][4];
        float dqs[kSets][4];
        int cinit[kSets][4];
        const bool q_active = (g >> 1) == (n >> 3);
        {
            int32x4 my_bq[kSets];
            float my_dq[kSets];
            int my_ci[kSets];
            const int pr = wq;
#pragma unroll
            for (int set = 0; set < kSets; ++set) {
                const int r = 8 * set + (n & 7);
                const bool row_ok = r < rows;
                const int t = group_of(p, r);
                const int hq = kvh * p.G + (r - t * p.G);
                const float *qrow = reinterpret_cast<const float *>(
                    p.q + (row_ok ? (int64_t)(rq.q0 + t) * p.q_nb1 + (int64_t)hq * p.q_nb2 : 0));
                const int blk = 2 * pr + (n >> 3);
                float x[16];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4a v4 = *reinterpret_cast<const float4a *>(qrow + 32 * blk + 16 * (g & 1) + 4 * j);
                    x[4 * j] = v4.x;
                    x[4 * j + 1] = v4.y;
                    x[4 * j + 2] = v4.z;
                    x[4 * j + 3] = v4.w;
                }
                const bool use = row_ok && q_active;
                // (0 times NaN or Inf is NaN: the block's scale then is NaN, and so is every logit of the
                // row; fmaxf and the codes would pass over a NaN)
                float amax = 0.0f, odd = 0.0f;
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    x[j] = use ? x[j] : 0.0f;
                    amax = fmaxf(amax, fabsf(x[j]));
                    odd = fmaf(x[j], 0.0f, odd);
                }
                amax = xmax16(amax);  // the other 16 values of the block
                const float d = amax / 127.f + xsum16(odd);
                const float id = amax != 0.0f ? 127.f / amax : 0.0f;
                int sumq = 0;
                uint32_t w4[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t w = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int qv = (int)rintf(x[4 * j + e] * id);
                        sumq += qv;
                        w |= (uint32_t)(qv & 0xff) << (8 * e);
                    }
                    w4[j] = w;
                }
                __builtin_memcpy(&my_bq[set], w4, 16);
                sumq = xsum16(sumq);
                const float dqv = (float)(_Float16)d * p.qscale;
                const int civ = -8 * sumq;
                const float dq2 = __int_as_float(xother32(__float_as_int(dqv)));  // inactive lanes: column n lives in lane ^ 32
                const int ci2 = xother32(civ);
                my_dq[set] = q_active ? dqv : dq2;
                my_ci[set] = q_active ? civ : ci2;
            }
#pragma unroll
            for (int set = 0; set < kSets; ++set) {
                uint8_t *o = qs_lds + ((pr * kSets + set) * 64 + lane) * kOpndBytes;
                *reinterpret_cast<int32x4 *>(o) = my_bq[set];
                *reinterpret_cast<float2 *>(o + 16) = make_float2(my_dq[set], __int_as_float(my_ci[set]));
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // operands published
#pragma unroll
            for (int pp = 0; pp < 4; ++pp)
#pragma unroll
                for (int set = 0; set < kSets; ++set) {
                    const uint8_t *o = qs_lds + ((pp * kSets + set) * 64 + lane) * kOpndBytes;
                    bq[set][pp] = *reinterpret_cast<const int32x4 *>(o);
                    const float2 dc = *reinterpret_cast<const float2 *>(o + 16);
                    dqs[set][pp] = dc.x;
                    cinit[set][pp] = __float_as_int(dc.y);
                }
        }
        // This lane's logit row (column n of the combined C): query position and validity.
        const int my_r = TWO ? n : (n & 7);
        const bool my_ok = my_r < rows;
        const int my_t = my_ok ? group_of(p, my_r) : 0;
        const int my_see = sees(rq, my_t);  // keys that the row sees
        const int my_pos = rq.pos0 + my_t;
        float my_slope = 0.0f;
        if (OPT && p.bias != 0.0f) my_slope = slope2(p, kvh * p.G + my_r - my_t * p.G);
        const bool row_writer = TWO || n < 8;  // lanes n >= 8 mirror rows 0-7 when only 8 exist
        // K operand: lane (g, n) reads key n's block 2*pair + (g >> 1), nibbles of half g & 1.
        // qs of block b sits at 18b + 2 in the head row: 4-aligned for odd b, 2 mod 4 for
        // even b. The five dwords from the aligned address below it stay inside two
        // adjacent slots of the row (block 7 spills one unused dword into the next).
        const int ka_blk_par = g >> 1;
        const uint32_t ka_shift = (ka_blk_par ? 0u : 16u) + 4u * (uint32_t)(g & 1);
        uint8_t *dk_comp = smem + kOffDk + wave * 256;  // [8 blocks][16 keys] fp16
        const int key0 = 16 * wq;                       // first key of this wavefront in a tile
        // P is stored in key order: this lane's four keys key0 + 4g + i
        const int p_col = key0 + 4 * g;
        int ka_off[4];  // LDS offsets of this lane's K windows (block pair pr), within a stage
#pragma unroll
        for (int pr = 0; pr < 4; ++pr)
            ka_off[pr] = lds_byte<false>(key0 + n, (18 * (2 * pr + ka_blk_par) + 2) & ~3);
        // d_k compaction: lane -> block lane >> 3, keys key0 + 4gg + 2hh and the next one
        const int dk_blk = lane >> 3, dk_gg = lane & 3, dk_hh = (lane >> 2) & 1;
        const int dk_src = lds_byte<false>(key0 + 4 * dk_gg + 2 * dk_hh, 18 * dk_blk);
        const int dk_dst = (dk_blk * 16 + 4 * dk_gg + 2 * dk_hh) * 2;

        // first tile with a key that the first token does not see (later ones see more)
        const int t_tail = max(sees(rq, 0) - k0, 0) / kTileKeys;
        int pid = n_tiles > 0 ? page_id(table, group_key(0, wq) >> p.lp) : 0;  // of this wavefront's 16 keys
        float m_ref = -INFINITY;   // base-2 reference max of row my_r (common to the workgroup)
        float m_used = -INFINITY;  // reference this wavefront used for the last tile's P
        float l_acc = 0.0f;        // this lane's share of the row's sum, relative to m_ref
        float l_prev = 0.0f;       // the last tile's share, relative to m_used
        // K stage of the tile (t mod kKStages, carried through the loop: LDS
        // addresses are then one add of a wave-uniform offset) and this lane's P
        // row in tile buffer 0
        int st = 0;
        _Float16 *const prow0 = pbuf + my_r * kPRow + p_col;

        for (int tt = 0; tt <= n_tiles; ++tt) {
            // the tile index is wave-uniform; with 16 rows the compiler loses track of that
            const int t = TWO ? __builtin_amdgcn_readfirstlane(tt) : tt;
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // K(t) and P(t-1) readable

            take_turns(t);
            // -- fold the last tile's sum into l under the workgroup's common max --
            if (t > 0) {
                const int pb = (t - 1) & 1;
                const uint4 fl = *reinterpret_cast<const uint4 *>(fbuf + pb * 4);
                if ((fl.x | fl.y | fl.z | fl.w) & 1u) {
                    const float *mr = mbuf + pb * 64;
                    const float mn = fmaxf(fmaxf(mr[my_r], mr[16 + my_r]), fmaxf(mr[32 + my_r], mr[48 + my_r]));
                    l_acc = l_acc * exp2_or_zero(m_ref, mn) + l_prev * exp2_or_zero(m_used, mn);
                    m_ref = mn;
                } else {
                    l_acc += l_prev;
                }
            }
            if (t == n_tiles) break;

            const int kt = k0 + tile_at(t) * kTileKeys;
            const bool there = (uint32_t)pid < (uint32_t)p.n_pages;
            if (t + 1 < n_tiles) pid = page_id(table, group_key(t + 1, wq) >> p.lp);
            const uint8_t *sK = smem + st * kTensorBytes;
            // keys that some row does not see
            const bool tail = tile_at(t) >= t_tail || !there;

            // A row r of QK is key key0 + r, so lane group g holds keys key0 + 4g + i.
            // -- compact d_k of those keys, [block][4g + i] ------------------------
            *reinterpret_cast<uint32_t *>(dk_comp + dk_dst) =
                lds16(sK + dk_src) | (lds16(sK + dk_src + kLdsRow) << 16);

            // -- QK: xs[i] = S[key key0+4g+i][row of column n] --------------------
            float xs[kSets][4];
#pragma unroll
            for (int set = 0; set < kSets; ++set)
#pragma unroll
                for (int i = 0; i < 4; ++i) xs[set][i] = 0.0f;
#pragma unroll
            for (int pr = 0; pr < 4; ++pr) {
                // key of A row n, block 2*pair + (g >> 1): five dwords from the aligned
                // address below its 16 qs bytes, shifted to the nibble half g & 1
                const uint8_t *ap = sK + ka_off[pr];
                const uint32_t w0 = lds32(ap), w1 = lds32(ap + 4), w2 = lds32(ap + 8), w3 = lds32(ap + 12),
                               w4 = lds32(ap + 16);
                uint32_t aw[4];
                aw[0] = __builtin_amdgcn_alignbit(w1, w0, ka_shift) & 0x0F0F0F0Fu;
                aw[1] = __builtin_amdgcn_alignbit(w2, w1, ka_shift) & 0x0F0F0F0Fu;
                aw[2] = __builtin_amdgcn_alignbit(w3, w2, ka_shift) & 0x0F0F0F0Fu;
                aw[3] = __builtin_amdgcn_alignbit(w4, w3, ka_shift) & 0x0F0F0F0Fu;
                int32x4 aop;
                __builtin_memcpy(&aop, aw, 16);
                const uint2 dk2 = *reinterpret_cast<const uint2 *>(dk_comp + ((2 * pr + (n >> 3)) * 16 + 4 * g) * 2);
                half4 dkh;  // d_k of keys key0+4g+i, block of column n
                __builtin_memcpy(&dkh, &dk2, 8);
#pragma unroll
                for (int set = 0; set < kSets; ++set) {
                    const int ci = cinit[set][pr];
                    int32x4 c = {ci, ci, ci, ci};
                    c = __builtin_amdgcn_mfma_i32_16x16x64_i8(aop, bq[set][pr], c, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        xs[set][i] = fmaf((float)c[i] * dqs[set][pr], (float)dkh[i], xs[set][i]);
                }
            }
            // even-block half (columns 0-7) + odd-block half (columns 8-15) of each logit
            float s[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (TWO) {  // lanes n < 8 take rows 0-7 (set 0), lanes n >= 8 rows 8-15 (set 1)
                    const float u = n < 8 ? xs[0][i] : xs[1][i];
                    const float w = n < 8 ? xs[1][i] : xs[0][i];
                    s[i] = u + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(w), 0x128, 0xf, 0xf, true));
                } else {
                    s[i] = xs[0][i] +
                           __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(xs[0][i]), 0x128, 0xf, 0xf, true));
                }
            }
            // (opaque: the compiler mixed the sums with what follows them, at 26 spilled
            // registers with 16 rows, 36 us instead of 28 for two tokens a request)
#pragma unroll
            for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(s[i]));
            if (OPT) {
                if (p.cap2 != 0.0f) cap_logits(s, p.cap2, p.cap_inv, 0.0f);
                if (p.bias != 0.0f) {
                    const int far = my_pos - (kt + key0 + 4 * g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[i] = fmaf(-my_slope, fabsf((float)(far - i)), s[i]);
                }
            }
            if (tail) {  // whatever the logit is, NaN of garbage bytes too
                const int see = there ? my_see - (kt + key0 + 4 * g) : 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i] = i < see ? s[i] : -INFINITY;
            }
            // -- softmax weights under the reference max (lazy, see the header) ---
            const float lim = m_ref + kSlack;
            bool need = __any((s[0] > lim) | (s[1] > lim) | (s[2] > lim) | (s[3] > lim));
            float mu = m_ref;
            if (need) {
                float mt = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
                mt = xmax32(xmax16(mt));
                mu = fmaxf(m_ref, mt);
            }
            if (!TWO && t == 0) {
                // The split's first tile (m_ref = -inf, so mu is this wavefront's
                // row maximum), up to 8 rows: the four score wavefronts agree on
                // each row's maximum over all 64 keys (through lbuf, free until the
                // statistics, and one more barrier, which the value wavefronts
                // match) and start from it, so the tile's P needs no rescale by the
                // value wavefronts and no maximum has moved.
                if (g == 0 && row_writer) lbuf[wq * 16 + my_r] = mu;
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // first-tile maxima
                mu = fmaxf(fmaxf(lbuf[my_r], lbuf[16 + my_r]), fmaxf(lbuf[32 + my_r], lbuf[48 + my_r]));
                m_ref = mu;
                need = false;
            }
            m_used = mu;
            // the reference plus the P shift: exact while |mu| < 2^21
            const float mb = (mu == -INFINITY ? 0.0f : mu) + kPShift;
            float pv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) pv[i] = __builtin_amdgcn_exp2f(s[i] - mb);
            l_prev = (pv[0] + pv[1]) + (pv[2] + pv[3]);
            const int buf = t & 1;
            if (row_writer) {
                half4 ph, pl;
                ph = half4{(_Float16)pv[0], (_Float16)pv[1], (_Float16)pv[2], (_Float16)pv[3]};
                uint32_t hw[2];
                __builtin_memcpy(hw, &ph, 8);
                float r[4];  // exact residual p - hi, read from the packed fp16 halves by v_fma_mix
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (i & 1)
                        asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "=v"(r[i]) : "v"(pv[i]), "v"(hw[i >> 1]));
                    else
                        asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,0] op_sel_hi:[0,0,1]" : "=v"(r[i]) : "v"(pv[i]), "v"(hw[i >> 1]));
                }
                pl = half4{(_Float16)r[0], (_Float16)r[1], (_Float16)r[2], (_Float16)r[3]};
                _Float16 *prow = prow0 + buf * (16 * kPRow);
                *reinterpret_cast<half4 *>(prow) = ph;
                *reinterpret_cast<half4 *>(prow + 64) = pl;
                if (g == 0) mbuf[(buf * 4 + wq) * 16 + my_r] = mu;
            }
            // keys of this wavefront that some row sees: bit 4g + i of the 16. P >= 0
            // (or NaN), so P != 0 is a nonzero bit pattern; the 16 lanes of group g
            // (one DPP row) OR their nibbles, the four groups then OR theirs.
            uint32_t alive = min(__float_as_uint(pv[0]), 1u) | (min(__float_as_uint(pv[1]), 1u) << 1) |
                             (min(__float_as_uint(pv[2]), 1u) << 2) | (min(__float_as_uint(pv[3]), 1u) << 3);
            alive |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)alive, 0x121, 0xf, 0xf, false);  // row_ror:1
            alive |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)alive, 0x122, 0xf, 0xf, false);  // row_ror:2
            alive |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)alive, 0x124, 0xf, 0xf, false);  // row_ror:4
            alive |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)alive, 0x128, 0xf, 0xf, false);  // row_ror:8
            alive = or16(alive << (4 * g));
            alive = or32(alive);
            if (lane == 0) fbuf[buf * 4 + wq] = (need ? 1u : 0u) | (alive << 16);
            st = st == kKStages - 1 ? 0 : st + 1;
        }

        // ---------------- this split's softmax statistics ------------------------
        l_acc = xsum32(xsum16(l_acc));
        if (g == 0 && row_writer) lbuf[wq * 16 + my_r] = l_acc;
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (wq == 0 && g == 0 && row_writer && my_ok) {
            const float L = (lbuf[my_r] + lbuf[16 + my_r]) + (lbuf[32 + my_r] + lbuf[48 + my_r]);
            float *ml = p.ml_d + ((int64_t)slot * p.rows_d + my_r) * 2;
            // (a row of NaN has seen keys, though none of them moved its maximum)
            store_through(ml, L != L ? L : m_ref);
            store_through(ml + 1, L);
        }
    } else {
        // ============ value wavefronts: O[rows][64 dims] += P V =================
        // ---------------- DMA plan of this wavefront ---------------------------
        // Value wavefronts issue every DMA (score wavefronts carry no DMA state):
        // wavefront vw the 16 keys 16vw.. of every tile, which lie on one page, 16
        // rows x 9 chunks of 16 bytes as two instructions of 64 lanes and one of 16.
        const int vw = wave - kScoreWaves;
        uint32_t koff[3], voff[3];
#pragma unroll
        for (int r = 0; r < 3; ++r) {
            koff[r] = slot_offset<false>(16 * vw, 64 * r + lane, kvh, (uint32_t)p.row_bytes);
            voff[r] = slot_offset<true>(16 * vw, 64 * r + lane, kvh, (uint32_t)p.row_bytes);
        }
        // keys past the last one re-read the last bytes of its row (they are masked off)
        const int t_whole = rq.kv / kTileKeys - pc.t0;  // tiles below it are whole
        auto issue = [&](int t, int id, const uint32_t (&off)[3], const uint8_t *pool, int64_t page_bytes, uint32_t dst) {
            const int key = group_key(t, vw);
            const uint8_t *src = pool + (int64_t)((uint32_t)id < (uint32_t)p.n_pages ? id : 0) * page_bytes +
                                 (int64_t)(key & (p.page - 1)) * p.row_bytes;
            if (tile_at(t) < t_whole) {
                dma16(off[0], src, dst);
                dma16(off[1], src, dst + 1024);
                if (lane < 16) dma16(off[2], src, dst + 2048);
            } else {
                const uint32_t lim = (uint32_t)(min(rq.kv - key, 16) * p.row_bytes - 16);
                dma16(min(off[0], lim), src, dst);
                dma16(min(off[1], lim), src, dst + 1024);
                if (lane < 16) dma16(min(off[2], lim), src, dst + 2048);
            }
        };
        auto issue_k = [&](int t, int st, int id) {  // st = t mod kKStages
            issue(t, id, koff, p.k, p.k_page, lds0 + st * kTensorBytes + 16 * kLdsRow * vw);
        };
        auto issue_v = [&](int t, int st, int id) {  // st = t mod kVStages
            issue(t, id, voff, p.v, p.v_page, lds0 + kOffV + st * kTensorBytes + 16 * kLdsRow * vw);
        };
        auto id_of = [&](int t) { return t < n_tiles ? page_id(table, group_key(t, vw) >> p.lp) : 0; };
        // The wait at interval t: K of tile t and V of tile t-1 must have landed.
        // The loop issues K(t+2) and V(t+1) at interval t, after K 0, K 1 and V 0
        // before the loop, so the younger DMAs at interval t are K(t+1) and V(t),
        // three instructions each, while t + 1 < n_tiles, V(t) when t + 1 == n_tiles,
        // none at the end.
        auto wait_interval = [&](int t) {
            if (t + 1 < n_tiles)
                asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            else if (t < n_tiles)
                asm volatile("s_waitcnt vmcnt(3) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            else
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        };

        // ---------------- K 0-1 and V 0 ------------------------------------------
        // (V stages 1-2 hold the Q operands until the loop's first barrier)
        static_assert(kKStages == 3 && kVStages == 3, "the stage counter below");
        int id1 = id_of(0), id2 = id_of(1);  // pages of tiles t + 1 and t + 2, one step ahead
        if (n_tiles > 0) issue_k(0, 0, id1);
        if (n_tiles > 1) issue_k(1, 1, id2);
        if (n_tiles > 0) issue_v(0, 0, id1);
        id1 = id2;
        id2 = id_of(2);
        if (!TWO) {
            // rows 8-15 of both P buffers (never written with 8 rows) hold zeros: the
            // residual operand of the lanes that carry hi parts (see the PV below)
            const int zi = vw * 64 + lane;  // 256 lanes x 4 fp16 = 2 buffers x 8 rows x 64 hi
            *reinterpret_cast<half4 *>(pbuf + ((zi >> 7) * 16 + 8 + ((zi >> 4) & 7)) * kPRow + 4 * (zi & 15)) =
                half4{0, 0, 0, 0};
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // Q operands published
        const int dq = wq;  // dims 64dq..64dq+63: blocks 2dq, 2dq+1
        // B operand from the nibbles: in the low bits of an fp16 a nibble is the subnormal
        // nib 2^-24, in bits 4-7 nib 2^-20; one packed fma makes either (nib - 8) 2^-10, exact
        // and normal. (The offset as one more MFMA against ones, sum A, cost 243 us instead of
        // 237 for 16 requests of 120000 keys.)
        const half8 kLo = (half8)(_Float16)16384.0f, kHi = (half8)(_Float16)1024.0f, kOffset = (half8)(_Float16)-0.0078125f;
        uint8_t *dv_comp = smem + kOffDv + vw * 256;  // [bl][half][g][j] fp16
        const int ra = n & kRowMask;  // P row of this lane's A operand
        // d_v compaction: lane -> block bl, half h, key group gg, pair jj: keys
        // 32h + 8gg + 2jj and the next one (B k-slots 8gg + 2jj, +1)
        const int cbl = lane >> 5, ch = (lane >> 4) & 1, cgg = (lane >> 2) & 3, cjj = lane & 3;
        const int ckey = 32 * ch + 8 * cgg + 2 * cjj;
        const int cdst = ((cbl * 2 + ch) * 4 + cgg) * 16 + 4 * cjj;  // bytes
        const uint32_t csrc = (uint32_t)lds_byte<true>(ckey, 18 * (2 * dq + cbl));
        // V bytes of this lane: B k-slot 8g + j is key 32h + 8g + j; its byte n of block
        // 2dq + bl sits at byte c = 2 + 18*(2dq + bl) + n of the head row, rotated by
        // v_rot = 2g slots for every row the lane reads; the dword holding it carries
        // it as byte c & 3.
        uint32_t vlane[2], vsel[2];  // v_perm selector: byte c&3 of the lower key's dword -> bits 0-7, of the upper -> 16-23
#pragma unroll
        for (int bl = 0; bl < 2; ++bl) {
            const int c = 2 + 18 * (2 * dq + bl) + n;
            vlane[bl] = (uint32_t)(lds_byte<true>(8 * g, c) & ~3);
            const uint32_t b = (uint32_t)(c & 3);
            vsel[bl] = b | (0x0cu << 8) | ((4u + b) << 16) | (0x0cu << 24);
        }

        // acc[2bl] = 2^-10 sum_k A (nib_lo - 8), acc[2bl + 1] the same of the high nibble, with
        // A = P d_v of block 2dq + bl: 2^10 acc[2bl + hi] = O[row 4g+i][dim 64dq + 32bl + 16hi + n].
        floatx4 acc[4];
#pragma unroll
        for (int T = 0; T < 4; ++T) acc[T] = floatx4{0.f, 0.f, 0.f, 0.f};
        // d_v enters A as d_v 2^E (E per wavefront, only ever lowered): P 2^6 <= 2^14
        // times |d_v 2^E| < 2 keeps A below 2^15, and the largest d_v near 2^-2
        // keeps A clear of fp16 subnormals, whatever the size of V. The partial O
        // is scaled back by 2^-E; l does not carry E.
        int e_dv = kMaxDvExp;
        uint32_t dv_thr = 0;  // fp16 magnitude bits of 2^(1 - E)
        half2v dv_s1, dv_s2;  // 2^floor(E/2), 2^(E - floor(E/2))
        auto set_dv_scale = [&](int e) {
            e_dv = e;
            const int x = 1 - e;
            dv_thr = x >= 16 ? 0x7C00u : (x >= -14 ? (uint32_t)(x + 15) << 10 : 1u << (x + 24));
            const int e1 = e >> 1, e2 = e - e1;
            const uint16_t b1 = (uint16_t)((e1 + 15) << 10), b2 = (uint16_t)((e2 + 15) << 10);
            _Float16 h1, h2;
            __builtin_memcpy(&h1, &b1, 2);
            __builtin_memcpy(&h2, &b2, 2);
            dv_s1 = half2v{h1, h1};
            dv_s2 = half2v{h2, h2};
        };
        set_dv_scale(kMaxDvExp);
        float m_acc[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // reference max of rows 4g+i
        // P rows of this lane in tile buffer 0 (see the PV below)
        const _Float16 *const arow0 = pbuf + ra * kPRow + 8 * g + (TWO || n < 8 ? 0 : 64);
        const _Float16 *const lrow0 = TWO ? arow0 + 64 : pbuf + (n ^ 8) * kPRow + 8 * g;

        int c = 0;  // t mod 3, carried through the loop (3 K and 3 V stages)
        for (int tt = 0; tt <= n_tiles; ++tt) {
            const int t = TWO ? __builtin_amdgcn_readfirstlane(tt) : tt;  // wave-uniform tile index
            const int c1 = c == 2 ? 0 : c + 1, c2 = c == 0 ? 2 : c - 1;  // (t + 1) mod 3, (t + 2) mod 3
            take_turns(t);
            wait_interval(t);
            const int id3 = id_of(t + 3);
            if (t + 2 < n_tiles) issue_k(t + 2, c2, id2);
            if (t + 1 < n_tiles) issue_v(t + 1, c1, id1);
            id1 = id2;
            id2 = id3;
            c = c1;
            if (t == 0) {
                // the score wavefronts' first-tile maxima exchange (no tile, no barrier)
                if (!TWO && n_tiles > 0) asm volatile("s_barrier" ::: "memory");
                continue;
            }

            const int tv = t - 1;  // PV of the tile whose P the score wavefronts wrote last
            const int pb = tv & 1;
            const uint32_t sv_off = (uint32_t)(kOffV + c2 * kTensorBytes);  // stage of V(t - 1), wave-uniform

            // flags of the score wavefronts: bit 0 = maximum moved, bits 16-31 = their
            // 16 keys that some row of the call can see (P != 0)
            const uint4 fl = *reinterpret_cast<const uint4 *>(fbuf + pb * 4);

            // -- P rows (k-slot order), read first: their latency runs under the
            // d_v compaction below. 16 rows: pa, pl = hi and lo of row n. Up to 8 rows:
            // A row n < 8 carries the hi part of P d_v of row n and A row n + 8 its lo
            // part (C rows r and r + 8 are summed at the end), so one set of MFMAs
            // serves both: pa = the P part the lane multiplies (hi of row n, lo of row
            // n - 8), pl = the hi part whose rounding residual the lane adds (zero row
            // n + 8, hi of row n - 8).
            half8 pa[2], pl[2];  // tile halves 0, 1
            {
                const _Float16 *arow = arow0 + pb * (16 * kPRow);
                const _Float16 *lrow = lrow0 + pb * (16 * kPRow);
                pa[0] = *reinterpret_cast<const half8 *>(arow);
                pa[1] = *reinterpret_cast<const half8 *>(arow + 32);
                pl[0] = *reinterpret_cast<const half8 *>(lrow);
                pl[1] = *reinterpret_cast<const half8 *>(lrow + 32);
            }

            // -- d_v of the slice's two blocks for all 64 keys, in B k-slot order --
            // A key no row sees (masked, past the range or past the cache end) gets
            // d_v = 0, so its bytes, whatever they hold, add exactly 0 as ggml's CPU
            // loop skips such keys.
            {
                const uint8_t *src = smem + sv_off + csrc;
                uint32_t da = lds16(src), db = lds16(src + kLdsRow);
                const uint64_t alive = (uint64_t)((fl.x >> 16) | (fl.y & 0xFFFF0000u)) |
                                       ((uint64_t)((fl.z >> 16) | (fl.w & 0xFFFF0000u)) << 32);
                da = (alive >> ckey) & 1 ? da : 0u;
                db = (alive >> (ckey + 1)) & 1 ? db : 0u;
                auto store_scaled = [&]() {  // d_v 2^E in two exact steps (2^E may exceed fp16)
                    uint32_t w = da | (db << 16);
                    half2v wh;
                    __builtin_memcpy(&wh, &w, 4);
                    wh = wh * dv_s1 * dv_s2;
                    __builtin_memcpy(&w, &wh, 4);
                    *reinterpret_cast<uint32_t *>(dv_comp + cdst) = w;
                };
                // a d_v at or above 2^(1 - E) lowers E so that the largest |d_v| of
                // the tile lands in [2^-2, 2^-1); O is rescaled by the exact power of
                // two and the tile's d_v are stored again. On the split's first tile
                // O is still zero: E comes straight from the tile's largest |d_v|.
                const uint32_t mag = max(da & 0x7FFFu, db & 0x7FFFu);
                if (!TWO && tv == 0) {
                    const int mx = wave_max((int)mag);
                    if (mx != 0) {
                        const int ex = mx >> 10;
                        const int lg = ex ? ex - 15 : (31 - __clz(mx)) - 24;  // floor(log2 max |d_v|)
                        set_dv_scale(min(-2 - lg, kMaxDvExp));
                    }
                    store_scaled();
                } else {
                store_scaled();
                if (__any(mag >= dv_thr)) {
                    const int mx = wave_max((int)mag);
                    const int ex = mx >> 10;
                    const int lg = ex ? ex - 15 : (31 - __clz(mx)) - 24;  // floor(log2 max |d_v|)
                    const int e_new = -2 - lg;
                    if (e_new < e_dv) {
                        const float f = __builtin_amdgcn_ldexpf(1.0f, e_new - e_dv);
#pragma unroll
                        for (int T = 0; T < 4; ++T) acc[T] *= f;
                        set_dv_scale(e_new);
                        store_scaled();
                    }
                }
                }
            }

            // -- the split's first tile: P is relative to the rows' common maxima
            if (!TWO && tv == 0) {
                const float *mr = mbuf + pb * 64;
#pragma unroll
                for (int i = 0; i < 4; ++i) m_acc[i] = mr[(4 * g + i) & kRowMask];
            }
            // -- a possible move of the reference max ---------------------------------
            if ((fl.x | fl.y | fl.z | fl.w) & 1u) {
                const float *mr = mbuf + pb * 64;
                float fac[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = (4 * g + i) & kRowMask;
                    const float mn = fmaxf(fmaxf(mr[r], mr[16 + r]), fmaxf(mr[32 + r], mr[48 + r]));
                    fac[i] = exp2_or_zero(m_acc[i], mn);
                    m_acc[i] = mn;
                }
                const floatx4 f4 = {fac[0], fac[1], fac[2], fac[3]};
#pragma unroll
                for (int T = 0; T < 4; ++T) acc[T] *= f4;
                // P of score wavefront w (keys 16w..16w+15: this lane's half-h slots 8g..8g+7
                // come from wavefront 2h + (g >> 1)) onto the new max
                float mw[4];
#pragma unroll
                for (int w = 0; w < 4; ++w) mw[w] = mr[16 * w + ra];
                const float mna = fmaxf(fmaxf(mw[0], mw[1]), fmaxf(mw[2], mw[3]));
                const _Float16 *prow = pbuf + (pb * 16 + ra) * kPRow + 8 * g;  // hi | lo of row ra
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const half8 ph = *reinterpret_cast<const half8 *>(prow + 32 * h);
                    const half8 plo = *reinterpret_cast<const half8 *>(prow + 64 + 32 * h);
                    // P alpha as hi = fp16(P alpha) and lo = fp16(P alpha - hi), both
                    // rounded once from the exact product by v_fma_mixlo_f16. Left to
                    // the compiler, the stored hi came from the fp32 product (rounded
                    // twice) and the hi subtracted for lo from the exact one, and where
                    // the product sat near an fp16 rounding midpoint the two differed:
                    // hi + lo one fp16 ulp of hi off.
                    const float al = exp2_or_zero(mw[2 * h + (g >> 1)], mna);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float sv = (float)ph[e] + (float)plo[e];  // exact: lo is below hi's ulp
                        uint32_t hw, lw;
                        asm("v_fma_mixlo_f16 %0, %1, %2, 0" : "=v"(hw) : "v"(sv), "v"(al));
                        asm("v_fma_mixlo_f16 %0, %1, %2, -%3 op_sel_hi:[0,0,1]" : "=v"(lw) : "v"(sv), "v"(al), "v"(hw));
                        const _Float16 hi = __builtin_bit_cast(_Float16, (uint16_t)hw);
                        const _Float16 lo = __builtin_bit_cast(_Float16, (uint16_t)lw);
                        pa[h][e] = TWO || n < 8 ? hi : lo;
                        pl[h][e] = TWO ? lo : (n < 8 ? (_Float16)0 : hi);
                    }
                }
            }

            // -- O += P V over the two halves of the tile and the slice's blocks ---
            // A = P d_v exactly as Ah + Al in packed fp16: Ph d_v has at most 22
            // significant bits, so its residual after rounding to fp16 (at most 11) is
            // exact in one fma; Pl d_v is 2^-11 of it and rounds once. Every MFMA
            // product is then exact in fp32.
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // the slice's V bytes for the 32 keys of this half, two keys per register:
                // x[4*bl + m] holds keys 32h + 8g + 2m (bits 0-7) and 32h + 8g + 2m + 1
                // (bits 16-23), byte n of block 2dq + bl's qs: adjacent rows, one
                // ds_read2_b32 each. A base per two pairs keeps both dword offsets within
                // ds_read2's 8 bits.
                uint32_t x[8];
#pragma unroll
                for (int bl = 0; bl < 2; ++bl)
#pragma unroll
                    for (int mp = 0; mp < 2; ++mp) {
                        uint32_t va = lds0 + sv_off + vlane[bl] + (uint32_t)((32 * h + 4 * mp) * kLdsRow);
                        const lds_u32 *r0 = reinterpret_cast<const lds_u32 *>((uintptr_t)va);
#pragma unroll
                        for (int m2 = 0; m2 < 2; ++m2)
                            x[4 * bl + 2 * mp + m2] = __builtin_amdgcn_perm(r0[(2 * m2 + 1) * (kLdsRow / 4)],
                                                                             r0[2 * m2 * (kLdsRow / 4)], vsel[bl]);
                    }
#pragma unroll
                for (int bl = 0; bl < 2; ++bl) {
                    const uint4 dv4 = *reinterpret_cast<const uint4 *>(dv_comp + ((bl * 2 + h) * 4 + g) * 16);
                    half8 dv8;
                    __builtin_memcpy(&dv8, &dv4, 16);
                    uint32_t wlo[4], whi[4];
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        wlo[m] = x[4 * bl + m] & 0x000F000Fu;
                        whi[m] = x[4 * bl + m] & 0x00F000F0u;
                    }
                    half8 blo, bhi;
                    __builtin_memcpy(&blo, wlo, 16);
                    __builtin_memcpy(&bhi, whi, 16);
                    // (nib 2^-24) 2^14 - 8 2^-10 and (nib 2^-20) 2^10 - 8 2^-10, exact
                    blo = __builtin_elementwise_fma(blo, kLo, kOffset);
                    bhi = __builtin_elementwise_fma(bhi, kHi, kOffset);
                    if (TWO) {
                        const half8 ah = pa[h] * dv8;
                        const half8 ar = __builtin_elementwise_fma(pa[h], dv8, -ah);
                        const half8 al = __builtin_elementwise_fma(pl[h], dv8, ar);
                        acc[2 * bl] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, blo, acc[2 * bl], 0, 0, 0);
                        acc[2 * bl + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bhi, acc[2 * bl + 1], 0, 0, 0);
                        acc[2 * bl] = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, blo, acc[2 * bl], 0, 0, 0);
                        acc[2 * bl + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, bhi, acc[2 * bl + 1], 0, 0, 0);
                    } else {
                        // hi lanes: pl = 0, so a = round(pa d_v); lo lanes: a = pl_lo d_v plus the
                        // exact residual of the hi part, rounded once
                        const half8 th = pl[h] * dv8;
                        const half8 tr = fma_minus(pl[h], dv8, th);
                        const half8 a = __builtin_elementwise_fma(pa[h], dv8, tr);
                        acc[2 * bl] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, blo, acc[2 * bl], 0, 0, 0);
                        acc[2 * bl + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bhi, acc[2 * bl + 1], 0, 0, 0);
                    }
                }
            }
        }

        // ---------------- this split's partial O (un-normalised) -----------------
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // pairs the statistics barrier
        const float o_scale = __builtin_amdgcn_ldexpf(1024.0f, -e_dv);
        auto store_row = [&](int row, int i) {
            float *dst = p.acc_d + ((int64_t)slot * p.rows_d + row) * 256 + 64 * dq + n;
#pragma unroll
            for (int bl = 0; bl < 2; ++bl) {
                store_through(dst + 32 * bl, acc[2 * bl][i] * o_scale);
                store_through(dst + 32 * bl + 16, acc[2 * bl + 1][i] * o_scale);
            }
        };
        if (!TWO) {
            // C row r + 8 (lanes of group g + 2, lane ^ 32) holds the lo part of row
            // r: one lane swap per pair of C values adds them, lanes 0-31 keeping
            // i = 0, 1 (rows 4g + i) and lanes 32-63 i = 2, 3 (rows 4(g - 2) + i),
            // so every lane stores two rows
            const bool up = lane >= 32;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                auto fold = [&](floatx4 &x) {
                    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x[i]), __float_as_uint(x[i + 2]),
                                                                    false, false);
                    x[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
                };
#pragma unroll
                for (int T = 0; T < 4; ++T) fold(acc[T]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = up ? 4 * (g - 2) + i + 2 : 4 * g + i;
                if (row < rows) store_row(row, i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 4 * g + i;
                if (row < rows) store_row(row, i);
            }
        }
    }
}


}  // namespace

int launch_few(const Call &c, hipStream_t s) {
    const bool two = c.rows_d > 8, opt = c.cap2 != 0.0f || c.bias != 0.0f;
    const dim3 grid(8, (unsigned)c.Hkv, (unsigned)((c.room + 7) / 8 + (c.rows_c ? 1 : 0)));
    typedef void (*Kernel)(Call);
    static const Kernel kernels[8] = {
        paged_few_kernel<false, false, false>, paged_few_kernel<true, false, false>, paged_few_kernel<false, true, false>,
        paged_few_kernel<true, true, false>,   paged_few_kernel<false, false, true>, paged_few_kernel<true, false, true>,
        paged_few_kernel<false, true, true>,   paged_few_kernel<true, true, true>};
    static std::once_flag once;  // the LDS limit is raised once per process
    static hipError_t err = hipSuccess;
    std::call_once(once, [] {
        for (Kernel k : kernels)
            if (err == hipSuccess) err = hipFuncSetAttribute((const void *)k, hipFuncAttributeMaxDynamicSharedMemorySize, kLdsBytes);
    });
    if (err != hipSuccess) return hip_status(err, "paged_attn LDS attribute");
    const int prof = profile_start("paged_decode", s);
    kernels[two + 2 * opt + 4 * (c.rows_c != 0)]<<<grid, dim3(kThreads), kLdsBytes, s>>>(c);
    profile_stop(prof, s);
    return hip_status(hipGetLastError(), "paged_attn launch");
}

}  // namespace paged
}  // namespace sqa
