// lora.hip - low-rank adapters of many requests beside a shared projection:
// out = base + scale[id] B[id] (A[id] (x sigmoid(gate))), an id per token.
//
// Bound by memory: x, gate, base and out once each (48 KB a token at 4096 + 2048 columns),
// the adapters in use out of L2; by latency for few tokens. Both kernels therefore do the
// two products in one launch, with A x in LDS between them.
//
// Few tokens (decode): a workgroup per token and part of the columns. Every byte that the
// first sums need is asked for at the start (A and B rows, base beside x), so one memory
// latency stands before them; x stays in registers, 8 ranks are summed at a time and folded
// over the lanes two by two; fp32 throughout. 48 tokens of 32 adapters at rank 16: 6.0 us
// (an empty launch: 3.6).
//
// More: a workgroup takes 16 tokens. x, gate and A come in as runs of whole rows, 128
// values of K at a time (256 up to rank 16), and are laid out in LDS (rows are a power of two apart in
// memory: loads in the shape of MFMA operands, 16 rows of 64 bytes, fell into one set of
// L1 and took 137 cycles each, 100 us for 4096 tokens at rank 64). The 8 wavefronts share
// a chunk's steps of K: t^T = A x^T on v_mfma_f32_16x16x32_f16, A as it is, x as an fp16
// pair: hi = fp16(x), lo = fp16((x - hi) 2^11), in sums of their own (the shift keeps lo
// clear of subnormals: 22 bits down to |x| = 2^-13, an absolute 2^-36 below). The partial
// t are added in LDS (where one is too large for fp16, or Inf or NaN of an x that is, the
// tile's t are taken again in fp32); then the wavefronts share the columns, out^T = B t^T with t as a
// pair in the same way, turned in LDS into rows of 64 columns (32 above rank 64, for want
// of registers) for base and out. The adapters of a tile are taken by kPasses workgroups in
// turn, each writing its tokens alone; no adapter's values reach another one's tokens, not
// even its NaN. 4096 tokens in runs of 512: rank 16 43 us, 4.7 TB/s (a copy: 4.98), rank 64
// 46, where A and B out of L2 are as many bytes as x and gate; in runs of 342 to 512, with
// tokens without adapter between them and others in the next call, 67.
#include <mutex>

#include "paged.hpp"

namespace sqa {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float float4a __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kMaxRank = 128;

struct Params {
    const char *base, *x, *gate;
    int64_t base_nb1, x_nb1, gate_nb1, dst_nb1;
    const _Float16 *a, *b;
    const int32_t *ids;
    const float *scale;
    char *dst;
    int K, N, r, n, M;
};

__device__ __forceinline__ floatx4 gated(floatx4 x, floatx4 g) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * g[i]));
    return x;
}

// ------------------------------------------------------------- few tokens

__device__ __forceinline__ float bits(uint32_t x) { return __uint_as_float(x); }

template <int kCtrl>
__device__ __forceinline__ float add_dpp(float x) {
    return x + bits((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), kCtrl, 0xf, 0xf, true));
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140;  // lane ^ 1, ^ 2, 7 - i, 15 - i

// Sums of 8 values over the wavefront: s[0], s[1] hold those of value 0 or 1, + 2 in odd
// rows of 16 lanes, + 4 in the upper half. A swap folds two values at once.
__device__ __forceinline__ void fold(float (&s)[8]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(s[q]), __float_as_uint(s[q + 4]), false, false);
        s[q] = bits(r[0]) + bits(r[1]);
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(s[q]), __float_as_uint(s[q + 2]), false, false);
        s[q] = bits(r[0]) + bits(r[1]);
        s[q] = add_dpp<kMirror>(add_dpp<kHalfMirror>(add_dpp<kXor2>(add_dpp<kXor1>(s[q]))));
    }
}

// Grid (tokens, parts of the columns); K <= 4096 kRuns. A wavefront keeps its values of x,
// runs of 512, 8 a lane, in registers and takes 8 ranks at a time; where K has fewer runs
// than there are wavefronts, groups of them share the ranks. Then 1 to 16 lanes take a
// column, 8 ranks each.
template <int kRuns>
__global__ __launch_bounds__(kThreads) void lora_token_kernel(Params p) {
    __shared__ __align__(16) float part[kWaves][kMaxRank];
    const int m = blockIdx.x, tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int id = p.ids[m];
    const float *base = reinterpret_cast<const float *>(p.base + m * p.base_nb1);
    float *dst = reinterpret_cast<float *>(p.dst + m * p.dst_nb1);
    const int quads = p.N / 4, q0 = (int)((int64_t)quads * blockIdx.y / gridDim.y),
              q1 = (int)((int64_t)quads * (blockIdx.y + 1) / gridDim.y);
    if (id < 0 || id >= p.n) {
        for (int q = q0 + tid; q < q1; q += kThreads)
            reinterpret_cast<floatx4 *>(dst)[q] = reinterpret_cast<const floatx4 *>(base)[q];
        return;
    }
    if (q0 == q1) return;  // fewer quads than parts
    const _Float16 *a = p.a + (int64_t)id * p.r * p.K, *b = p.b + (int64_t)id * p.N * p.r;
    // Everything that the first sums need is on its way together (addresses clamped, not
    // branched around: a load in a branch waits for the ones before it).
    const int runs = (p.K + 511) / 512, lw = runs > 4 ? 3 : runs > 2 ? 2 : runs - 1;  // log2 of the wavefronts along K
    const int wk = wave & ((1 << lw) - 1), group = wave >> lw, groups = kWaves >> lw, batches = p.r / 8;
    const float *x = reinterpret_cast<const float *>(p.x + m * p.x_nb1);
    const float *g = p.gate ? reinterpret_cast<const float *>(p.gate + m * p.gate_nb1) : nullptr;
    auto at = [&](int i) { return 512 * (wk + kWaves * i) + 8 * lane; };  // (lw < 3 has one run a wavefront)
    floatx4 xv[kRuns][2], gv[kRuns][2];
#pragma unroll
    for (int i = 0; i < kRuns; ++i)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int k = min(at(i), p.K - 8) + 4 * q;
            xv[i][q] = *reinterpret_cast<const float4a *>(x + k);
            if (g) gv[i][q] = *reinterpret_cast<const float4a *>(g + k);
        }
    half8 av[2][8];
    auto load_a = [&](int s, int batch, int i) {
        const _Float16 *row = a + (int64_t)min(batch, batches - 1) * 8 * p.K + min(at(i), p.K - 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) av[s][j] = *reinterpret_cast<const half8 *>(row + (int64_t)j * p.K);
    };
    load_a(0, group, 0);
    // columns: 2^ll lanes of a column, chunk `ch` of 8 ranks
    constexpr int kB = 4;
    const int ll = batches > 8 ? 4 : batches > 4 ? 3 : batches > 2 ? 2 : batches - 1;
    const int ch = lane & ((1 << ll) - 1), c_own = 4 * q0 + (64 >> ll) * wave + (lane >> ll), c_step = kThreads >> ll;
    half8 bv[2][kB];
    float old[2][kB];
    auto load_b = [&](int s, int c) {
#pragma unroll
        for (int q = 0; q < kB; ++q) {
            const int cc = min(c + q * c_step, 4 * q1 - 1);
            bv[s][q] = *reinterpret_cast<const half8 *>(b + (int64_t)cc * p.r + 8 * min(ch, batches - 1));
            old[s][q] = base[cc];
        }
    };
    const float sc = p.scale ? p.scale[id] : 1.0f;
    load_b(0, c_own);
#pragma unroll
    for (int i = 0; i < kRuns; ++i)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            if (g) xv[i][q] = gated(xv[i][q], gv[i][q]);
            if (at(i) >= p.K) xv[i][q] = floatx4{0.f, 0.f, 0.f, 0.f};
        }
    auto sum = [&](int s, int i, float (&to)[8]) {
        const bool inside = at(i) < p.K;
        const bool whole = 512 * (wk + kWaves * i + 1) <= p.K;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            half8 v = av[s][j];
            if (!whole) v = inside ? v : half8{};  // (its x is 0, but 0 times Inf is not)
#pragma unroll
            for (int q = 0; q < 8; ++q) to[j] = fmaf(xv[i][q >> 2][q & 3], (float)v[q], to[j]);
        }
    };
    auto put = [&](int batch, float (&s)[8]) {
        fold(s);
        if ((lane & 15) == 0) {
            float *to = &part[wk][8 * batch + 2 * ((lane >> 4) & 1) + 4 * (lane >> 5)];
            to[0] = s[0], to[1] = s[1];
        }
    };
    for (int batch = group; batch < batches; batch += (kRuns == 1 ? 2 : 1) * groups) {
        if (kRuns == 1) {
            float s[8] = {}, u[8] = {};
            load_a(1, batch + groups, 0);
            sum(0, 0, s);
            put(batch, s);
            load_a(0, batch + 2 * groups, 0);
            sum(1, 0, u);
            if (batch + groups < batches) put(batch + groups, u);
        } else {
            float s[8] = {};
#pragma unroll
            for (int i = 0; i < kRuns; ++i) {
                load_a((i + 1) & 1, i + 1 < kRuns ? batch : batch + groups, (i + 1) % kRuns);
                sum(i & 1, i, s);
            }
            put(batch, s);
        }
    }
    __syncthreads();
    float t[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) t[q] = 0.0f;
    for (int w = 0; w < 1 << lw; ++w) {
        const floatx4 *from = reinterpret_cast<const floatx4 *>(&part[w][8 * min(ch, batches - 1)]);
        const floatx4 u = from[0], v = from[1];
#pragma unroll
        for (int q = 0; q < 4; ++q) t[q] += u[q], t[4 + q] += v[q];
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) t[q] *= sc;
    auto columns = [&](int s, int c) {
#pragma unroll
        for (int q = 0; q < kB; ++q) {
            float o = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) o = fmaf(t[i], (float)bv[s][q][i], o);
            if (ch >= batches) o = 0.0f;
            if (ll > 0) o = add_dpp<kXor1>(o);
            if (ll > 1) o = add_dpp<kXor2>(o);
            if (ll > 2) o = add_dpp<kHalfMirror>(o);
            if (ll > 3) o = add_dpp<kMirror>(o);
            if (ch == 0 && c + q * c_step < 4 * q1) dst[c + q * c_step] = old[s][q] + o;
        }
    };
    for (int c = c_own; c < 4 * q1; c += 2 * kB * c_step) {
        load_b(1, c + kB * c_step);
        columns(0, c);
        load_b(0, c + 2 * kB * c_step);
        columns(1, c + kB * c_step);
    }
}

// ----------------------------------------------------------------- tiles

constexpr int kTile = 16;   // tokens of a workgroup
constexpr int kPasses = 4;  // workgroups that share a tile's adapters

// Sizes of a form: RT tiles of 16 ranks, r <= 16 RT.
template <int RT>
struct Form {
    static constexpr int kR = 16 * RT;
    // values of K between two barriers (256 at rank 64: 72 us against 67.5 for 4096 tokens)
    static constexpr int kChunk = RT == 1 ? 256 : 128;
    static constexpr int kStepWaves = kChunk / 32, kRankWaves = kWaves / kStepWaves;  // of a chunk: steps of 32, groups of ranks
    static constexpr int kTiles = RT / kRankWaves;      // rank tiles of a wavefront
    static constexpr int kRow = kChunk * 2 + 16;        // bytes of a staged row (16 more: its rows on other banks)
    static constexpr int kX = 2 * kTile * kRow, kStage = kX + kR * kRow;  // x hi, x lo, A
    static constexpr int kT = kTile * (kR + 4) * 4;     // t: [token][rank]
    static constexpr int kCols = RT == 8 ? 32 : 64;     // columns that a wavefront takes at a time
    static constexpr int kOutRow = kCols * 4 + 16, kOut = kWaves * kTile * kOutRow;
    static constexpr int kPart = kWaves * kTiles * 16 * kTile * 4;
    static constexpr int kBytes = kT + (2 * kStage > kOut ? 2 * kStage : kOut);
    static_assert(kPart <= 2 * kStage && kBytes <= 160 * 1024, "LDS");
};

// hi = fp16(x) and lo = fp16((x - hi) 2^11). x opaque: where it is a product, the compiler
// took hi from the fp32 product and the hi that it subtracts from the exact one, and hi + lo
// was an fp16 ulp of hi off where the two differ.
__device__ __forceinline__ void split(float x, _Float16 &hi, _Float16 &lo) {
    asm volatile("" : "+v"(x));
    hi = (_Float16)x;
    lo = (_Float16)((x - (float)hi) * 2048.0f);
}

// t of a tile's tokens of adapter cur in plain fp32, a wavefront to a value: for values that fp16 does not hold.
__device__ __forceinline__ void rank_sums(const Params &p, int cur, float sc, int m0, const int *ids, float *t, int t_row) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int e = wave; e < kTile * p.r; e += kWaves) {
        const int m = e & (kTile - 1), j = e / kTile;
        if (ids[m] != cur) continue;
        const float *x = reinterpret_cast<const float *>(p.x + (m0 + m) * p.x_nb1);
        const float *g = p.gate ? reinterpret_cast<const float *>(p.gate + (m0 + m) * p.gate_nb1) : nullptr;
        const _Float16 *a = p.a + ((int64_t)cur * p.r + j) * p.K;
        float s = 0.0f;
        for (int k = 4 * lane; k < p.K; k += 256) {
            floatx4 v = *reinterpret_cast<const float4a *>(x + k);
            if (g) v = gated(v, *reinterpret_cast<const float4a *>(g + k));
#pragma unroll
            for (int i = 0; i < 4; ++i) s = fmaf(v[i], (float)a[k + i], s);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
        if (lane == 0) t[m * t_row + j] = s * sc;
    }
}

// MFMA operands (lane = 16 g + n): A[n][8g..8g+7], B[8g..8g+7][n], C[4g..4g+3][n].
template <int RT, bool GATE>
__global__ __launch_bounds__(kThreads, 2) void lora_tile_kernel(Params p) {
    typedef Form<RT> F;
    typedef _Float16 half4 __attribute__((ext_vector_type(4)));
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int ids[kTile], over;
    float *t = reinterpret_cast<float *>(smem);  // [token][kR + 4]
    uint8_t *stage = smem + F::kT;
    constexpr int kTRow = F::kR + 4;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, n = lane & 15;
    // Workgroups go round-robin to the 8 XCDs: an XCD gets a run of tiles, which share
    // adapters (in its L2) more often than not.
    const int tiles = (int)gridDim.x, xcd = (int)blockIdx.x & 7, per = tiles >> 3, rem = tiles & 7;
    const int m0 = (xcd * per + min(xcd, rem) + ((int)blockIdx.x >> 3)) * kTile;
    const int tokens = min(p.M - m0, kTile);
    int id = p.ids[m0 + min(n, tokens - 1)];
    id = n < tokens && id >= 0 && id < p.n ? id : -1;
    if (tid < kTile) ids[tid] = tid < tokens ? id : -2;
    __syncthreads();
    uint64_t todo = __ballot(id >= 0 && g == 0);
    bool rest = blockIdx.y == 0;  // tokens without adapter go with the first pass of the first workgroup
    if (!todo) {
        if (!rest) return;
        for (int e = tid; e < tokens * (p.N / 4); e += kThreads) {
            const int m = e / (p.N / 4), c = e - m * (p.N / 4);
            reinterpret_cast<floatx4 *>(p.dst + (m0 + m) * p.dst_nb1)[c] =
                reinterpret_cast<const floatx4 *>(p.base + (m0 + m) * p.base_nb1)[c];
        }
        return;
    }
    // this thread's values of a chunk: kNX times 4 of a token, kNA times 8 of a rank
    constexpr int kNX = kTile * F::kChunk / 4 / kThreads, kNA = (F::kR * F::kChunk / 8 + kThreads - 1) / kThreads;
    constexpr int kQuads = F::kChunk / 4, kOcts = F::kChunk / 8;
    const float *xr[kNX], *gr[kNX];
    int x_at[kNX];
#pragma unroll
    for (int i = 0; i < kNX; ++i) {
        const int e = tid + kThreads * i, m = e / kQuads, k = 4 * (e - m * kQuads);
        const int64_t row = m0 + min(m, tokens - 1);
        xr[i] = reinterpret_cast<const float *>(p.x + row * p.x_nb1) + k;
        gr[i] = GATE ? reinterpret_cast<const float *>(p.gate + row * p.gate_nb1) + k : nullptr;
        x_at[i] = m * F::kRow + 2 * k;
    }
    // (tiles that begin elsewhere in K, on other channels of memory, lose more to A, which
    // neighbours then no longer read together: 80 us against 74 at 4096 tokens)
    const int chunks = p.K / F::kChunk;
    for (int pass = 0; todo; ++pass) {
        const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(todo));
        todo &= ~__ballot(id == cur && g == 0);
        if ((pass & (kPasses - 1)) != (int)blockIdx.y) continue;
        const _Float16 *a = p.a + (int64_t)cur * p.r * p.K, *b = p.b + (int64_t)cur * p.N * p.r;
        const float sc = p.scale ? p.scale[cur] : 1.0f;
        const _Float16 *ar[kNA];
        int a_at[kNA];
#pragma unroll
        for (int i = 0; i < kNA; ++i) {
            const int e = tid + kThreads * i, j = min(e / kOcts, F::kR - 1), k = 8 * (e % kOcts);
            ar[i] = a + (int64_t)min(j, p.r - 1) * p.K + k;  // rows past r: the last one again, their t is not used
            a_at[i] = F::kX + j * F::kRow + 2 * k;
        }
        floatx4 xv[2][kNX], gv[2][kNX];
        half8 av[2][kNA];
        auto load = [&](int s, int c) {  // chunk c into register set s
            const int k = min(c, chunks - 1) * F::kChunk;
#pragma unroll
            for (int i = 0; i < kNX; ++i) {
                xv[s][i] = *reinterpret_cast<const float4a *>(xr[i] + k);
                if (GATE) gv[s][i] = *reinterpret_cast<const float4a *>(gr[i] + k);
            }
#pragma unroll
            for (int i = 0; i < kNA; ++i) av[s][i] = *reinterpret_cast<const half8 *>(ar[i] + k);
        };
        auto put = [&](int s, int buf) {  // register set s into LDS
            uint8_t *to = stage + buf * F::kStage;
#pragma unroll
            for (int i = 0; i < kNX; ++i) {
                const floatx4 v = GATE ? gated(xv[s][i], gv[s][i]) : xv[s][i];
                half4 h, l;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    _Float16 a, b;
                    split(v[q], a, b);
                    h[q] = a, l[q] = b;
                }
                *reinterpret_cast<half4 *>(to + x_at[i]) = h;
                *reinterpret_cast<half4 *>(to + F::kX / 2 + x_at[i]) = l;
            }
#pragma unroll
            for (int i = 0; i < kNA; ++i) *reinterpret_cast<half8 *>(to + a_at[i]) = av[s][i];
        };
        floatx4 hi[F::kTiles], lo[F::kTiles];
#pragma unroll
        for (int q = 0; q < F::kTiles; ++q) hi[q] = lo[q] = floatx4{0.f, 0.f, 0.f, 0.f};
        const int step = wave % F::kStepWaves, rank0 = 16 * F::kTiles * (wave / F::kStepWaves);
        const int op = n * F::kRow + 64 * step + 16 * g;  // of an operand's row n in the stage
        load(0, 0);
        load(1, 1);
        __syncthreads();  // (a pass before: its output staging is read)
        put(0, 0);
        load(0, 2);
        // chunk c from LDS, chunk c + 1 into the other buffer, chunk c + 3 on its way
        for (int c0 = 0; c0 < chunks; c0 += 2) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                __syncthreads();
                if (c0 + u < chunks) {
                    const uint8_t *from = stage + u * F::kStage;
                    const half8 xh = *reinterpret_cast<const half8 *>(from + op), xl = *reinterpret_cast<const half8 *>(from + F::kX / 2 + op);
#pragma unroll
                    for (int q = 0; q < F::kTiles; ++q) {
                        const half8 aq = *reinterpret_cast<const half8 *>(from + F::kX + (rank0 + 16 * q) * F::kRow + op);
                        hi[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(aq, xh, hi[q], 0, 0, 0);
                        lo[q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(aq, xl, lo[q], 0, 0, 0);
                    }
                }
                put(u ^ 1, u ^ 1);
                load(u ^ 1, c0 + u + 3);
            }
        }
        __syncthreads();
        // the first columns' base and B, before the barriers of the sum
        constexpr int kS = (F::kR + 31) / 32, kCols = F::kCols, kCT = kCols / 16, kNB = kTile * kCols / 4 / 64;
        const int groups = (p.N + kCols - 1) / kCols;
        floatx4 old[2][kNB];
        half8 bv[2][kCT][kS];
        auto load_cols = [&](int s, int grp) {
            grp = min(grp, groups - 1);
#pragma unroll
            for (int i = 0; i < kNB; ++i) {
                const int e = lane + 64 * i, m = e / (kCols / 4), c = min(grp * kCols + 4 * (e % (kCols / 4)), p.N - 4);
                old[s][i] = *reinterpret_cast<const floatx4 *>(p.base + (m0 + min(m, tokens - 1)) * p.base_nb1 + 4 * c);
            }
#pragma unroll
            for (int u = 0; u < kCT; ++u)
#pragma unroll
                for (int q = 0; q < kS; ++q) {
                    const int c = min(grp * kCols + 16 * u, p.N - 16) + n, k = 32 * q + 8 * g;
                    bv[s][u][q] = *reinterpret_cast<const half8 *>(b + (int64_t)c * p.r + min(k, p.r - 8));
                    bv[s][u][q] = k < p.r ? bv[s][u][q] : half8{};  // past r: 0 (times t, 0 there)
                }
        };
        load_cols(0, wave);
        if (tid == 0) over = 0;
        float *part = reinterpret_cast<float *>(stage);  // [step wave][rank][token]
#pragma unroll
        for (int q = 0; q < F::kTiles; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                part[(step * F::kR + rank0 + 16 * q + 4 * g + i) * kTile + n] = fmaf(lo[q][i], 1.0f / 2048.0f, hi[q][i]);
        __syncthreads();
        for (int e = tid; e < F::kR * kTile; e += kThreads) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < F::kStepWaves; ++w) s += part[w * F::kR * kTile + e];
            s = e >> 4 < p.r ? s * sc : 0.0f;
            t[(e & 15) * kTRow + (e >> 4)] = s;
            // too large for fp16, or Inf or NaN of an x that is
            if (!(fabsf(s) < 65504.0f) && ids[e & 15] == cur) over = 1;
        }
        __syncthreads();
        // then t again in fp32, and 2^-e t of a token's own e in the columns
        float up = 1.0f, down = 1.0f;
        if (__builtin_expect(__builtin_amdgcn_readfirstlane(over) != 0, 0)) {
            rank_sums(p, cur, sc, m0, ids, t, kTRow);
            __syncthreads();
            float top = 0.0f;
            for (int j = 0; j < p.r; ++j) top = fmaxf(top, fabsf(t[n * kTRow + j]));
            const int e = max((int)(__float_as_uint(top) >> 23) - 127 - 14, 0);  // top 2^-e < 2^15
            down = __builtin_amdgcn_ldexpf(1.0f, -e), up = __builtin_amdgcn_ldexpf(1.0f, e);
        }
        // t of the lane's token, ranks 32q + 8g ..
        half8 th[kS], tl[kS];
#pragma unroll
        for (int q = 0; q < kS; ++q)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                _Float16 a, b;
                split(32 * q + 8 * g < F::kR ? t[n * kTRow + 32 * q + 8 * g + i] * down : 0.0f, a, b);
                th[q][i] = a, tl[q][i] = b;
            }
        // out^T = B t^T of kCols columns, turned in LDS so that base and out are whole rows of them
        uint8_t *turned = stage + wave * kTile * F::kOutRow;
        for (int g0 = wave; g0 < groups; g0 += 2 * kWaves) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int grp = g0 + s * kWaves;
                load_cols(s ^ 1, grp + kWaves);
                if (grp >= groups) continue;
#pragma unroll
                for (int u = 0; u < kCT; ++u) {
                    floatx4 h = {0.f, 0.f, 0.f, 0.f}, l = h;
#pragma unroll
                    for (int q = 0; q < kS; ++q) {
                        h = __builtin_amdgcn_mfma_f32_16x16x32_f16(bv[s][u][q], th[q], h, 0, 0, 0);
                        l = __builtin_amdgcn_mfma_f32_16x16x32_f16(bv[s][u][q], tl[q], l, 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) h[i] = fmaf(l[i], 1.0f / 2048.0f, h[i]) * up;
                    *reinterpret_cast<floatx4 *>(turned + n * F::kOutRow + 4 * (16 * u + 4 * g)) = h;
                }
                // (a wavefront's own staging: its LDS operations are in order)
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int i = 0; i < kNB; ++i) {
                    const int e = lane + 64 * i, m = e / (kCols / 4), c = grp * kCols + 4 * (e % (kCols / 4));
                    const floatx4 add = *reinterpret_cast<const floatx4 *>(turned + m * F::kOutRow + 16 * (e % (kCols / 4)));
                    const int own = ids[m];
                    floatx4 o;
#pragma unroll
                    for (int q = 0; q < 4; ++q) o[q] = own == cur ? old[s][i][q] + add[q] : old[s][i][q];
                    // (dst may be base: a value is read before it is written, by this wavefront alone;
                    // past L2, which the adapters need: 71 us against 74 at 4096 tokens)
                    if (c < p.N && (own == cur || (own == -1 && rest)))
                        __builtin_nontemporal_store(o, reinterpret_cast<floatx4 *>(p.dst + (m0 + m) * p.dst_nb1 + 4 * c));
                }
                __builtin_amdgcn_wave_barrier();
            }
        }
        rest = false;
    }
}

}  // namespace

int launch_lora_add(const sqa_tensor &base, const sqa_tensor &x, const sqa_tensor *gate, const sqa_tensor &a,
                    const sqa_tensor &b, const sqa_tensor &ids, const sqa_tensor *scale, const sqa_tensor &dst,
                    hipStream_t s) {
    const Params p{(const char *)base.data, (const char *)x.data, gate ? (const char *)gate->data : nullptr,
                   (int64_t)base.nb[1], (int64_t)x.nb[1], gate ? (int64_t)gate->nb[1] : 0, (int64_t)dst.nb[1],
                   (const _Float16 *)a.data, (const _Float16 *)b.data, (const int32_t *)ids.data,
                   scale ? (const float *)scale->data : nullptr, (char *)dst.data, (int)x.ne[0], (int)base.ne[0],
                   (int)a.ne[1], (int)a.ne[2], (int)x.ne[1]};
    const int prof = profile_start("lora_add", s);
    // A workgroup per token up to two a CU: with K 4096 and N 2048, 512 tokens that change
    // between 8 adapters take 12.8 us at rank 16, 26.7 at 64, 43.1 at 128, where tiles take
    // 32.3, 53.2, 83.4; that share them by 128 12.8, 26.7, 43.8 against 19.5, 30.7, 45.9. 768
    // that share take 18.7, 39.0, 62.8 against 22.8, 33.9, 50.1; that change 18.5, 38.7, 62.1
    // against 34.9, 55.4, 85.4. A token's workgroup reads its adapter whole out of L2: at rank 64
    // the 512 read 400 MB, 15 TB/s.
    if (p.M <= 512 && p.K <= 16 * 1024) {
        // (below 97 tokens parts of the columns fill the other CUs)
        const dim3 grid((unsigned)p.M, p.M <= 32 ? 4 : p.M <= 96 ? 2 : 1);
        if (p.K <= 4096) lora_token_kernel<1><<<grid, dim3(kThreads), 0, s>>>(p);
        else lora_token_kernel<4><<<grid, dim3(kThreads), 0, s>>>(p);
    } else {
        const dim3 grid((unsigned)((p.M + kTile - 1) / kTile), kPasses);
        typedef void (*Kernel)(Params);
        static const Kernel kernels[2][4] = {
            {lora_tile_kernel<1, false>, lora_tile_kernel<2, false>, lora_tile_kernel<4, false>, lora_tile_kernel<8, false>},
            {lora_tile_kernel<1, true>, lora_tile_kernel<2, true>, lora_tile_kernel<4, true>, lora_tile_kernel<8, true>}};
        static const int lds[4] = {Form<1>::kBytes, Form<2>::kBytes, Form<4>::kBytes, Form<8>::kBytes};
        static std::once_flag once;  // the LDS limit is raised once per process
        static hipError_t err = hipSuccess;
        std::call_once(once, [] {
            for (int g = 0; g < 2; ++g)
                for (int i = 0; i < 4; ++i)
                    if (err == hipSuccess)
                        err = hipFuncSetAttribute((const void *)kernels[g][i], hipFuncAttributeMaxDynamicSharedMemorySize, lds[i]);
        });
        if (err != hipSuccess) return hip_status(err, "lora_add LDS attribute");
        const int rt = p.r <= 16 ? 0 : p.r <= 32 ? 1 : p.r <= 64 ? 2 : 3;
        kernels[p.gate != nullptr][rt]<<<grid, dim3(kThreads), lds[rt], s>>>(p);
    }
    profile_stop(prof, s);
    return hip_status(hipGetLastError(), "lora_add launch");
}

}  // namespace sqa
