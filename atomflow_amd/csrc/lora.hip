// lora.hip — low-rank adapters of many requests beside a shared projection, for gfx950.
//
//   y_out[i, j] = y[i, j] + scale[a] * sum_r B[a, j, r] * v[i, s(j), r],   a = ids[i]
//   v[i, s, r]  = sum_k A[a, s, r, k] x[i, k],                             r < rank[a]
//
// Two launches. `down` computes v over tiles of up to 64 tokens; K is cut into at most eight parts,
// whose sums it leaves in the workspace, or adds itself where the tiles alone fill the device. `up`
// adds the parts, and its tiles' products to y. Both run on the matrix cores (16x16x32, fp16
// operands, fp32 sums), with the adapter's rows as the first operand and the tokens as the second,
// so a token's sums depend on no other token.
//
// Tokens come in any order. A tile's workgroups each take some of the adapters that its tokens
// name, every J-th from the j-th on, and gather that adapter's tokens, 16 to an operand: a prompt's
// tile has one adapter, a decode batch's up to 64, side by side, and the weights of each are read once
// per tile. No plan, no sort, no host data: ids, ranks and scales may change between the replays of a
// graph.
//
// Sums: K's parts and the order in which they are added are fixed by k alone, and every form adds
// a token's products in the same order, so a token's row has the same bits whatever the launch.
//
// Measured (down + up): 1 token, 4096 -> 6144 columns in three slices, rank 16: 4.0 + 4.6 us, two
// chains of loads; 45 tokens of 24 adapters, 4096 -> 28672, rank 32: 6.8 + 12.9 us (62 MB); 2011
// tokens, 14336 -> 4096, rank 16: 18.4 + 16.1 us (98 MB); 8192 tokens, 4096 -> 28672, rank 64:
// 45 + 225 us (y at 4.2 TB/s read and written).
#include <algorithm>
#include <type_traits>

#include "af_common.h"
#include "af_device.h"
#include "af_lora_split.h"

namespace af {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// y's rows start at any element
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kMaxSlices = AF_LORA_MAX_SLICES;
constexpr int kMaxRank = 128;
constexpr int kTile = 64;     // tokens of a tile: one to a lane
constexpr int kCols = 256;    // `up`: columns of a workgroup, the gathering form's
constexpr int kSpan = 1024;   // and the other one's
constexpr int kGroup = 8;     // `up`: column blocks that a tile's workgroups take one after the other
constexpr int kParts = kLoraParts;

struct LoraArgs {
    const uint16_t* x;
    int64_t x_stride;
    int m;
    const int32_t* ids;
    const uint16_t* a;      // [n_adapters][n_slices * rmax][k]
    const uint16_t* b;      // [n_adapters][n][rmax]
    const int32_t* ranks;
    const float* scales;
    int n_adapters, rmax, rows, k, n;  // rows = n_slices * rmax
    const void* y;
    int64_t y_stride;
    void* y_out;
    int64_t y_out_stride;
    float* v;               // [splits][m][rows]
    int parts, part_k;
    int splits;             // parts, or 1: `down` adds them
    int down_tile, down_tiles, down_items, down_side;  // `down`: tokens of a tile, tiles, (tile, rows, part)s
    int tiles, side;        // `up`: tiles of kTile tokens
    int n_slices;
    int slice_begin[kMaxSlices + 1];
    int slice_block[kMaxSlices + 1];  // `up`: first column block of each slice
    int items;                        // `up`: (column block, tile) pairs
};

__device__ __forceinline__ f16x8 load_f16x8(const uint16_t* p) {
    return __builtin_bit_cast(f16x8, *reinterpret_cast<const u32x4*>(p));
}

// The adapters that a tile's tokens name, in order of first appearance. Lane t holds token t's.
struct Adapters {
    uint64_t todo;
    int id;
    uint64_t mask;  // the tokens of the adapter that next() found
    int order;      // lane j: the j-th of them, counted in the tile
    int count;      // how many
    __device__ __forceinline__ Adapters(int id, bool valid) : todo(__ballot(valid)), id(id) {}
    // Skips `skip` adapters; false when there is none behind them.
    __device__ __forceinline__ bool next(int skip, int& adapter) {
        while (todo) {
            const int lead = __builtin_ctzll(todo);
            adapter = __builtin_amdgcn_readlane(id, lead);
            mask = __ballot(id == adapter) & todo;
            todo &= ~mask;
            if (skip-- > 0) continue;
            // the adapter's tokens to the front lanes, the others behind them
            const int lane = threadIdx.x & 63;
            const uint64_t below = (uint64_t(1) << lane) - 1;
            count = __builtin_popcountll(mask);
            const int before = __builtin_popcountll(mask & below);
            const int to = (mask >> lane) & 1 ? before : count + lane - before;
            order = __builtin_amdgcn_ds_permute(4 * to, lane);
            return true;
        }
        return false;
    }
    // Token of place j (the last one where there are fewer).
    __device__ __forceinline__ int token(int j) const { return __shfl(order, min(j, count - 1)); }
};

__device__ __forceinline__ int rank_of(const LoraArgs& p, int adapter) {
    return p.ranks ? min(max(p.ranks[adapter], 0), p.rmax) : p.rmax;
}

// Workgroups go round the eight XCDs. An item has `side` of them, which share out its tile's
// adapters: first every item's first one, then every item's second one, most of which find nothing
// to do. (Workgroups start in order, dealt out to an XCD's shader engines in turn, and one that
// finds no room there keeps those behind it waiting. Side by side instead, two to an item, all
// first ones fell on half of the engines, at twice the time; and the order is one further in each
// round, so that a tile of many adapters has its workgroups on different engines.)
struct Turn {
    int xcd, nth, skip;  // nth item of the XCD
    __device__ __forceinline__ explicit Turn(int items) {
        const int per_xcd = (items + 7) / 8, i = int(blockIdx.x) / 8;
        xcd = int(blockIdx.x) % 8;
        skip = i / per_xcd;
        nth = (i + skip) % per_xcd;
    }
};

// ---- down: v ------------------------------------------------------------------------------
// A part of K is four chains of products, each from zero, added one after the other; then the parts
// are. MT 16-token tiles by NT 16-row tiles of A in every wave, operands straight from memory into
// registers.
template <int MT, int NT>
struct Operands {
    const uint16_t* x[MT];
    const uint16_t* a[NT];
    __device__ __forceinline__ Operands(const LoraArgs& p, const Adapters& some, int t0, int base, int adapter,
                                        int rank, int row0, int lane) {
        const int sub = 8 * (lane >> 4);
#pragma unroll
        for (int i = 0; i < MT; ++i)
            x[i] = p.x + size_t(t0 + some.token(base + 16 * i + (lane & 15))) * p.x_stride + sub;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int r = row0 + 16 * i + (lane & 15);
            const bool ok = r < p.rows && r % p.rmax < rank;
            // (a row past the rank touches its own sums alone, and those are not used)
            a[i] = p.a + (size_t(adapter) * p.rows + (ok ? r : row0)) * p.k + sub;
        }
    }
};

template <int MT, int NT, int U>
__device__ __forceinline__ void multiply(const f16x8 (&xf)[U][MT], const f16x8 (&af)[U][NT], int u,
                                         f32x4 (&acc)[MT][NT]) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(af[u][j], xf[u][i], acc[i][j], 0, 0, 0);
}

// A tile's sum s to v. Lane: token lane & 15, rows 4 * (lane >> 4) ... of the tile.
__device__ __forceinline__ void store_v(const LoraArgs& p, const Adapters& some, int split, int t0, int place, int r,
                                        int rank, f32x4 s) {
    const int token = some.token(place);
    if (place < some.count && r < p.rows) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if ((r + e) % p.rmax >= rank) s[e] = 0.0f;
        *reinterpret_cast<f32x4*>(p.v + (size_t(split) * p.m + t0 + token) * p.rows + r) = s;
    }
}

// Up to 16 tokens of an adapter, from place `base` on, by all four waves: of each of the parts, a
// wave takes one chain, kUnroll steps' loads before the first product; the four sums meet in LDS.
template <int NT>
__device__ __forceinline__ void few_tokens(const LoraArgs& p, const Adapters& todo, f32x4 (&sums)[4][NT][64], int t0,
                                           int base, int adapter, int rank, int row0, int part0, int part1,
                                           int split, int lane, int wave) {
    constexpr int kUnroll = 4, kOwn = (NT + 3) / 4;
    const Operands<1, NT> at(p, todo, t0, base, adapter, rank, row0, lane);
    const int sub = 8 * (lane >> 4), kw = p.part_k / 4;
    f32x4 total[kOwn] = {};
#pragma unroll 1
    for (int part = part0; part < part1; ++part) {
        f32x4 acc[1][NT] = {};
        f16x8 xf[kUnroll][1], af[kUnroll][NT];
        int k = part * p.part_k + wave * kw;
        const int k1 = min(k + kw, p.k);
#pragma unroll 1
        for (; k + 32 * kUnroll <= k1; k += 32 * kUnroll) {
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                xf[u][0] = load_f16x8(at.x[0] + k + 32 * u);
#pragma unroll
                for (int i = 0; i < NT; ++i) af[u][i] = load_f16x8(at.a[i] + k + 32 * u);
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) multiply<1, NT>(xf, af, u, acc);
        }
        if (k < k1) {  // k is a multiple of 8: whole pieces of 8, or none
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const bool in = k + 32 * u + sub < k1;
                if (k + 32 * u >= k1) break;
                xf[u][0] = in ? load_f16x8(at.x[0] + k + 32 * u) : f16x8{};
#pragma unroll
                for (int i = 0; i < NT; ++i) af[u][i] = in ? load_f16x8(at.a[i] + k + 32 * u) : f16x8{};
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                if (k + 32 * u >= k1) break;
                multiply<1, NT>(xf, af, u, acc);
            }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) sums[wave][j][lane] = acc[0][j];
        __syncthreads();
#pragma unroll
        for (int o = 0; o < kOwn; ++o) {
            const int t = min(wave + 4 * o, NT - 1);
            total[o] += ((sums[0][t][lane] + sums[1][t][lane]) + sums[2][t][lane]) + sums[3][t][lane];
        }
        __syncthreads();
    }
#pragma unroll
    for (int o = 0; o < kOwn; ++o) {
        const int t = wave + 4 * o;
        if (t >= NT) break;
        store_v(p, todo, split, t0, base + (lane & 15), row0 + 16 * t + 4 * (lane >> 4), rank, total[o]);
    }
}

// Few tiles: a workgroup takes one part and 16 rows (with 64 rows a workgroup, 2 tokens, 13952 ->
// twice rank 64 took 10.7 us instead of 5.4).
__global__ __launch_bounds__(256) void lora_down_kernel(const LoraArgs p) {
    __shared__ f32x4 sums[4][1][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const Turn turn(p.down_items);
    const int item = 8 * turn.nth + turn.xcd;
    if (item >= p.down_items) return;
    const int t0 = item % p.down_tiles * p.down_tile, rest = item / p.down_tiles;
    const int part = rest % p.parts, row0 = rest / p.parts * 16;
    int id = -1;
    if (lane < p.down_tile && t0 + lane < p.m) id = p.ids[t0 + lane];
    Adapters todo(id, id >= 0 && id < p.n_adapters);
    int adapter;
    for (int skip = turn.skip; todo.next(skip, adapter); skip = p.down_side - 1) {
        const int rank = rank_of(p, adapter);
        if (rank == 0) continue;
#pragma unroll 1
        for (int base = 0; base < todo.count; base += 16)
            few_tokens<1>(p, todo, sums, t0, base, adapter, rank, row0, part, part + 1, part, lane, wave);
    }
}

// More tiles: 64 tokens by 16 NT rows, all waves on the same 64 of K at a time, which memory writes
// straight to LDS (two pieces of 64 ahead), 8 lanes to the 128 bytes of a row. Neighbouring lanes
// of a first or second operand are rows apart, so that loading operands from memory costs the
// address unit 64 cycles an instruction; this way it is 16. A wave takes 16 of the tokens. With
// p.splits a workgroup takes one part of K, else all of them.
template <int NT>
__global__ __launch_bounds__(256) void lora_down_lds_kernel(const LoraArgs p) {
    constexpr int kRows = kTile + 16 * NT;       // LDS: the tokens' rows of x, then rows of A, of 128 bytes
    constexpr int kStages = 3;  // (with 6, two workgroups to a compute unit instead of three: 20 us became 30)
    constexpr int kLoadsA = (2 * NT + 3) / 4, kLoads = 2 + kLoadsA;  // of a wave, for each piece
    __shared__ __attribute__((aligned(1024))) uint8_t stage[kStages][kRows * 128];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const Turn turn(p.down_items);
    const int item = 8 * turn.nth + turn.xcd;
    if (item >= p.down_items) return;
    const int t0 = item % p.down_tiles * kTile, rest = item / p.down_tiles;
    const int split = rest % p.splits, row0 = rest / p.splits * (16 * NT);
    int id = -1;
    if (t0 + lane < p.m) id = p.ids[t0 + lane];
    Adapters todo(id, id >= 0 && id < p.n_adapters);
    const LoraRange range = lora_range(p.k, p.part_k, p.splits, split);
    const int k0 = range.k0, pieces = range.pieces;  // (one at least: no part is empty)
    const uint32_t lds0 = lds_address(stage);

    int adapter;
    for (int skip = turn.skip; todo.next(skip, adapter); skip = p.down_side - 1) {
        const int rank = rank_of(p, adapter);
        if (rank == 0) continue;
        if (todo.count <= 16) {
            const int part = p.splits == 1 ? 0 : split;
            few_tokens<NT>(p, todo, *reinterpret_cast<f32x4(*)[4][NT][64]>(stage), t0, 0, adapter, rank, row0, part,
                           p.splits == 1 ? p.parts : part + 1, split, lane, wave);
            continue;
        }
        // Load j of a lane: row 8 j + lane / 8 of its 16 bytes; rows' 16 bytes are kept in the
        // order (piece ^ row) & 7, so that an operand's lanes read different banks.
        const int in_row = lane >> 3, piece = (lane & 7) ^ in_row;
        const uint16_t* from[kLoads];
        uint32_t to[kLoads];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = 16 * wave + 8 * j + in_row;
            from[j] = p.x + size_t(t0 + todo.token(r)) * p.x_stride + k0 + 8 * piece;
            to[j] = lds0 + uint32_t(16 * wave + 8 * j) * 128;
        }
#pragma unroll
        for (int j = 0; j < kLoadsA; ++j) {
            const int first = 8 * ((wave + 4 * j) % (2 * NT));  // (two waves may load the same rows)
            const int r = row0 + first + in_row;
            const bool ok = r < p.rows && r % p.rmax < rank;
            // (a row past the rank, or a place past the tokens, touches its own sums alone)
            from[2 + j] = p.a + (size_t(adapter) * p.rows + (ok ? r : row0)) * p.k + k0 + 8 * piece;
            to[2 + j] = lds0 + uint32_t(kTile + first) * 128;
        }
        constexpr uint32_t kBytes = kRows * 128;
        uint32_t fill = 0;  // the next load's place
        int ahead = pieces;  // loads to come
        auto load = [&] {
            if (ahead <= 0) return;
            // (past K the loads repeat what is there)
            const int back = --ahead == 0 ? lora_pull_back(p.k, range, piece) : 0;
#pragma unroll
            for (int j = 0; j < kLoads; ++j) {
                lds_dma16(from[j] + back, to[j] + fill);
                from[j] += 64;
            }
            fill = fill == (kStages - 1) * kBytes ? 0 : fill + kBytes;
        };
        for (int i = 0; i < kStages - 1; ++i) load();
        const bool mine = 16 * wave < todo.count;
        const int chain = p.part_k / 256;  // pieces of a chain
        int in_chain = chain, chains = 4;  // left
        uint32_t take = 0;
        f32x4 acc[1][NT] = {}, part[NT] = {}, total[NT] = {};
#pragma unroll 1
        for (int left = pieces; left > 0; --left) {
            // the piece is there when at most the loads of the next one are on their way
            if (left > 1)
                wait_vmcnt<kLoads>();
            else
                wait_vmcnt<0>();
            __syncthreads();  // (and every wave is done with the piece before, whose place the next load takes)
            load();
            if (mine) {
                const uint8_t* at = stage[0] + take + (lane & 15) * 128;
                f16x8 xf[2][1], af[2][NT];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int slot = 16 * (((4 * u + (lane >> 4)) ^ lane) & 7);
                    auto get = [&](int row) {
                        return __builtin_bit_cast(f16x8, *reinterpret_cast<const u32x4*>(at + slot + row * 128));
                    };
                    xf[u][0] = get(16 * wave);
#pragma unroll
                    for (int j = 0; j < NT; ++j) af[u][j] = get(kTile + 16 * j);
                }
                if (left == 1) {
                    const int k = k0 + 64 * (pieces - 1) + 8 * (lane >> 4);
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        if (k + 32 * u >= p.k) {
                            xf[u][0] = f16x8{};
#pragma unroll
                            for (int j = 0; j < NT; ++j) af[u][j] = f16x8{};
                        }
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) multiply<1, NT>(xf, af, u, acc);
                if (--in_chain == 0 || left == 1) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) part[j] += acc[0][j], acc[0][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    in_chain = chain;
                    if (--chains == 0 || left == 1) {
#pragma unroll
                        for (int j = 0; j < NT; ++j) total[j] += part[j], part[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                        chains = 4;
                    }
                }
            }
            take = take == (kStages - 1) * kBytes ? 0 : take + kBytes;
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
            store_v(p, todo, split, t0, 16 * wave + (lane & 15), row0 + 16 * j + 4 * (lane >> 4), rank, total[j]);
        // The next adapter writes here. No load is on its way: each wave has awaited its last piece's
        // (there is one), and stands behind every other wave's wait since that piece's barrier.
        __syncthreads();
    }
}

// ---- up: y_out = y + scale * B v ------------------------------------------------------------
// v in two fp16 halves, v = 2^e (hi + lo): 22 bits, so that fp16 matrix instructions lose nothing
// that fp32 sums would keep (one fp16 half alone would be off by half a step of fp16, as much as
// y's own rounding). e follows the token's largest v, so that neither half leaves fp16's range.
__device__ __forceinline__ int scale_exponent(float top) {
    const int e = int((__builtin_bit_cast(uint32_t, top) >> 23) & 255) - 127;
    return e == 128 ? 0 : max(e, -100) - 12;  // largest v to [2^12, 2^13); not finite: as it is
}

__device__ __forceinline__ float pow2f(int e) { return __builtin_ldexpf(1.0f, e); }

// Eight neighbouring elements of y as they lie in memory; load_part and store_part: n of them, 1 ..
// 8.
template <typename Y>
struct Run8;
template <>
struct Run8<uint16_t> {
    u32x4 w;
    __device__ __forceinline__ void load(const uint16_t* p) { w = *reinterpret_cast<const u32x4_a2*>(p); }
    __device__ __forceinline__ void store(uint16_t* p) const { *reinterpret_cast<u32x4_a2*>(p) = w; }
    __device__ __forceinline__ void load_part(const uint16_t* p, int n) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = p[min(2 * i, n - 1)] | uint32_t(p[min(2 * i + 1, n - 1)]) << 16;
    }
    __device__ __forceinline__ void store_part(uint16_t* p, int n) const {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = uint16_t(w[i >> 1] >> (16 * (i & 1)));
    }
    __device__ __forceinline__ float get(int i) const { return h2f(uint16_t(w[i >> 1] >> (16 * (i & 1)))); }
    __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = uint32_t(f2h(v[2 * i])) | (uint32_t(f2h(v[2 * i + 1])) << 16);
    }
};
template <>
struct Run8<float> {
    f32x4 w[2];
    __device__ __forceinline__ void load(const float* p) {
        w[0] = *reinterpret_cast<const f32x4_a4*>(p);
        w[1] = *reinterpret_cast<const f32x4_a4*>(p + 4);
    }
    __device__ __forceinline__ void store(float* p) const {
        *reinterpret_cast<f32x4_a4*>(p) = w[0];
        *reinterpret_cast<f32x4_a4*>(p + 4) = w[1];
    }
    __device__ __forceinline__ void load_part(const float* p, int n) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i >> 2][i & 3] = p[min(i, n - 1)];
    }
    __device__ __forceinline__ void store_part(float* p, int n) const {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = w[i >> 2][i & 3];
    }
    __device__ __forceinline__ float get(int i) const { return w[i >> 2][i & 3]; }
    __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i >> 2][i & 3] = v[i];
    }
};

// v's fp16 halves of a tile, in LDS: rows of 32 KS ranks and 16 bytes.
template <int KS>
struct Halves {
    static constexpr int kLd = 32 * KS + 8;
    static constexpr int kPer = 8 * KS;  // threads that work on a token's v, four ranks each
    __attribute__((aligned(16))) uint16_t hi[kTile * kLd];
    __attribute__((aligned(16))) uint16_t lo[kTile * kLd];
    float back[kTile];
    // Ranks r0 .. r0 + 3 of slice s of token t: the parts' sums, times the scale.
    static __device__ __forceinline__ f32x4 load(const LoraArgs& p, int t, int s, int r0, float scale,
                                                 bool split) {
        const float* src = p.v + size_t(t) * p.rows + s * p.rmax + r0;
        f32x4 v = *reinterpret_cast<const f32x4*>(src);
        if (split) {
            const size_t step = size_t(p.m) * p.rows;
            f32x4 part[kParts];
#pragma unroll
            for (int q = 1; q < kParts; ++q)
                part[q] = *reinterpret_cast<const f32x4*>(src + min(q, p.splits - 1) * step);
#pragma unroll
            for (int q = 1; q < kParts; ++q)
                if (q < p.splits) v += part[q];
        }
        return v * scale;
    }
    // The kPer threads of a place bring its v, in neighbouring lanes.
    __device__ __forceinline__ void put(int place, int r0, f32x4 v) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, __builtin_bit_cast(uint32_t, float(v[i])) & 0x7fffffffu);
#pragma unroll
        for (int o = 1; o < kPer; o *= 2) top = max(top, uint32_t(__shfl_xor(int(top), o)));
        const int e = scale_exponent(__builtin_bit_cast(float, top));
        const float down = pow2f(-e);
        uint16_t h[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float w = v[i] * down;
            h[i] = f2h(w);
            l[i] = (h[i] & 0x7c00u) == 0x7c00u ? uint16_t(0) : f2h(w - h2f(h[i]));
        }
        auto two = [](const uint16_t(&x)[4], int i) { return uint32_t(x[i]) | (uint32_t(x[i + 1]) << 16); };
        *reinterpret_cast<uint2*>(hi + place * kLd + r0) = make_uint2(two(h, 0), two(h, 2));
        *reinterpret_cast<uint2*>(lo + place * kLd + r0) = make_uint2(two(l, 0), two(l, 2));
        if (r0 == 0) back[place] = pow2f(e);
    }
};

// 64 columns of an adapter's B as four first operands: row 4 g + i of the t-th (g, i the result's
// lane group and element) is column 32 (t / 2) + 8 g + 4 (t % 2) + i, so that a lane ends up with
// two runs of 8 columns of one token, and a token's four lanes with 64 (fp16) bytes in a row.
template <int KS>
struct Columns {
    f16x8 f[4][KS];
    // From column c on, those below col1 (the others repeat the last one).
    __device__ __forceinline__ void load(const LoraArgs& p, int adapter, int c, int col1, int rank, int lane) {
        const int from = min(c, col1 - 1);
        const int last = (rank - 1) & ~7;  // (ranks of the adapter alone are read)
        const uint16_t* at = p.b + (size_t(adapter) * p.n + from) * p.rmax;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int r = lane & 15;
            const int col = 32 * (t >> 1) + 8 * (r >> 2) + 4 * (t & 1) + (r & 3);
            const int off = min(col, col1 - 1 - from) * p.rmax;
#pragma unroll
            for (int q = 0; q < KS; ++q)
                f[t][q] = load_f16x8(at + off + min(32 * q + 8 * (lane >> 4), last));
        }
    }
    // What lies behind the adapter's rank is not used.
    __device__ __forceinline__ void cut(int rank, int lane) {
#pragma unroll
        for (int q = 0; q < KS; ++q) {
            u32x4 keep;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 32 * q + 8 * (lane >> 4) + 2 * i;
                keep[i] = (r < rank ? 0xffffu : 0u) | (r + 1 < rank ? 0xffff0000u : 0u);
            }
#pragma unroll
            for (int t = 0; t < 4; ++t)
                f[t][q] = __builtin_bit_cast(f16x8, __builtin_bit_cast(u32x4, f[t][q]) & keep);
        }
    }
    // acc = B (hi + lo) of 16 places.
    __device__ __forceinline__ void product(const Halves<KS>& v, int place, int lane, f32x4 (&acc)[4]) const {
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int q = 0; q < KS; ++q) {
            const f16x8 h = load_f16x8(v.hi + place * Halves<KS>::kLd + 32 * q + 8 * (lane >> 4));
            const f16x8 l = load_f16x8(v.lo + place * Halves<KS>::kLd + 32 * q + 8 * (lane >> 4));
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[u][q], l, acc[u], 0, 0, 0);
                acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[u][q], h, acc[u], 0, 0, 0);
            }
        }
    }
};

// y += up * sum
template <typename Y>
__device__ __forceinline__ void add_run(Run8<Y>& y, const f32x4 (&sum)[2], float up) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = y.get(e) + up * sum[e >> 2][e & 3];
    y.set(v);
}
template <typename Y>
__device__ __forceinline__ void add_run(Run8<Y>& y, const f32x4 (&acc)[4], int half, float up) {
    const f32x4 sum[2] = {acc[2 * half], acc[2 * half + 1]};
    add_run(y, sum, up);
}

// Where a workgroup of `up` works: each XCD gets neighbouring items, which are the tiles by kGroup
// column blocks (whose part of B stays in its L2), then the next column blocks.
struct Place {
    bool any;
    int s, t0, col0, col1;
    __device__ __forceinline__ Place(const LoraArgs& p, const Turn& turn, int tile, int cols) {
        const int item = turn.xcd * ((p.items + 7) / 8) + turn.nth;
        any = item < p.items;
        const int group = item / (p.tiles * kGroup), in_group = item - group * (p.tiles * kGroup);
        const int width = max(1, min(kGroup, p.slice_block[p.n_slices] - group * kGroup));
        const int block = group * kGroup + in_group % width;
        t0 = in_group / width * tile;
        s = 0;
        while (s + 1 < p.n_slices && block >= p.slice_block[s + 1]) ++s;
        col0 = p.slice_begin[s] + (block - p.slice_block[s]) * cols;
        col1 = min(col0 + cols, p.slice_begin[s + 1]);
    }
};

// A tile's rows as they are (no adapter, or one of rank 0): columns [col0, col1) of its gathered
// tokens.
template <typename Y>
__device__ __forceinline__ void copy_rows(const LoraArgs& p, const Adapters& some, int t0, int col0, int col1) {
    const int runs = (col1 - col0 + 7) / 8, total = some.count * runs;
#pragma unroll 1
    for (int from = threadIdx.x; from - int(threadIdx.x) < total; from += 4 * 256) {
        Run8<Y> r[4];
        const Y* src[4];
        Y* dst[4];
        int n[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = min(from + 256 * u, total - 1);
            const int t = t0 + some.token(i / runs), col = col0 + 8 * (i % runs);
            n[u] = col1 - col;
            src[u] = static_cast<const Y*>(p.y) + size_t(t) * p.y_stride + col;
            dst[u] = static_cast<Y*>(p.y_out) + size_t(t) * p.y_out_stride + col;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (n[u] >= 8)
                r[u].load(src[u]);
            else
                r[u].load_part(src[u], n[u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (from + 256 * u >= total) continue;
            if (n[u] >= 8)
                r[u].store(dst[u]);
            else
                r[u].store_part(dst[u], n[u]);
        }
    }
}

// A slice's last columns [c, col1), fewer than 64, of an adapter's gathered tokens.
template <int KS, typename Y>
__device__ __forceinline__ void last_columns(const LoraArgs& p, const Adapters& some, const Columns<KS>& b,
                                             const Halves<KS>& halves, int t0, int c, int col1, int lane) {
    const int sub = c + 8 * (lane >> 4), n = col1 - sub;
#pragma unroll 1
    for (int base = 0; base < some.count; base += 16) {
        const int place = base + (lane & 15);
        const size_t t = size_t(t0 + some.token(place));
        f32x4 acc[4];
        b.product(halves, place, lane, acc);
        const float up = halves.back[place];
        const Y* from = static_cast<const Y*>(p.y) + t * p.y_stride + sub;
        Y* to = static_cast<Y*>(p.y_out) + t * p.y_out_stride + sub;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (place >= some.count || n <= 32 * h) continue;
            Run8<Y> z;
            z.load_part(from + 32 * h, n - 32 * h);
            add_run(z, acc, h, up);
            z.store_part(to + 32 * h, n - 32 * h);
        }
    }
}

// Many tiles: a tile's tokens of one adapter, gathered, by kSpan columns of one slice; rank up to
// 32 KS. v is read and cut in halves once; then each wave takes 64 columns at a time, whose B and y
// have been on their way since the 64 columns before. The products go through LDS, 16 tokens at a
// time, to lanes that have y as it lies in memory: 8 lanes to the 64 columns of a token. (With a
// token's y in the lanes that hold its products, neighbouring lanes are rows apart, and the address
// unit takes 64 cycles for an instruction instead of 16.)
template <int MT, int KS, typename Y>
__global__ __launch_bounds__(256, 2) void lora_up_span_kernel(const LoraArgs p) {
    constexpr int kPer = Halves<KS>::kPer, kSlots = 256 / kPer;
    constexpr int kTurnLd = 68;  // (16 rows of 16 bytes fall on different banks)
    __shared__ Halves<KS> halves;
    __shared__ __attribute__((aligned(16))) float turned[4][16 * kTurnLd];
    int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const Turn turn(p.items);
    const Place at(p, turn, kTile, kSpan);
    if (!at.any) return;
    const bool copy = p.y != p.y_out;  // tokens without an adapter are copied
    int id = -1;
    const bool token_in = at.t0 + lane < p.m;
    if (token_in) id = p.ids[at.t0 + lane];
    if (id < 0 || id >= p.n_adapters) id = -1;
    Adapters todo(id, token_in && (copy || id >= 0));
    const int first = at.col0 + 64 * wave;
    const int end = at.col0 + (at.col1 - at.col0) / 64 * 64;  // of the whole runs of 64 columns

    int adapter;
    for (int skip = turn.skip; todo.next(skip, adapter); skip = p.side - 1) {
        asm volatile("" : "+v"(lane));  // (what hangs on the lane is not worked out, and kept, before)
        const int rank = adapter >= 0 ? rank_of(p, adapter) : 0;
        if (rank == 0) {  // y as it is, bit for bit
            if (copy) copy_rows<Y>(p, todo, at.t0, at.col0, at.col1);
            continue;
        }
        const float scale = p.scales ? p.scales[adapter] : 1.0f;
        const int r0 = lane % kPer * 4;
#pragma unroll 1
        for (int base = 0; base < todo.count; base += kSlots) {
            const int place = base + (64 * wave + lane) / kPer;
            const int t = at.t0 + todo.token(place);
            f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
            if (place < todo.count && r0 < rank) v = Halves<KS>::load(p, t, at.s, r0, scale, p.splits > 1);
            halves.put(place, r0, v);
        }
        __syncthreads();
        for (int base = 0; base < todo.count; base += 16 * MT) {
            if (first >= end) break;
            // run j of a lane: token 8 j + lane / 8, columns 8 (lane % 8) ...
            const Y* from[2 * MT];
            Y* to[2 * MT];
#pragma unroll
            for (int j = 0; j < 2 * MT; ++j) {
                const size_t t = size_t(at.t0 + todo.token(base + 8 * j + (lane >> 3)));
                from[j] = static_cast<const Y*>(p.y) + t * p.y_stride + 8 * (lane & 7);
                to[j] = static_cast<Y*>(p.y_out) + t * p.y_out_stride + 8 * (lane & 7);
            }
            auto load_y = [&](Run8<Y>(&y)[2 * MT], int c) {
#pragma unroll
                for (int j = 0; j < 2 * MT; ++j)
                    y[j].load(from[j] + c);
            };
            auto work = [&](Run8<Y>(&y)[2 * MT], Columns<KS>& b, int c) {
                b.cut(rank, lane);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    f32x4 acc[4];
                    b.product(halves, base + 16 * i + (lane & 15), lane, acc);
                    float* put = turned[wave] + (lane & 15) * kTurnLd + 8 * (lane >> 4);
                    asm volatile("" ::: "memory");  // (the wave's own LDS operations keep their order)
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        *reinterpret_cast<f32x4*>(put + 32 * (t >> 1) + 4 * (t & 1)) = acc[t];
                    asm volatile("" ::: "memory");
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int j = 2 * i + h, place = base + 8 * j + (lane >> 3);
                        const float* get = turned[wave] + (8 * h + (lane >> 3)) * kTurnLd + 8 * (lane & 7);
                        const f32x4 sum[2] = {*reinterpret_cast<const f32x4*>(get),
                                              *reinterpret_cast<const f32x4*>(get + 4)};
                        add_run(y[j], sum, halves.back[place]);
                        if (place < todo.count) y[j].store(to[j] + c);
                    }
                }
            };
            // Two sets of registers in turn. The loads ahead are not conditional (past the end they
            // repeat the last columns): a branch would make the compiler copy, and so await, them.
            Columns<KS> b0, b1;
            Run8<Y> y0[2 * MT], y1[2 * MT];
            const int last = first + (end - 1 - first) / 256 * 256;
            b0.load(p, adapter, first, at.col1, rank, lane);
            load_y(y0, first);
            int c = first;
#pragma unroll 1
            for (; c + 256 < end; c += 512) {
                b1.load(p, adapter, c + 256, at.col1, rank, lane);
                load_y(y1, c + 256);
                work(y0, b0, c);
                b0.load(p, adapter, min(c + 512, last), at.col1, rank, lane);
                load_y(y0, min(c + 512, last));
                work(y1, b1, c + 256);
            }
            if (c < end) work(y0, b0, c);
        }
        if (end < at.col1 && wave == (end - at.col0) / 64 % 4) {
            Columns<KS> b;
            b.load(p, adapter, end, at.col1, rank, lane);
            b.cut(rank, lane);
            last_columns<KS, Y>(p, todo, b, halves, at.t0, end, at.col1, lane);
        }
        __syncthreads();
    }
}

// Fewer tiles: a tile's tokens of one adapter, gathered, by 256 columns of one slice, 64 to a wave.
// B and y of the first 16 tokens are on their way while v is read and cut in halves. (64 tokens at
// a time measured the same or, 2011 tokens by 4096 columns, 19 us instead of 17.)
template <int KS, typename Y>
__global__ __launch_bounds__(256, KS == 1 ? 5 : KS == 2 ? 4 : 3) void lora_up_kernel(const LoraArgs p) {
    constexpr int kPer = Halves<KS>::kPer, kSlots = 256 / kPer;  // tokens whose v is read at a time
    __shared__ Halves<KS> halves;
    int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const Turn turn(p.items);
    const Place at(p, turn, kTile, kCols);
    if (!at.any) return;
    const int c = at.col0 + 64 * wave;     // the wave's columns,
    const bool whole = c + 64 <= at.col1;  // all of which there are

    const bool copy = p.y != p.y_out;  // tokens without an adapter are copied
    int id = -1;
    const bool token_in = at.t0 + lane < p.m;
    if (token_in) id = p.ids[at.t0 + lane];
    if (id < 0 || id >= p.n_adapters) id = -1;
    Adapters todo(id, token_in && (copy || id >= 0));

    int adapter;
    for (int skip = turn.skip; todo.next(skip, adapter); skip = p.side - 1) {
        asm volatile("" : "+v"(lane));  // (what hangs on the lane is not worked out, and kept, before)
        const int rank = adapter >= 0 ? rank_of(p, adapter) : 0;
        if (rank == 0) {  // y as it is, bit for bit
            if (copy) copy_rows<Y>(p, todo, at.t0, at.col0, at.col1);
            continue;
        }
        Columns<KS> b;
        b.load(p, adapter, c, at.col1, rank, lane);
        // Tokens from place `base` on, 16 to a tile. (A place past the adapter's tokens reads the
        // last one's y.)
        auto row = [&](int place, int64_t stride) {
            return size_t(at.t0 + todo.token(place)) * stride + c + 8 * (lane >> 4);
        };
        Run8<Y> y[2];
        auto load_y = [&](int base) {
            const Y* run = static_cast<const Y*>(p.y) + row(base + (lane & 15), p.y_stride);
            run = whole ? run : reinterpret_cast<const Y*>(p.v);  // (anything that is there)
            y[0].load(run);
            y[1].load(run + 32);
        };
        load_y(0);
        const float scale = p.scales ? p.scales[adapter] : 1.0f;
        const int r0 = lane % kPer * 4;
#pragma unroll 1
        for (int base = 0; base < todo.count; base += kSlots) {
            const int place = base + (64 * wave + lane) / kPer;
            const int t = at.t0 + todo.token(place);
            f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
            if (place < todo.count && r0 < rank) v = Halves<KS>::load(p, t, at.s, r0, scale, p.splits > 1);
            halves.put(place, r0, v);
        }
        __syncthreads();
        b.cut(rank, lane);
        if (whole) {
#pragma unroll 1
            for (int base = 0; base < todo.count; base += 16) {
                if (base > 0) load_y(base);
                const int place = base + (lane & 15);
                f32x4 acc[4];
                b.product(halves, place, lane, acc);
                const float up = halves.back[place];
                add_run(y[0], acc, 0, up);
                add_run(y[1], acc, 1, up);
                Y* run = static_cast<Y*>(p.y_out) + row(place, p.y_out_stride);
                if (place < todo.count) {
                    y[0].store(run);
                    y[1].store(run + 32);
                }
            }
        } else if (c < at.col1) {  // the slice's last columns, fewer than 64
            last_columns<KS, Y>(p, todo, b, halves, at.t0, c, at.col1, lane);
        }
        __syncthreads();
    }
}

// ---- launch ---------------------------------------------------------------------------------
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int lora_check(const af_lora* l) {
    if (!l || l->n_adapters <= 0 || l->max_rank <= 0 || l->n_slices <= 0 || l->k <= 0 || l->n <= 0)
        return AF_ERR_INVALID_ARG;
    if (l->max_rank % 8 || l->max_rank > kMaxRank || l->n_slices > kMaxSlices || l->k % 8 ||
        l->k > (1 << 24) || l->n > (1 << 24) || l->n_adapters > (1 << 20))
        return AF_ERR_UNSUPPORTED;
    int begin = 0;
    for (int s = 0; s < l->n_slices; ++s) {
        if (l->slice_end[s] <= begin) return AF_ERR_INVALID_ARG;
        begin = l->slice_end[s];
    }
    return begin == l->n ? AF_OK : AF_ERR_INVALID_ARG;
}

void launch_down_lds(const LoraArgs& p, dim3 grid, int nt, hipStream_t s) {
    switch (nt) {
        case 1: hipLaunchKernelGGL(lora_down_lds_kernel<1>, grid, dim3(256), 0, s, p); break;
        case 2: hipLaunchKernelGGL(lora_down_lds_kernel<2>, grid, dim3(256), 0, s, p); break;
        case 3: hipLaunchKernelGGL(lora_down_lds_kernel<3>, grid, dim3(256), 0, s, p); break;
        default: hipLaunchKernelGGL(lora_down_lds_kernel<4>, grid, dim3(256), 0, s, p); break;
    }
}

template <int MT, typename Y>
void launch_up_span(const LoraArgs& p, dim3 grid, hipStream_t s) {
    if (p.rmax <= 32)
        hipLaunchKernelGGL((lora_up_span_kernel<MT, 1, Y>), grid, dim3(256), 0, s, p);
    else if (p.rmax <= 64)
        hipLaunchKernelGGL((lora_up_span_kernel<MT, 2, Y>), grid, dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((lora_up_span_kernel<1, 4, Y>), grid, dim3(256), 0, s, p);
}

template <typename Y>
void launch_up(const LoraArgs& p, dim3 grid, hipStream_t s) {
    if (p.rmax <= 32)
        hipLaunchKernelGGL((lora_up_kernel<1, Y>), grid, dim3(256), 0, s, p);
    else if (p.rmax <= 64)
        hipLaunchKernelGGL((lora_up_kernel<2, Y>), grid, dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((lora_up_kernel<4, Y>), grid, dim3(256), 0, s, p);
}

}  // namespace
}  // namespace af

using namespace af;

extern "C" size_t af_lora_workspace_size(const af_lora* lora, int m) {
    if (lora_check(lora) || m < 0) return 0;
    return align_up(size_t(lora_split(lora->k).parts) * size_t(m > 0 ? m : 1) * lora->n_slices *
                        lora->max_rank * sizeof(float),
                    256);
}

extern "C" int af_lora_add(const void* x, int64_t x_stride, int m, const int32_t* d_ids,
                           const af_lora* lora, const void* y, int64_t y_stride, void* y_out,
                           int64_t y_out_stride, int y_dtype, void* workspace,
                           size_t workspace_bytes, af_stream_t stream) {
    if (int st = lora_check(lora)) return st;
    if (y_dtype != AF_FP16 && y_dtype != AF_FP32) return AF_ERR_UNSUPPORTED;
    const size_t esz = y_dtype == AF_FP16 ? 2 : 4;
    if (!lora->a || !lora->b || m < 0 || x_stride < lora->k || x_stride % 8 ||
        y_stride < lora->n || y_out_stride < lora->n)
        return AF_ERR_INVALID_ARG;
    if (!aligned16(lora->a) || !aligned16(lora->b) || !aligned_to(lora->ranks, 4) ||
        !aligned_to(lora->scales, 4))
        return AF_ERR_INVALID_ARG;
    if (m == 0) return AF_OK;
    if (!x || !d_ids || !y || !y_out || !aligned16(x) || !aligned_to(d_ids, 4) ||
        !aligned_to(y, esz) || !aligned_to(y_out, esz))
        return AF_ERR_INVALID_ARG;
    if (y == y_out && y_stride != y_out_stride) return AF_ERR_INVALID_ARG;
    if (m > (1 << 20)) return AF_ERR_UNSUPPORTED;
    if (!workspace || !aligned16(workspace) || workspace_bytes < af_lora_workspace_size(lora, m))
        return AF_ERR_WORKSPACE;

    LoraArgs p{};
    p.x = static_cast<const uint16_t*>(x);
    p.x_stride = x_stride;
    p.m = m;
    p.ids = d_ids;
    p.a = static_cast<const uint16_t*>(lora->a);
    p.b = static_cast<const uint16_t*>(lora->b);
    p.ranks = lora->ranks;
    p.scales = lora->scales;
    p.n_adapters = lora->n_adapters;
    p.rmax = lora->max_rank;
    p.rows = lora->n_slices * lora->max_rank;
    p.k = lora->k;
    p.n = lora->n;
    p.y = y;
    p.y_stride = y_stride;
    p.y_out = y_out;
    p.y_out_stride = y_out_stride;
    p.v = static_cast<float*>(workspace);
    const LoraSplit split = lora_split(p.k);
    p.parts = split.parts;
    p.part_k = split.part_k;
    p.n_slices = lora->n_slices;

    // the most adapters that n tokens in a row can name
    auto named = [&](int n) { return std::min(std::min(m, n), p.n_adapters); };
    hipStream_t s = static_cast<hipStream_t>(stream);
    // Batches of up to 256 tokens are mostly decoded ones, few to an adapter; above, prompt chunks.
    const bool chunks = m > 256;
    const int row_tiles = ceil_div(p.rows, 16);
    const int row_groups = ceil_div(row_tiles, 4), nt = ceil_div(row_tiles, row_groups);
    p.tiles = ceil_div(m, kTile);

    // `up` streams spans of columns where there is one for every compute unit or so (8192 tokens by
    // 28672 columns: 222 us, by single blocks 278; 2000 tokens: 53 and 61; 3000 tokens by 4096
    // columns: 18 and 14).
    const bool span = chunks && int64_t(p.tiles) * p.n >= int64_t(256) * kSpan;
    const int cols = span ? kSpan : kCols;
    int blocks = 0;
    for (int i = 0; i < p.n_slices; ++i) {
        p.slice_begin[i + 1] = lora->slice_end[i];
        p.slice_block[i] = blocks;
        blocks += ceil_div(lora->slice_end[i] - p.slice_begin[i], cols);
    }
    p.slice_block[p.n_slices] = blocks;
    if (int64_t(blocks) * p.tiles > (1 << 22)) return AF_ERR_UNSUPPORTED;
    p.items = blocks * p.tiles;
    auto blocks_of = [](int items, int side) { return dim3(unsigned(align_up(size_t(items), 8)) * side); };

    // The tiles' rows come through LDS where workgroups of 64 tokens and a part of K, or all of it,
    // are enough for the device (2011 tokens, 14336 -> rank 16: 20 us, by registers 25; 3000
    // tokens, 4096 -> rank 16: 9 and 11; 8192 tokens, 4096 -> twice rank 64: 46, by registers 84,
    // with the parts left to `up` 61 and `up` 242 instead of 222). More workgroups to an item cost
    // time where they find nothing to do, and save it where a tile names many adapters: 45 tokens
    // of 24 adapters: `up` with 25 of them 17 us, with 9 12.5, with 4 15.5.
    if (chunks && p.tiles * row_groups * p.parts >= 96) {
        p.splits = p.tiles * row_groups >= 192 ? 1 : p.parts;
        p.down_tiles = p.tiles;
        p.down_items = p.tiles * row_groups * p.splits;
        p.down_side = std::min(named(kTile), std::max(6, 1024 / p.down_items));
        launch_down_lds(p, blocks_of(p.down_items, p.down_side), nt, s);
    } else {
        p.splits = p.parts;
        // Tiles of 16 tokens read an adapter's rows more often, but side by side: 62 tokens of one
        // adapter, 11720 -> 2 x rank 16: 4.1 us, with 64 tokens to a tile 9.7; 246 of three, 4872
        // -> 2 x rank 64: 13 and 8.2.
        const bool few = int64_t(ceil_div(m, 16)) * row_tiles * p.parts * named(16) <= 256;
        p.down_tile = chunks || few ? 16 : kTile;
        p.down_tiles = ceil_div(m, p.down_tile);
        p.down_items = p.down_tiles * row_tiles * p.parts;
        p.down_side = std::min(named(p.down_tile), std::max(chunks ? 2 : 1, 1024 / p.down_items));
        hipLaunchKernelGGL(lora_down_kernel, blocks_of(p.down_items, p.down_side), dim3(256), 0, s, p);
    }
    AF_TRY_LAUNCH();

    if (span) {
        p.side = std::min(named(kTile) + (y != y_out), std::max(2, 2048 / p.items));
        if (y_dtype == AF_FP16)
            launch_up_span<4, uint16_t>(p, blocks_of(p.items, p.side), s);
        else
            launch_up_span<2, float>(p, blocks_of(p.items, p.side), s);
        AF_TRY_LAUNCH();
        return AF_OK;
    }
    p.side = std::min(named(kTile) + (y != y_out), std::max(1, (chunks ? 2048 : 1024) / p.items));
    const dim3 up = blocks_of(p.items, p.side);
    if (y_dtype == AF_FP16)
        launch_up<uint16_t>(p, up, s);
    else
        launch_up<float>(p, up, s);
    AF_TRY_LAUNCH();
    return AF_OK;
}
