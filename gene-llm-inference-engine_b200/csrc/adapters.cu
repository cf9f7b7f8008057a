// Low-rank adapters of many requests beside a shared projection:
//   out[t, n] += scale_a * sum_j up_a[n, j] * (sum_k x[t, k] down_a[s(n) * r + j, k]),  a = the adapter of row t (none: nothing),
// s(n) the slice of column n (q | k | v, or gate | up, stacked in one output, each with a pair of matrices of its own).
//
// The rows of a step are cut into tiles of one adapter each (found by the tiles' blocks themselves in steps of up to 1,024 rows, else once a step by
// adapter_plan). A cluster of CTAs takes a tile: every CTA multiplies its share of K, the partial sums [rows, S r] are added through
// distributed shared memory, and every CTA writes its share of the columns. x, out and the weights cross memory once; the r values in between never do.
//
// What bounds it: single tokens the chain read, sum, exchange, read, add (eight tokens at 2,048 x 2,048, rank 16: 5.3 us); prompts the bytes of x
// and out, each in a phase of its own that starts with an exchange (2,048 rows of 4,096 into 6,144, rank 16: 33 us for 18 us of bytes: 10 us until x is through, 3 for the
// exchanges, 20 for out); high ranks also the tensor cores and what feeds them (8,192 rows of 14,336 into 4,096, rank 64: 124 us, 70, 4 and 50 of them so).
#include <climits>
#include <type_traits>

#include <cooperative_groups.h>

#include "common.cuh"
#include "device_limit.h"

namespace gi {

namespace cg = cooperative_groups;

constexpr int kPlanThreads = 1024, kPlanEach = 8;
constexpr int kPlanAdaptersMost = 8192;        // counters of the plan's block in shared memory
constexpr int kAdapterRanksMost = 512;         // S * r
constexpr int kAdapterSlicesMost = 4;
constexpr int kAdapterClusterMost = 8;

// A plan: [0] tiles, then the rows in the adapters' order [T], then (adapter, first place, rows) of every tile.
struct PlanView {
    const int* p;
    int T;
    __device__ __forceinline__ int tiles() const { return p[0]; }
    __device__ __forceinline__ const int* rows() const { return p + 1; }
    __device__ __forceinline__ const int* tile(int i) const { return p + 1 + T + 3 * static_cast<size_t>(i); }
};

// One block: rows counted by adapter, the adapters' first places and tiles by a scan, then every row to its place (a warp's rows of one
// adapter take theirs together, in order).
__global__ void __launch_bounds__(kPlanThreads) adapter_plan_kernel(const int* row_adapter, int T, int A, int tile_rows, int* plan) {
    pdl_prologue();
    extern __shared__ int counts[];            // [A]: rows, then the next free place
    __shared__ int warp_rows[32], warp_tiles[32], base_rows, base_tiles;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int a = threadIdx.x; a < A; a += kPlanThreads) counts[a] = 0;
    if (threadIdx.x == 0) base_rows = base_tiles = 0;
    __syncthreads();
    // up to kPlanEach rows a thread stay in registers, all asked for at once; further ones are read again
    auto adapter = [&](int t) {
        const int a = t < T ? row_adapter[t] : -1;
        return a >= 0 && a < A ? a : -1;
    };
    int held[kPlanEach];
    unsigned held_same[kPlanEach];             // the lanes with the same adapter
#pragma unroll
    for (int i = 0; i < kPlanEach; ++i) held[i] = adapter(i * kPlanThreads + threadIdx.x);
    auto alike = [&](int a) {                  // (neighbouring rows mostly have one adapter)
        return __all_sync(0xffffffffu, a == __shfl_sync(0xffffffffu, a, 0)) ? 0xffffffffu : __match_any_sync(0xffffffffu, a);
    };
    auto count = [&](int a, unsigned same) {
        if (a >= 0 && lane == __ffs(same) - 1) atomicAdd(&counts[a], __popc(same));
    };
#pragma unroll
    for (int i = 0; i < kPlanEach; ++i)
        if (i * kPlanThreads < T) { held_same[i] = alike(held[i]); count(held[i], held_same[i]); }
    for (int t0 = kPlanEach * kPlanThreads; t0 < T; t0 += kPlanThreads) {
        const int a = adapter(t0 + threadIdx.x);
        count(a, alike(a));
    }
    __syncthreads();
    int* tiles = plan + 1 + T;
    for (int a0 = 0; a0 < A; a0 += kPlanThreads) {
        const int a = a0 + threadIdx.x;
        const int rows = a < A ? counts[a] : 0, mine = (rows + tile_rows - 1) / tile_rows;
        int r = rows, q = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, r, o), y = __shfl_up_sync(0xffffffffu, q, o);
            if (lane >= o) { r += x; q += y; }
        }
        if (lane == 31) { warp_rows[warp] = r; warp_tiles[warp] = q; }
        __syncthreads();
        int first = base_rows + r - rows, tile = base_tiles + q - mine;
        for (int w = 0; w < warp; ++w) { first += warp_rows[w]; tile += warp_tiles[w]; }
        if (a < A) counts[a] = first;
        for (int i = 0; i < mine; ++i) {
            tiles[3 * (tile + i)] = a;
            tiles[3 * (tile + i) + 1] = first + i * tile_rows;
            tiles[3 * (tile + i) + 2] = min(tile_rows, rows - i * tile_rows);
        }
        __syncthreads();
        if (threadIdx.x == kPlanThreads - 1) { base_rows = first + rows; base_tiles = tile + mine; }
        __syncthreads();
    }
    if (threadIdx.x == 0) plan[0] = base_tiles;
    auto put = [&](int t, int a, unsigned same) {
        const int leader = __ffs(same) - 1;
        int place = 0;
        if (a >= 0 && lane == leader) place = atomicAdd(&counts[a], __popc(same));
        place = __shfl_sync(0xffffffffu, place, leader) + __popc(same & ((1u << lane) - 1));
        if (a >= 0) plan[1 + place] = t;
    };
#pragma unroll
    for (int i = 0; i < kPlanEach; ++i)
        if (i * kPlanThreads < T) put(i * kPlanThreads + threadIdx.x, held[i], held_same[i]);
    for (int t0 = kPlanEach * kPlanThreads; t0 < T; t0 += kPlanThreads) {
        const int a = adapter(t0 + threadIdx.x);
        put(t0 + threadIdx.x, a, alike(a));
    }
}

struct AdapterArgs {
    const void* x;
    long long ldx;
    const void* down;
    const void* up;
    const float* scales;
    PlanView plan;
    void* out;
    long long ldo;
    int A, used, K, N, r, S, tile_rows;        // used: adapters that occur at most; tile_rows 0: no plan, plan.p are the rows' adapters
    int ends[kAdapterSlicesMost];              // a slice's last column + 1
    int wide;                                  // eight neighbouring columns from a multiple of eight on lie on 16 bytes in every row of out
};

constexpr int kAdapterThreads = 256, kAdapterWarps = kAdapterThreads / 32;
constexpr int kDirectRows = 1024, kDirectEach = kDirectRows / kAdapterThreads;      // steps of up to so many rows have no plan: a tile's blocks look its rows up themselves
constexpr int kDirectAdapters = 1024;          // (of so many adapters)
constexpr int kFewTokens = 256;                // rows up to which they are taken for single tokens, each with an adapter of its own as a rule

// The rows of tile `which` of `M` rows (with a plan: of the `M` rows from `piece` on of a plan's tile) into rows[0 .. M); false: there are none.
template <int M>
__device__ __forceinline__ bool find_rows(const PlanView& plan, int A, int tile_rows, int which, int* rows, int& adapter, int& n, int* scratch) {
    if (tile_rows == 0 && plan.T <= 32) {
        // every warp for itself: a row begins a tile if the rows of its adapter ahead of it fill whole tiles (eight single tokens: 0.5 us instead of 1.4)
        const int lane = threadIdx.x & 31;
        const int mine = lane < plan.T ? plan.p[lane] : -1;
        const bool valid = mine >= 0 && mine < A;
        const unsigned same = __match_any_sync(0xffffffffu, valid ? mine : -1 - lane), ahead = (1u << lane) - 1;
        const int rank = __popc(same & ahead);
        const bool leads = valid && rank % M == 0;
        const unsigned leaders = __ballot_sync(0xffffffffu, leads), its = __ballot_sync(0xffffffffu, leads && __popc(leaders & ahead) == which);
        if (its == 0) return false;
        const int leader = __ffs(its) - 1, place = rank - __shfl_sync(0xffffffffu, rank, leader);
        adapter = __shfl_sync(0xffffffffu, mine, leader);
        const bool in = mine == adapter && place >= 0 && place < M;
        n = __popc(__ballot_sync(0xffffffffu, in));
        if (threadIdx.x < 32) {
            for (int i = lane; i < M; i += 32) rows[i] = -1;
            __syncwarp();
            if (in) rows[place] = lane;
        }
    } else if (tile_rows == 0) {
        // rows counted by adapter, the adapters' first tiles by a scan, then the ranks of the rows of the one that has tile `which`
        __shared__ int s_counts[kDirectAdapters], s_adapter, s_tile;
        constexpr int kEach = kDirectAdapters / kAdapterThreads;
        const int i = threadIdx.x, lane = i & 31, warp = i >> 5;
        int mine[kDirectEach];
#pragma unroll
        for (int e = 0; e < kDirectEach; ++e) mine[e] = i + e * kAdapterThreads < plan.T ? plan.p[i + e * kAdapterThreads] : -1;
#pragma unroll
        for (int k = 0; k < kEach; ++k) s_counts[i + k * kAdapterThreads] = 0;
        for (int k = i; k < M; k += kAdapterThreads) rows[k] = -1;
        if (i == 0) s_adapter = -1;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kDirectEach; ++e) {
            if (e * kAdapterThreads >= plan.T) break;
            const bool valid = mine[e] >= 0 && mine[e] < A;
            if (__all_sync(0xffffffffu, mine[e] == __shfl_sync(0xffffffffu, mine[e], 0))) {      // (a prompt's rows)
                if (valid && lane == 0) atomicAdd(&s_counts[mine[e]], 32);
            } else if (valid) {
                atomicAdd(&s_counts[mine[e]], 1);
            }
        }
        __syncthreads();
        int tiles[kEach], sum = 0;
#pragma unroll
        for (int k = 0; k < kEach; ++k) { tiles[k] = (s_counts[i * kEach + k] + M - 1) / M; sum += tiles[k]; }
        int run = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += v;
        }
        if (lane == 31) scratch[warp] = run;
        __syncthreads();
        run -= sum;
        for (int w = 0; w < warp; ++w) run += scratch[w];
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            if (which >= run && which < run + tiles[k]) { s_adapter = i * kEach + k; s_tile = which - run; }
            run += tiles[k];
        }
        __syncthreads();
        adapter = s_adapter;
        if (adapter < 0) return false;
        const int first = s_tile * M;
        n = min(M, s_counts[adapter] - first);
        __syncthreads();                       // the scratch is free again
#pragma unroll
        for (int e = 0; e < kDirectEach; ++e) {
            const unsigned same = __ballot_sync(0xffffffffu, mine[e] == adapter);
            if (lane == 0) scratch[e * kAdapterWarps + warp] = __popc(same);
        }
        __syncthreads();
        int before = 0;                        // the adapter's rows ahead, in the order (turn, warp, lane)
#pragma unroll
        for (int e = 0; e < kDirectEach; ++e) {
            if (e * kAdapterThreads >= plan.T) break;
            for (int w = 0; w < kAdapterWarps; ++w) {
                if (w == warp) {
                    const unsigned same = __ballot_sync(0xffffffffu, mine[e] == adapter);
                    const int place = before + __popc(same & ((1u << lane) - 1)) - first;
                    if (mine[e] == adapter && place >= 0 && place < M) rows[place] = i + e * kAdapterThreads;
                }
                before += scratch[e * kAdapterWarps + w];
            }
        }
    } else {
        const int per_tile = (tile_rows + M - 1) / M, tile = which / per_tile, piece = which % per_tile;
        if (tile >= plan.tiles()) return false;
        const int* info = plan.tile(tile);
        adapter = info[0];
        n = min(M, info[2] - piece * M);
        if (n <= 0) return false;              // (the plan's tile ends ahead of this piece of it)
        for (int i = threadIdx.x; i < M; i += kAdapterThreads) rows[i] = i < n ? plan.rows()[info[1] + piece * M + i] : -1;
    }
    __syncthreads();
    return true;
}

// ---- any type, any size: on the CUDA cores, in 32 bits ----
constexpr int kPlainThreads = kAdapterThreads, kPlainRows = 32, kPlainCols = 64, kPlainK = 32;

template <typename T, typename TO>
__global__ void __launch_bounds__(kPlainThreads) adapter_plain_kernel(AdapterArgs a) {
    pdl_prologue();
    extern __shared__ float h[];               // [2][kPlainRows][S r]: this CTA's partial sums, then the whole sums
    __shared__ float xs[kPlainRows][kPlainK + 1], ds[kPlainCols][kPlainK + 1];
    __shared__ int s_rows[kPlainRows], s_scratch[kDirectEach * kAdapterWarps];
    cg::cluster_group cluster = cg::this_cluster();
    const int part = cluster.block_rank(), parts = cluster.num_blocks();
    int adapter, rows;
    if (!find_rows<kPlainRows>(a.plan, a.A, a.tile_rows, blockIdx.x / parts, s_rows, adapter, rows, s_scratch)) return;     // (the whole cluster)
    const int cols = a.S * a.r;
    const T* down = static_cast<const T*>(a.down) + static_cast<size_t>(adapter) * cols * a.K;
    const T* x = static_cast<const T*>(a.x);
    const int k_share = ((a.K + parts - 1) / parts + kPlainK - 1) / kPlainK * kPlainK;
    const int k_begin = min(a.K, part * k_share), k_end = min(a.K, k_begin + k_share);
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    for (int c0 = 0; c0 < cols; c0 += kPlainCols) {
        float acc[2][4] = {};
        for (int k0 = k_begin; k0 < k_end; k0 += kPlainK) {
            __syncthreads();
            for (int i = threadIdx.x; i < kPlainRows * kPlainK; i += kPlainThreads) {
                const int row = s_rows[i / kPlainK], k = k0 + i % kPlainK;
                xs[i / kPlainK][i % kPlainK] = row >= 0 && k < k_end ? to_float(x[row * a.ldx + k]) : 0.f;
            }
            for (int i = threadIdx.x; i < kPlainCols * kPlainK; i += kPlainThreads) {
                const int c = c0 + i / kPlainK, k = k0 + i % kPlainK;
                ds[i / kPlainK][i % kPlainK] = c < cols && k < k_end ? to_float(down[static_cast<size_t>(c) * a.K + k]) : 0.f;
            }
            __syncthreads();
#pragma unroll 8
            for (int k = 0; k < kPlainK; ++k) {
                const float x0 = xs[2 * ty][k], x1 = xs[2 * ty + 1][k];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float w = ds[tx + 16 * i][k];
                    acc[0][i] = fmaf(x0, w, acc[0][i]);
                    acc[1][i] = fmaf(x1, w, acc[1][i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c0 + tx + 16 * i < cols) {
                h[(2 * ty) * cols + c0 + tx + 16 * i] = acc[0][i];
                h[(2 * ty + 1) * cols + c0 + tx + 16 * i] = acc[1][i];
            }
    }
    cluster.sync();
    const float scale = a.scales[adapter];
    float* sum = h + kPlainRows * cols;
    for (int i = threadIdx.x; i < kPlainRows * cols; i += kPlainThreads) {
        float v = 0.f;
        for (int p = 0; p < parts; ++p) v += *cluster.map_shared_rank(h + i, p);
        sum[i] = v * scale;
    }
    cluster.sync();                            // no CTA leaves while another reads its sums
    const T* up = static_cast<const T*>(a.up) + static_cast<size_t>(adapter) * a.N * a.r;
    TO* out = static_cast<TO*>(a.out);
    const int n_share = (a.N + parts - 1) / parts, n_begin = min(a.N, part * n_share), n_end = min(a.N, n_begin + n_share);
    for (int n = n_begin + threadIdx.x; n < n_end; n += kPlainThreads) {
        int slice = 0;
        while (n >= a.ends[slice]) ++slice;
        float acc[kPlainRows] = {};
        for (int j = 0; j < a.r; ++j) {
            const float w = to_float(up[static_cast<size_t>(n) * a.r + j]);
            const float* at = sum + slice * a.r + j;
#pragma unroll
            for (int i = 0; i < kPlainRows; ++i) acc[i] = fmaf(at[i * cols], w, acc[i]);
        }
#pragma unroll
        for (int i = 0; i < kPlainRows; ++i)
            if (i < rows) {
                TO* o = out + s_rows[i] * a.ldo + n;
                *o = from_float<TO>(to_float(*o) + acc[i]);
            }
    }
}

// ---- bfloat16 on the tensor cores (mma.sync m16n8k16) ----
// Rows are the M side in both products, the ranks (then the output's columns) the N side. Lane (g, c) = (lane / 4, lane % 4) holds of A rows g and
// g + 8, of B column g, and of both the k slots 2c, 2c + 1, 2c + 8, 2c + 9. Which values of k sit in these slots is free as long as A and B agree: reading
// straight from memory a lane takes neighbours of a row (8 c .. 8 c + 7 for two steps of k, or 4 c .. 4 c + 3 for one), 64 or 32 bytes a row for its four lanes.
// Between the products a row's r sums are kept as three bfloat16 pieces, each what the ones before leave, which hold all 24 bits (two showed as 1.8e-6 of a 32-bit
// result against 2e-7, and as the whole of a bfloat16 one whose terms cancel; 8,192 rows of 14,336 into 4,096 at rank 64 with two 121 us, with three 128 us).
constexpr int kFewRows = 16, kBlockCols = 32, kPieces = 3;

__device__ __forceinline__ void mma_bf16(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void load_matrices(unsigned (&m)[4], unsigned address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(m[0]), "=r"(m[1]), "=r"(m[2]), "=r"(m[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ unsigned shared_address(const void* p) { return static_cast<unsigned>(__cvta_generic_to_shared(p)); }

// The k slot of a rank within its 16: ranks 4 c .. 4 c + 3 sit in slots 2c, 2c + 1, 2c + 8, 2c + 9.
__device__ __forceinline__ int rank_slot(int j) { return (j & ~15) + 2 * ((j >> 2) & 3) + ((j & 2) << 2) + (j & 1); }

// The next piece of a value (its bits), which is taken off it. All pieces but the last stay below what is left, so that none of them is zero and all have the value's
// sign, unless it is zero: with an infinite weight the products then are the infinity that the value's is, and no zero times infinity comes up that the value has not.
// What is infinite or no number itself is its own piece every time, and none is rounded up to an infinity. (The last piece of a value below 2^-117 may vanish.)
__device__ __forceinline__ unsigned next_piece(float& v, bool last) {
    const unsigned u = __float_as_uint(v), size = u & 0x7fffffffu;
    if (size >= 0x7f800000u) return u >> 16 | (size > 0x7f800000u ? 0x40u : 0u);
    if (last) return __bfloat16_as_ushort(__float2bfloat16_rn(v));
    const unsigned p = size ? (u - 1) & 0xffff0000u : 0u;
    v -= __uint_as_float(p);
    return p >> 16;
}
// .. of two neighbouring values (an even rank first).
__device__ __forceinline__ unsigned next_piece(float& v0, float& v1, bool last) {
    const unsigned p0 = next_piece(v0, last);
    return p0 | next_piece(v1, last) << 16;
}

// kSteps steps of k (16 ranks each) of 32 columns of `up`. Which column is column g of tile q is chosen so that a lane's values of a row are runs
// of 16 bytes and the runs of its four lanes fill whole sectors: 32-bit outputs 16 (q / 2) + 4 (g / 2) + 2 (q % 2) + g % 2, two runs of
// four; bfloat16 ones 8 (g / 2) + 2 q + g % 2, one run of eight.
template <int kSteps> struct UpFragments {
    unsigned b[4][kSteps][2];                  // [tile of columns][step][half]
};
template <int kSteps, typename TO>
__device__ __forceinline__ void load_up(UpFragments<kSteps>& f, const __nv_bfloat16* up, int r, int rank0, int cols) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int col = sizeof(TO) == 4 ? 16 * (q >> 1) + 4 * (g >> 1) + 2 * (q & 1) + (g & 1) : 8 * (g >> 1) + 2 * q + (g & 1);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int j = rank0 + 16 * s + 4 * c;
            uint2 v = {0u, 0u};
            if (col < cols && j < r) v = __ldg(reinterpret_cast<const uint2*>(up + static_cast<size_t>(col) * r + j));
            f.b[q][s][0] = v.x;
            f.b[q][s][1] = v.y;
        }
    }
}

// A block of up to 32 columns within one slice.
struct ColumnBlock {
    int col, cols, slice;
};
__device__ __forceinline__ ColumnBlock column_block(const AdapterArgs& a, int i) {
    int begin = 0;
#pragma unroll
    for (int s = 0; s < kAdapterSlicesMost - 1; ++s) {
        const int n = (a.ends[s] - begin + kBlockCols - 1) / kBlockCols;
        if (i < n || s == a.S - 1) return {begin + i * kBlockCols, min(kBlockCols, a.ends[s] - begin - i * kBlockCols), s};
        i -= n;
        begin = a.ends[s];
    }
    return {begin + i * kBlockCols, min(kBlockCols, a.ends[kAdapterSlicesMost - 1] - begin - i * kBlockCols), kAdapterSlicesMost - 1};
}

// What a bfloat16 output holds in a lane's runs of a block, asked for ahead of the products (32-bit outputs are added to at the memory's side).
template <int MT, typename TO> struct OldValues {
    uint4 v[sizeof(TO) == 2 ? MT : 1][2];
};
__device__ __forceinline__ bool is_wide(const AdapterArgs& a, const ColumnBlock& block) { return a.wide && block.col % 8 == 0 && block.cols == kBlockCols; }
template <int MT, typename TO>
__device__ __forceinline__ void load_old(OldValues<MT, TO>& old, const AdapterArgs& a, const ColumnBlock& block, int row0, const int* rows) {
    if constexpr (sizeof(TO) == 2) {
        if (!is_wide(a, block)) return;
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        const TO* out = static_cast<const TO*>(a.out) + block.col + 8 * c;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int row = rows[row0 + 16 * m + 8 * half + g];
                if (row >= 0) old.v[m][half] = *reinterpret_cast<const uint4*>(out + row * a.ldo);
            }
    }
}

// The second product of a warp: a block's columns for `MT` tiles of 16 rows from row0 on. pieces: shared [piece][`piece_bytes`: rows x ld] bfloat16
// in the ranks' slots. fresh: f does not hold the block's first ranks yet.
template <int MT, int kSteps, typename TO>
__device__ __forceinline__ void expand(const AdapterArgs& a, UpFragments<kSteps>& f, bool fresh, const OldValues<MT, TO>& old, const __nv_bfloat16* up,
                                       const ColumnBlock& block, unsigned pieces, unsigned piece_bytes, int ld, int row0, const int* rows) {
    constexpr int kRun = 16 / sizeof(TO), kRuns = 8 / kRun;
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const bool wide = is_wide(a, block);
    TO* out = static_cast<TO*>(a.out) + block.col + kRun * c;
    float acc[MT][4][4] = {};
    for (int rank0 = 0; rank0 < (kSteps == 4 ? a.r : 1); rank0 += 64) {
        if (fresh || rank0) load_up<kSteps, TO>(f, up, a.r, rank0, block.cols);
        const int k0 = block.slice * ((a.r + 15) & ~15) + rank0;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            if (kSteps < 4 || rank0 + 16 * s < a.r) {
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const unsigned at = ((row0 + 16 * m + (lane & 15)) * ld + k0 + 16 * s + 8 * (lane >> 4)) * 2;
#pragma unroll
                    for (int p = 0; p < kPieces; ++p) {
                        unsigned h[4];
                        load_matrices(h, pieces + p * piece_bytes + at);
#pragma unroll
                        for (int q = 0; q < 4; ++q) mma_bf16(acc[m][q], h[0], h[1], h[2], h[3], f.b[q][s][0], f.b[q][s][1]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int row = rows[row0 + 16 * m + 8 * half + g];
            if (row < 0) continue;
            float v[8];
#pragma unroll
            for (int q = 0; q < 4; ++q) { v[2 * q] = acc[m][q][2 * half]; v[2 * q + 1] = acc[m][q][2 * half + 1]; }
            TO* at = out + row * a.ldo;
#pragma unroll
            for (int u = 0; u < kRuns; ++u) {
                if (wide && sizeof(TO) == 4) {
                    // every value is added to once a call, so an addition at the memory's side, with nothing to wait for, gives the same bits in
                    // any order (2,048 rows x 6,144 columns: 16 us for the second product, 22 us with loads and stores)
                    const float* y = v + 4 * u;
                    asm volatile("red.global.add.v4.f32 [%0], {%1,%2,%3,%4};" :: "l"(at + 16 * u), "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]) : "memory");
                } else if (wide) {
                    uint4 x = old.v[sizeof(TO) == 2 ? m : 0][half];
                    unsigned* w = reinterpret_cast<unsigned*>(&x);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const __nv_bfloat162 s = __floats2bfloat162_rn(__uint_as_float(w[i] << 16) + v[2 * i], __uint_as_float(w[i] & 0xffff0000u) + v[2 * i + 1]);
                        w[i] = *reinterpret_cast<const unsigned*>(&s);
                    }
                    *reinterpret_cast<uint4*>(at + 16 * u) = x;
                } else {
#pragma unroll
                    for (int i = 0; i < kRun; ++i)
                        if (kRun * c + 16 * u + i < block.cols) at[16 * u + i] = from_float<TO>(to_float(at[16 * u + i]) + v[kRun * u + i]);
                }
            }
        }
}

__device__ __forceinline__ int column_blocks(const AdapterArgs& a) {
    int n = 0, begin = 0;
#pragma unroll
    for (int s = 0; s < kAdapterSlicesMost; ++s)
        if (s < a.S) { n += (a.ends[s] - begin + kBlockCols - 1) / kBlockCols; begin = a.ends[s]; }
    return n;
}

// Four sums of a row of the tile over the cluster's CTAs (whose partial sums lie at the same place), times scale.
__device__ __forceinline__ float4 cluster_total(const float* at, float scale, cg::cluster_group& cluster, int parts) {
    float4 x[kAdapterClusterMost];
#pragma unroll
    for (int p = 0; p < kAdapterClusterMost; ++p)
        if (p < parts) x[p] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(at, p));
    float4 v = x[0];
#pragma unroll
    for (int p = 1; p < kAdapterClusterMost; ++p)
        if (p < parts) { v.x += x[p].x; v.y += x[p].y; v.z += x[p].z; v.w += x[p].w; }
    return make_float4(v.x * scale, v.y * scale, v.z * scale, v.w * scale);
}

// Few rows (single tokens): everything comes straight from memory into the lanes that multiply it. A warp takes every eighth 32 values of the CTA's
// share of K; the warps' sums meet in shared memory, the CTAs' through the cluster.
constexpr int kFewCols = 64;
template <int kSteps, typename TO>
__global__ void __launch_bounds__(kAdapterThreads, 2) adapter_few_kernel(AdapterArgs a) {
    pdl_prologue();
    extern __shared__ __align__(16) float h[]; // [kFewRows][S r], then the pieces
    __shared__ float2 sums[kAdapterWarps][kFewRows][kFewCols / 2 + 4];
    __shared__ int s_rows[kFewRows], s_scratch[kDirectEach * kAdapterWarps];
    cg::cluster_group cluster = cg::this_cluster();
    const int part = cluster.block_rank(), parts = cluster.num_blocks();
    int adapter, n;
    if (!find_rows<kFewRows>(a.plan, a.A, a.tile_rows, blockIdx.x / parts, s_rows, adapter, n, s_scratch)) return;     // (the whole cluster)
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    const int cols = a.S * a.r, rp = (a.r + 15) & ~15, ld = a.S * rp + 8;
    const __nv_bfloat16* down = static_cast<const __nv_bfloat16*>(a.down) + static_cast<size_t>(adapter) * cols * a.K;
    const __nv_bfloat16* up = static_cast<const __nv_bfloat16*>(a.up) + static_cast<size_t>(adapter) * a.N * a.r;
    __nv_bfloat16* pieces = reinterpret_cast<__nv_bfloat16*>(h + kFewRows * cols);
    const float scale = a.scales[adapter];
    if (rp != a.r)                             // the slots of ranks that are not there
        for (int i = threadIdx.x; i < kFewRows * ld / 2 * kPieces; i += kAdapterThreads) reinterpret_cast<unsigned*>(pieces)[i] = 0u;
    const int share = ((a.K + parts - 1) / parts + 31) / 32 * 32, k_begin = min(a.K, part * share), k_end = min(a.K, k_begin + share);
    const int row_g = s_rows[g], row_h = s_rows[g + 8];
    const __nv_bfloat16* x_g = static_cast<const __nv_bfloat16*>(a.x) + max(row_g, 0) * a.ldx;
    const __nv_bfloat16* x_h = static_cast<const __nv_bfloat16*>(a.x) + max(row_h, 0) * a.ldx;
    // the warp's first columns of the second product, asked for ahead of all (they wait for nobody)
    const int blocks = column_blocks(a), per = (blocks + parts - 1) / parts, first = part * per + warp, last = min(blocks, (part + 1) * per);
    UpFragments<kSteps> f;
    ColumnBlock block = {0, 0, 0};
    if (first < last) {
        block = column_block(a, first);
        load_up<kSteps, TO>(f, up + static_cast<size_t>(block.col) * a.r, a.r, 0, block.cols);
    }
    for (int c0 = 0; c0 < cols; c0 += kFewCols) {
        float acc[kFewCols / 8][4] = {};
        for (int k0 = k_begin + 32 * warp; k0 < k_end; k0 += 32 * kAdapterWarps) {
            const int k = k0 + 8 * c;
            const bool there = k < k_end;
            uint4 x0 = {0u, 0u, 0u, 0u}, x1 = x0, w[kFewCols / 8];
            if (there && row_g >= 0) x0 = __ldg(reinterpret_cast<const uint4*>(x_g + k));
            if (there && row_h >= 0) x1 = __ldg(reinterpret_cast<const uint4*>(x_h + k));
#pragma unroll
            for (int t = 0; t < kFewCols / 8; ++t) {
                const int j = c0 + 8 * t + g;
                w[t] = make_uint4(0u, 0u, 0u, 0u);
                if (there && j < cols) w[t] = __ldg(reinterpret_cast<const uint4*>(down + static_cast<size_t>(j) * a.K + k));
            }
#pragma unroll
            for (int t = 0; t < kFewCols / 8; ++t) {
                if (c0 + 8 * t < cols) {
                    mma_bf16(acc[t], x0.x, x1.x, x0.y, x1.y, w[t].x, w[t].y);
                    mma_bf16(acc[t], x0.z, x1.z, x0.w, x1.w, w[t].z, w[t].w);
                }
            }
        }
        if (c0) __syncthreads();
#pragma unroll
        for (int t = 0; t < kFewCols / 8; ++t)
            if (c0 + 8 * t < cols) {
                sums[warp][g][4 * t + c] = make_float2(acc[t][0], acc[t][1]);
                sums[warp][g + 8][4 * t + c] = make_float2(acc[t][2], acc[t][3]);
            }
        __syncthreads();
        const int some = min(kFewCols, cols - c0);
        for (int i = threadIdx.x; i < kFewRows * kFewCols / 2; i += kAdapterThreads) {
            const int row = i / (kFewCols / 2), pair = i % (kFewCols / 2);
            if (2 * pair >= some) continue;
            float2 v = sums[0][row][pair];
#pragma unroll
            for (int w = 1; w < kAdapterWarps; ++w) { const float2 y = sums[w][row][pair]; v.x += y.x; v.y += y.y; }
            *reinterpret_cast<float2*>(h + row * cols + c0 + 2 * pair) = v;
        }
    }
    cluster.sync();
    for (int i = threadIdx.x; i < kFewRows * cols / 4; i += kAdapterThreads) {
        const int row = 4 * i / cols, col = 4 * i % cols;
        float4 v = cluster_total(h + row * cols + col, scale, cluster, parts);
        __nv_bfloat16* to = pieces + row * ld + (col / a.r) * rp + rank_slot(col % a.r);
#pragma unroll
        for (int p = 0; p < kPieces; ++p, to += kFewRows * ld) {
            *reinterpret_cast<unsigned*>(to) = next_piece(v.x, v.y, p == kPieces - 1);
            *reinterpret_cast<unsigned*>(to + 8) = next_piece(v.z, v.w, p == kPieces - 1);
        }
    }
    cluster.barrier_arrive();                  // no CTA leaves while another reads its sums
    __syncthreads();
    for (int i = first; i < last; i += kAdapterWarps) {
        const ColumnBlock now = block;
        UpFragments<kSteps> next;
        if (i + kAdapterWarps < last) {
            block = column_block(a, i + kAdapterWarps);
            load_up<kSteps, TO>(next, up + static_cast<size_t>(block.col) * a.r, a.r, 0, block.cols);
        }
        OldValues<1, TO> old;
        load_old<1, TO>(old, a, now, 0, s_rows);
        expand<1, kSteps, TO>(a, f, false, old, up + static_cast<size_t>(now.col) * a.r, now, shared_address(pieces), 2 * kFewRows * ld, ld, 0, s_rows);
        f = next;
    }
    cluster.barrier_wait();
}

// Many rows: x and `down` pass through a ring of stages of 64 values of K in shared memory (rows of 128 bytes, 16-byte pieces exchanged by the row's last
// three bits); warps share the rows in groups of 32 (16 where the tile has 64) and a stage's steps of k in two halves. With one pass over K (S r up to 64)
// the sums and their pieces lie where the ring was, else the sums have a place of their own.
template <int M, bool kOnePass> struct ManyShape {
    static constexpr int kStageBytes = (M + 64) * 128;
    static constexpr int kStages = (kOnePass ? 98304 : 81920) / kStageBytes;
    static constexpr int kGroups = M < 64 ? M / 16 : 4, kSplits = kAdapterWarps / kGroups, kTiles = M / 16 / kGroups, kSteps = 4 / kSplits;
};
constexpr int kManyCols = 64;                  // ranks of a pass over K

__device__ __forceinline__ void copy_16(unsigned to, const void* from, int bytes) {      // bytes: 16, or 0 for zeros (from is then an address of some memory)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(to), "l"(from), "r"(bytes) : "memory");
}

template <int M, bool kOnePass, int kSteps, typename TO>
__global__ void __launch_bounds__(kAdapterThreads, 2) adapter_many_kernel(AdapterArgs a) {
    pdl_prologue();
    using Shape = ManyShape<M, kOnePass>;
    constexpr int kTiles = Shape::kTiles;
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ int s_rows[M], s_scratch[kDirectEach * kAdapterWarps];
    cg::cluster_group cluster = cg::this_cluster();
    const int part = cluster.block_rank(), parts = cluster.num_blocks();
    int adapter, n;
    if (!find_rows<M>(a.plan, a.A, a.tile_rows, blockIdx.x / parts, s_rows, adapter, n, s_scratch)) return;     // (the whole cluster)
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    const int cols = a.S * a.r, rp = (a.r + 15) & ~15, ld = a.S * rp + 8, hs = cols + 8;
    const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(a.x);
    const __nv_bfloat16* down = static_cast<const __nv_bfloat16*>(a.down) + static_cast<size_t>(adapter) * cols * a.K;
    const __nv_bfloat16* up = static_cast<const __nv_bfloat16*>(a.up) + static_cast<size_t>(adapter) * a.N * a.r;
    float* h = reinterpret_cast<float*>(ring + (kOnePass ? 0 : Shape::kStages * Shape::kStageBytes));        // [M][hs]
    __nv_bfloat16* pieces = reinterpret_cast<__nv_bfloat16*>(ring + (kOnePass ? M * hs * sizeof(float) : 0));
    const float scale = a.scales[adapter];
    const int share = ((a.K + parts - 1) / parts + 63) / 64 * 64, k_begin = min(a.K, part * share), k_end = min(a.K, k_begin + share);
    const int stages = (k_end - k_begin + 63) / 64;
    const unsigned ring_at = shared_address(ring);
    const int group = warp % Shape::kGroups, split = warp / Shape::kGroups;
    // what a thread copies: 16 bytes of every 32nd row, always the same ones of the 128
    const int copy_row = threadIdx.x >> 3, copy_k = 8 * (threadIdx.x & 7);
    const unsigned copy_to = copy_row * 128 + (((threadIdx.x & 7) ^ (copy_row & 7)) << 4);
    const __nv_bfloat16* x_rows[M / 32];
    int x_bytes[M / 32];
#pragma unroll
    for (int i = 0; i < M / 32; ++i) {
        const int row = s_rows[copy_row + 32 * i];
        x_bytes[i] = row >= 0 ? 16 : 0;
        x_rows[i] = x + max(row, 0) * a.ldx + (row >= 0 ? k_begin + copy_k : 0);
    }
    // where a lane's fragments lie in a stage: their 16-byte piece for step s is exchanged by 2 s
    const unsigned x_at = (group * kTiles * 16 + (lane & 15)) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
    const int w_row = (lane & 7) + ((lane >> 4) << 3);
    const unsigned w_at = (M + w_row) * 128 + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
    for (int c0 = 0; c0 < (kOnePass ? 1 : cols); c0 += kManyCols) {
        const int some = min(kManyCols, cols - c0);
        const int w_rows = (some + 15) & ~15;
        int w_bytes[2];
        const __nv_bfloat16* w_from[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bool there = copy_row + 32 * i < some;
            w_bytes[i] = there ? 16 : 0;
            w_from[i] = down + (there ? static_cast<size_t>(c0 + copy_row + 32 * i) * a.K + k_begin + copy_k : 0);
        }
        auto fetch = [&](int stage, int slot) {
            const unsigned at = ring_at + slot * Shape::kStageBytes + copy_to;
            const int k = 64 * stage;
            if (k_begin + k + 64 <= k_end) {
#pragma unroll
                for (int i = 0; i < M / 32; ++i) copy_16(at + i * 32 * 128, x_rows[i] + (x_bytes[i] ? k : 0), x_bytes[i]);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (copy_row + 32 * i < w_rows) copy_16(at + (M + i * 32) * 128, w_from[i] + (w_bytes[i] ? k : 0), w_bytes[i]);
            } else {                           // the last stage may end early
                const bool in = k_begin + k + copy_k < k_end;
#pragma unroll
                for (int i = 0; i < M / 32; ++i) copy_16(at + i * 32 * 128, in && x_bytes[i] ? x_rows[i] + k : x, in ? x_bytes[i] : 0);
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (copy_row + 32 * i < w_rows) copy_16(at + (M + i * 32) * 128, in && w_bytes[i] ? w_from[i] + k : down, in ? w_bytes[i] : 0);
            }
        };
        float acc[kTiles][kManyCols / 8][4] = {};
#pragma unroll
        for (int i = 0; i < Shape::kStages - 1; ++i) {
            if (i < stages) fetch(i, i);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        int slot = 0, next = Shape::kStages - 1;
        for (int i = 0; i < stages; ++i) {
            asm volatile("cp.async.wait_group %0;" :: "n"(Shape::kStages - 2) : "memory");
            __syncthreads();                   // the stage is there for all, and the one before it is free
            if (i + Shape::kStages - 1 < stages) fetch(i + Shape::kStages - 1, next);
            asm volatile("cp.async.commit_group;" ::: "memory");
            const unsigned at = ring_at + slot * Shape::kStageBytes;
            next = slot;
            slot = slot + 1 == Shape::kStages ? 0 : slot + 1;
#pragma unroll
            for (int s = 0; s < Shape::kSteps; ++s) {
                const int step = Shape::kSteps * split + s;
                unsigned xa[kTiles][4], w[kManyCols / 16][4];          // (a step's fragments first: its products then wait for nothing)
#pragma unroll
                for (int m = 0; m < kTiles; ++m) load_matrices(xa[m], (at + x_at + m * 16 * 128) ^ (step << 5));
#pragma unroll
                for (int t = 0; t < kManyCols / 16; ++t)
                    if (16 * t < some) load_matrices(w[t], (at + w_at + t * 16 * 128) ^ (step << 5));
#pragma unroll
                for (int t = 0; t < kManyCols / 16; ++t)
                    if (16 * t < some) {
#pragma unroll
                        for (int m = 0; m < kTiles; ++m) {
                            mma_bf16(acc[m][2 * t], xa[m][0], xa[m][1], xa[m][2], xa[m][3], w[t][0], w[t][1]);
                            mma_bf16(acc[m][2 * t + 1], xa[m][0], xa[m][1], xa[m][2], xa[m][3], w[t][2], w[t][3]);
                        }
                    }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int p = 0; p < Shape::kSplits; ++p) {          // the warps that share the steps add up in their order
            __syncthreads();
            if (p == split)
#pragma unroll
                for (int m = 0; m < kTiles; ++m)
#pragma unroll
                    for (int t = 0; t < kManyCols / 8; ++t)
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const int row = (group * kTiles + m) * 16 + g + 8 * half, col = 8 * t + 2 * c;
                            if (col < some) {
                                float2* to = reinterpret_cast<float2*>(h + row * hs + c0 + col);
                                float2 v = make_float2(acc[m][t][2 * half], acc[m][t][2 * half + 1]);
                                if (p) { v.x += to->x; v.y += to->y; }
                                *to = v;
                            }
                        }
        }
    }
    __syncthreads();
    if (rp != a.r)                             // the slots of ranks that are not there
        for (int i = threadIdx.x; i < M * ld / 2 * kPieces; i += kAdapterThreads) reinterpret_cast<unsigned*>(pieces)[i] = 0u;
    // the warp's first columns of the second product are asked for before the cluster meets
    const int blocks = column_blocks(a), per = (blocks + parts - 1) / parts, first = part * per + warp, last = min(blocks, (part + 1) * per);
    UpFragments<kSteps> f;
    ColumnBlock block = {0, 0, 0};
    if (first < last) {
        block = column_block(a, first);
        load_up<kSteps, TO>(f, up + static_cast<size_t>(block.col) * a.r, a.r, 0, block.cols);
    }
    cluster.sync();
    // every CTA adds up its share of the tile's sums and gives their pieces to all
    const int fours = M * cols / 4, four_share = (fours + parts - 1) / parts, fours_end = min(fours, (part + 1) * four_share);
    for (int i = part * four_share + threadIdx.x; i < fours_end; i += kAdapterThreads) {
        const int row = 4 * i / cols, col = 4 * i % cols;
        float4 v = cluster_total(h + row * hs + col, scale, cluster, parts);
        __nv_bfloat16* to = pieces + row * ld + (col / a.r) * rp + rank_slot(col % a.r);
#pragma unroll
        for (int q = 0; q < kPieces; ++q, to += M * ld) {
            const unsigned p0 = next_piece(v.x, v.y, q == kPieces - 1), p1 = next_piece(v.z, v.w, q == kPieces - 1);
#pragma unroll
            for (int p = 0; p < kAdapterClusterMost; ++p)
                if (p < parts) {
                    *reinterpret_cast<unsigned*>(cluster.map_shared_rank(to, p)) = p0;
                    *reinterpret_cast<unsigned*>(cluster.map_shared_rank(to + 8, p)) = p1;
                }
        }
    }
    cluster.sync();
    OldValues<2, TO> old;
    if (first < last) load_old<2, TO>(old, a, block, 0, s_rows);
    for (int i = first; i < last; i += kAdapterWarps) {
        const ColumnBlock now = block;
        const __nv_bfloat16* from = up + static_cast<size_t>(now.col) * a.r;
        UpFragments<kSteps> after;             // of the next columns
        constexpr bool kAhead = kSteps < 4;      // (with four steps of ranks the registers are full)
        if (i + kAdapterWarps < last) {
            block = column_block(a, i + kAdapterWarps);
            if (kAhead) load_up<kSteps, TO>(after, up + static_cast<size_t>(block.col) * a.r, a.r, 0, block.cols);
        }
        for (int row0 = 0; row0 < n; row0 += 32) {
            OldValues<2, TO> next;             // of the turn that follows
            if (row0 + 32 < n) load_old<2, TO>(next, a, now, row0 + 32, s_rows);
            else if (i + kAdapterWarps < last) load_old<2, TO>(next, a, block, 0, s_rows);
            expand<2, kSteps, TO>(a, f, kSteps == 4 && a.r > 64 && row0 > 0, old, from, now, shared_address(pieces), 2 * M * ld, ld, row0, s_rows);
            old = next;
        }
        if (kAhead) f = after;
        else if (i + kAdapterWarps < last) load_up<kSteps, TO>(f, up + static_cast<size_t>(block.col) * a.r, a.r, 0, block.cols);
    }
}

// ---- 32-bit on the CUDA cores ----
// 700 rows of 2,048 into 2,048 at rank 12: 14 us (2.7 us of bytes), what bounds it the latency of the stages and the exchanges; 2,048 rows of 14,336 into
// 4,096 at rank 64: 213 us, 0.3 of the multiply-add rate, bound by the reads of shared memory. A tile's own count of rows bounds its work: one row of
// 4,096 at rank 16 10.6 us (15.9 us with all 32 rows of the tile), 8 rows of 2,048 into 8,192 at rank 32 19 us (30 us).
// x and `down` pass through a ring of stages of 32 values of K (rows of 128 bytes, 16-byte pieces exchanged by the row's last three bits). Of 16 neighbouring
// threads each has four columns of `kRows` rows, or with few ranks (S r below 64) a share of every stage's K instead, so that none is idle.
template <int kRows> struct FloatShape {
    static constexpr int kTile = 16 * kRows, kStageBytes = (kTile + 64) * 128, kStages = kRows == 1 ? 7 : kRows == 2 ? 6 : 5;
};
// Where a column's first 16-byte piece of a stage lies: the column's last three bits in reverse, so that eight neighbouring threads, whatever their share of
// columns and of pieces, read eight different ones (42 rows of 14,336 at rank 12, where four threads share K, tiles of 32 rows: 33 us, 42 us with the bits as they are).
__device__ __forceinline__ int piece_of(int col) { return (col & 1) << 2 | (col & 2) | (col >> 2 & 1); }
template <int kRows>
__global__ void __launch_bounds__(kAdapterThreads, 2) adapter_float_kernel(AdapterArgs a) {
    pdl_prologue();
    using Shape = FloatShape<kRows>;
    constexpr int M = Shape::kTile;
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ int s_rows[M], s_scratch[kDirectEach * kAdapterWarps];
    cg::cluster_group cluster = cg::this_cluster();
    const int part = cluster.block_rank(), parts = cluster.num_blocks();
    int adapter, n;
    if (!find_rows<M>(a.plan, a.A, a.tile_rows, blockIdx.x / parts, s_rows, adapter, n, s_scratch)) return;     // (the whole cluster)
    const int cols = a.S * a.r, hs = cols + 4;
    const float* x = static_cast<const float*>(a.x);
    const float* down = static_cast<const float*>(a.down) + static_cast<size_t>(adapter) * cols * a.K;
    const float* up = static_cast<const float*>(a.up) + static_cast<size_t>(adapter) * a.N * a.r;
    float* h = reinterpret_cast<float*>(ring + Shape::kStages * Shape::kStageBytes);         // [M][hs]: this CTA's sums
    float* sums = reinterpret_cast<float*>(ring);                                            // [M][hs]: the whole ones, where the ring was
    const float scale = a.scales[adapter];
    const int share = ((a.K + parts - 1) / parts + 31) / 32 * 32, k_begin = min(a.K, part * share), k_end = min(a.K, k_begin + share);
    const int stages = (k_end - k_begin + 31) / 32;
    const unsigned ring_at = shared_address(ring);
    const int copy_row = threadIdx.x >> 3, copy_k = 4 * (threadIdx.x & 7);
    const unsigned copy_to = copy_row * 128 + (((threadIdx.x & 7) ^ (copy_row & 7)) << 4), copy_col_to = copy_row * 128 + (((threadIdx.x & 7) ^ piece_of(copy_row)) << 4);
    constexpr int kCopies = (M + 31) / 32;
    const float* x_rows[kCopies];
    int x_bytes[kCopies];
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
        const int row = copy_row + 32 * i < M ? s_rows[copy_row + 32 * i] : -1;
        x_bytes[i] = row >= 0 ? 16 : 0;
        x_rows[i] = x + max(row, 0) * a.ldx;
    }
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    // `kThere` of the thread's rows for the columns c0 ..
    auto pass = [&](int c0, auto rows) {
        constexpr int kThere = decltype(rows)::value;
        const int some = min(64, cols - c0);
        int log_groups = 0;                    // threads across the columns: 2^log_groups of 16, the others share K
        while ((4 << log_groups) < some) ++log_groups;
        const int groups = 1 << log_groups, across = tx & (groups - 1), split = tx >> log_groups, splits = 16 >> log_groups;
        auto fetch = [&](int stage, int slot) {
            const unsigned at = ring_at + slot * Shape::kStageBytes;
            const int k = k_begin + 32 * stage + copy_k;
            const bool in = k < k_end;
#pragma unroll
            for (int i = 0; i < kCopies; ++i)
                if (copy_row + 32 * i < M) copy_16(at + copy_to + i * 32 * 128, in ? x_rows[i] + k : x, in ? x_bytes[i] : 0);
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (copy_row + 32 * i < 4 * groups) {
                    const bool there = in && copy_row + 32 * i < some;
                    copy_16(at + copy_col_to + (M + i * 32) * 128, there ? down + static_cast<size_t>(c0 + copy_row + 32 * i) * a.K + k : down, there ? 16 : 0);
                }
        };
        float acc[kThere][4] = {};
        __syncthreads();                       // (a further pass: the ring is free again)
#pragma unroll
        for (int i = 0; i < Shape::kStages - 1; ++i) {
            if (i < stages) fetch(i, i);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        int slot = 0, next = Shape::kStages - 1;
        for (int i = 0; i < stages; ++i) {
            asm volatile("cp.async.wait_group %0;" :: "n"(Shape::kStages - 2) : "memory");
            __syncthreads();                   // the stage is there for all, and the one before it is free
            if (i + Shape::kStages - 1 < stages) fetch(i + Shape::kStages - 1, next);
            asm volatile("cp.async.commit_group;" ::: "memory");
            const unsigned char* at = ring + slot * Shape::kStageBytes;
            next = slot;
            slot = slot + 1 == Shape::kStages ? 0 : slot + 1;
            for (int q = split; q < 8; q += splits) {
                float4 xv[kThere], w[4];
#pragma unroll
                for (int m = 0; m < kThere; ++m) {
                    const int row = ty + 16 * m;
                    xv[m] = *reinterpret_cast<const float4*>(at + row * 128 + ((q ^ (row & 7)) << 4));
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int col = across + groups * j;
                    w[j] = *reinterpret_cast<const float4*>(at + (M + col) * 128 + ((q ^ piece_of(col)) << 4));
                }
#pragma unroll
                for (int m = 0; m < kThere; ++m)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        acc[m][j] = fmaf(xv[m].x, w[j].x, acc[m][j]);
                        acc[m][j] = fmaf(xv[m].y, w[j].y, acc[m][j]);
                        acc[m][j] = fmaf(xv[m].z, w[j].z, acc[m][j]);
                        acc[m][j] = fmaf(xv[m].w, w[j].w, acc[m][j]);
                    }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int m = 0; m < kThere; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float v = acc[m][j];
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) {
                    const float y = __shfl_xor_sync(0xffffffffu, v, o);
                    if (o >= groups) v += y;   // (the threads that share K)
                }
                const int col = across + groups * j;
                if (split == 0 && col < some) h[(ty + 16 * m) * hs + c0 + col] = v;
            }
    };
    for (int c0 = 0; c0 < cols; c0 += 64)
        if (kRows == 1 || n <= 16) pass(c0, std::integral_constant<int, 1>{});
        else if constexpr (kRows > 1) pass(c0, std::integral_constant<int, kRows>{});
    cluster.sync();
    // every CTA adds up its share of the tile's sums and gives them to all
    const int fours = n * cols / 4, four_share = (fours + parts - 1) / parts, fours_end = min(fours, (part + 1) * four_share);
    for (int i = part * four_share + threadIdx.x; i < fours_end; i += kAdapterThreads) {
        const int row = 4 * i / cols, col = 4 * i % cols;
        const float4 v = cluster_total(h + row * hs + col, scale, cluster, parts);
#pragma unroll
        for (int p = 0; p < kAdapterClusterMost; ++p)
            if (p < parts) *reinterpret_cast<float4*>(cluster.map_shared_rank(sums + row * hs + col, p)) = v;
    }
    cluster.sync();
    float* out = static_cast<float*>(a.out);
    const int n_share = (a.N + parts - 1) / parts, n_begin = min(a.N, part * n_share), n_end = min(a.N, n_begin + n_share);
    // a column a thread, `kEach` rows from row0 on
    auto expand = [&](auto rows, int row0, int first, int step) {
        constexpr int kEach = decltype(rows)::value;
        for (int col = n_begin + first; col < n_end; col += step) {
            int slice = 0;
#pragma unroll
            for (int s = 0; s < kAdapterSlicesMost - 1; ++s) slice += s < a.S - 1 && col >= a.ends[s];
            const float* at = sums + row0 * hs + slice * a.r;
            const float* w_at = up + static_cast<size_t>(col) * a.r;
            float acc[kEach] = {};
            for (int j = 0; j < a.r; j += 4) {
                const float4 w = __ldg(reinterpret_cast<const float4*>(w_at + j));
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const float4 v = *reinterpret_cast<const float4*>(at + i * hs + j);
                    acc[i] = fmaf(v.x, w.x, fmaf(v.y, w.y, fmaf(v.z, w.z, fmaf(v.w, w.w, acc[i]))));
                }
            }
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int row = s_rows[row0 + i];
                if (row >= 0) asm volatile("red.global.add.f32 [%0], %1;" :: "l"(out + row * a.ldo + col), "f"(acc[i]) : "memory");
            }
        }
    };
    // (few rows: all threads across the columns; many: half of the rows a thread)
    if (n <= 4) {
        expand(std::integral_constant<int, 4>{}, 0, threadIdx.x, kAdapterThreads);
    } else if (kRows == 1 || n <= 16) {
        expand(std::integral_constant<int, 16>{}, 0, threadIdx.x, kAdapterThreads);
    } else if constexpr (kRows > 1) {
        const int row0 = (threadIdx.x >> 7) * (M / 2);
        if (row0 < n) expand(std::integral_constant<int, M / 2>{}, row0, threadIdx.x & 127, 128);
    }
}

template <typename... KArgs, typename... Args>
inline void launch_tile_clusters(void (*kernel)(KArgs...), long long tiles, int parts, int threads, size_t smem, cudaStream_t stream, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(tiles * parts));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = g_pdl_enabled ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = parts;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    counted(cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...));
}

// The tiles that a launch may have, and how many there are as a rule: every adapter could leave a tile that is not full, in large steps few do.
struct TileCount { long long most, busy; };
inline TileCount tile_count(const AdapterArgs& a, int rows) {
    const long long adapters = a.used < a.plan.T ? a.used : a.plan.T, full = (a.plan.T + rows - 1) / rows;
    if (a.tile_rows) return {(a.plan.T / a.tile_rows + adapters) * ((a.tile_rows + rows - 1) / rows), full};
    const long long most = a.plan.T / rows + adapters;
    return {most, a.plan.T <= kFewTokens ? most : full};
}
// CTAs of a cluster: as many as two a multiprocessor have room for (`slack`: twice as many). Powers of two: clusters of three and six, which would
// fill more places, do not all find theirs at once (3,000 rows into 16,384 columns, 94 tiles: clusters of two 141 us, of three 186 us).
inline int cluster_parts(long long tiles, int slack) {
    int parts = 1;
    while (parts < kAdapterClusterMost && 2 * parts * tiles <= 2LL * sm_count() * slack) parts *= 2;
    return parts;
}

template <typename Kernel>
int launch_adapter(Kernel kernel, SharedLimit& limit, const AdapterArgs& a, int rows, size_t smem, size_t most, cudaStream_t st) {
    const cudaError_t e = limit.allow(reinterpret_cast<const void*>(kernel), static_cast<int>(most));
    GI_REQUIRE(e == cudaSuccess, "adapter_product: %s", cudaGetErrorString(e));
    const TileCount tiles = tile_count(a, rows);
    const int parts = cluster_parts(tiles.busy, a.plan.T <= kFewTokens ? 2 : 1);
    launch_tile_clusters(kernel, tiles.most, parts, kAdapterThreads, smem, st, a);
    return check_launch("adapter_product");
}

template <typename T, typename TO>
int launch_plain(const AdapterArgs& a, cudaStream_t st) {
    static SharedLimit limit;
    return launch_adapter(&adapter_plain_kernel<T, TO>, limit, a, kPlainRows, 2ull * kPlainRows * a.S * a.r * sizeof(float),
                          2ull * kPlainRows * kAdapterRanksMost * sizeof(float), st);
}

inline size_t pieces_bytes(const AdapterArgs& a, int rows) {
    return 2ull * kPieces * rows * (a.S * ((a.r + 15) / 16 * 16) + 8);
}
inline size_t sums_bytes(const AdapterArgs& a, int rows) { return 4ull * rows * (a.S * a.r + 8); }
template <typename Shape> constexpr size_t ring_bytes() { return static_cast<size_t>(Shape::kStages) * Shape::kStageBytes; }

// Whether what lies where the ring was fits there.
template <int M, bool kOnePass> inline bool fits(const AdapterArgs& a) {
    return (kOnePass ? sums_bytes(a, M) : 0) + pieces_bytes(a, M) <= ring_bytes<ManyShape<M, kOnePass>>();
}

template <int kSteps, typename TO>
int launch_few(const AdapterArgs& a, cudaStream_t st) {
    static SharedLimit limit;
    return launch_adapter(&adapter_few_kernel<kSteps, TO>, limit, a, kFewRows, 4ull * kFewRows * a.S * a.r + pieces_bytes(a, kFewRows),
                          150 * 1024, st);
}

template <int M, bool kOnePass, int kSteps, typename TO>
int launch_many(const AdapterArgs& a, cudaStream_t st) {
    static SharedLimit limit;
    const size_t ring = ring_bytes<ManyShape<M, kOnePass>>();
    return launch_adapter(&adapter_many_kernel<M, kOnePass, kSteps, TO>, limit, a, M, kOnePass ? ring : ring + sums_bytes(a, M),
                          210 * 1024, st);
}

template <int kRows>
int launch_float(const AdapterArgs& a, cudaStream_t st) {
    static SharedLimit limit;
    using Shape = FloatShape<kRows>;
    return launch_adapter(&adapter_float_kernel<kRows>, limit, a, Shape::kTile,
                          ring_bytes<Shape>() + 4ull * Shape::kTile * (a.S * a.r + 4), 160 * 1024, st);
}

int launch_f32(const AdapterArgs& a, cudaStream_t st) {
    const bool pieces = a.K % 4 == 0 && a.ldx % 4 == 0 && a.r % 4 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0 &&
                        reinterpret_cast<uintptr_t>(a.down) % 16 == 0 && reinterpret_cast<uintptr_t>(a.up) % 16 == 0;
    if (!pieces) return launch_plain<float, float>(a, st);
    // (tiles of 32 and of 64 rows, four prompts: 14,336 into 4,096 at rank 64, 2,000 rows 266 and 296 us, 2,500 503 and 396; 2,048 into 2,048 at rank 16 28 and 27, 46 and 40:
    // beyond about 2,100 rows tiles of 32 take a second round. 1,500 rows 265 and 206 us, 28 and 25: there tiles of 64 would be faster)
    if (a.plan.T >= 2048 && a.S * a.r <= 256) return launch_float<4>(a, st);
    // (tiles of 16 and of 32 rows: 260 rows of 14,336 into 4,096 at rank 64, four adapters, 104 and 123 us, 400 rows of 24 adapters 176 and 132; tiles of 16 rows: 250 rows of 4,096 into 4,096, two adapters of rank 64, 45 us, of 32 66 us, and 42 of
    // 14,336 at rank 12 26 and 33 us; 150 of 8,192 into 2,048, four of rank 64, 58 and 53 us)
    if (a.plan.T <= kFewTokens) return launch_float<1>(a, st);
    return launch_float<2>(a, st);
}

template <int kSteps, typename TO>
int launch_steps(const AdapterArgs& a, cudaStream_t st) {
    // (tiles of 16 rows, or of 32 through the ring: 260 rows of four adapters, 2,048 into 16,384 at rank 32, 19 and 25 us, 14,336 into 4,096 at rank 64 21 and 25; 400 rows of 24
    // adapters 33 and 28, 46 and 29: where each adapter may leave a tile that is not full, small ones are too many)
    if (a.plan.T <= kFewTokens) return launch_few<kSteps, TO>(a, st);
    if (a.S * a.r <= kManyCols) {
        // (tiles of 32 and of 64 rows, four prompts: 4,096 into 6,144 at rank 16, 2,000 rows 38 and 46 us, 2,500 54 and 53, 6,000 107 and 99; 8,192 into 2,048 24 and 24, 36 and
        // 34, 62 and 54; 14,336 into 4,096 at rank 64 48 and 44, 80 and 68, 148 and 121: up to about 2,100 rows tiles of 32 run in one round of clusters of four)
        if (a.plan.T <= 2048 && fits<32, true>(a)) return launch_many<32, true, kSteps, TO>(a, st);
        if (fits<64, true>(a)) return launch_many<64, true, kSteps, TO>(a, st);
    }
    // (several passes: tiles of 32 rows leave two blocks a multiprocessor, 1,000 rows into [q; k; v] at rank 64 43 us, of 64 rows 71 us)
    if (fits<32, false>(a)) return launch_many<32, false, kSteps, TO>(a, st);
    return launch_few<kSteps, TO>(a, st);
}

template <typename TO>
int launch_bf16(const AdapterArgs& a, cudaStream_t st) {
    // 16-byte pieces of x and `down`, 8-byte ones of `up`
    const bool pieces = a.K % 8 == 0 && a.ldx % 8 == 0 && a.r % 4 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0 &&
                        reinterpret_cast<uintptr_t>(a.down) % 16 == 0 && reinterpret_cast<uintptr_t>(a.up) % 8 == 0;
    if (!pieces) return launch_plain<__nv_bfloat16, TO>(a, st);
    return a.r <= 16 ? launch_steps<1, TO>(a, st) : a.r <= 32 ? launch_steps<2, TO>(a, st) : launch_steps<4, TO>(a, st);
}

}  // namespace gi

using namespace gi;

// Rows of a step whose products need no plan, with so many adapters.
extern "C" int gi_adapter_direct_rows(int A) { return A <= kDirectAdapters ? kDirectRows : 0; }
// Ranks of all slices together, and adapters, at most.
extern "C" int gi_adapter_ranks_most() { return kAdapterRanksMost; }
extern "C" int gi_adapter_adapters_most() { return kPlanAdaptersMost; }

static int gi_adapter_plan_impl(const int* row_adapter, int T, int A, int tile_rows, int* plan, void* stream) {
    GI_REQUIRE(T >= 0 && A > 0 && tile_rows > 0, "adapter_plan: sizes must be positive (T=%d, adapters=%d, tile rows=%d)", T, A, tile_rows);
    GI_REQUIRE(A <= kPlanAdaptersMost, "adapter_plan: %d adapters exceed the limit of %d", A, kPlanAdaptersMost);
    launch_kernel((adapter_plan_kernel), dim3(1), dim3(kPlanThreads), A * sizeof(int), static_cast<cudaStream_t>(stream), row_adapter, T, A, tile_rows, plan);
    return check_launch("adapter_plan");
}

// x [T, K] with ldx values between rows; down [A, S r, K]; up [A, N, r]; out [T, N] with ldo values between rows; end0 ..: the slices' last columns + 1.
// used: so many adapters occur at most. tile_rows > 0: plan is adapter_plan's; 0 (up to gi_adapter_direct_rows() rows): plan is row_adapter [T] itself.
static int gi_adapter_product_impl(const void* x, long long ldx, int dtype, const void* down, const void* up, const float* scales, const int* plan, int T,
                                   int A, int used, int tile_rows, void* out, long long ldo, int out_dtype, int K, int N, int r, int S, int end0, int end1,
                                   int end2, int end3, void* stream) {
    if (T == 0) return 0;
    GI_REQUIRE(T > 0 && A > 0 && used > 0 && K > 0 && N > 0 && r > 0 && tile_rows >= 0, "adapter_product: sizes must be positive (T=%d, adapters=%d, K=%d, N=%d, rank=%d)",
               T, A, K, N, r);
    GI_REQUIRE(tile_rows > 0 || T <= gi_adapter_direct_rows(A), "adapter_product: %d rows need a plan", T);
    GI_REQUIRE(S >= 1 && S <= kAdapterSlicesMost, "adapter_product: %d slices (1 to %d)", S, kAdapterSlicesMost);
    GI_REQUIRE(static_cast<long long>(S) * r <= kAdapterRanksMost, "adapter_product: %d slices of rank %d exceed %d", S, r, kAdapterRanksMost);
    AdapterArgs a = {x, ldx, down, up, scales, {plan, T}, out, ldo, A, used, K, N, r, S, tile_rows, {end0, end1, end2, end3}, 0};
    int before = 0;
    for (int s = 0; s < S; ++s) {
        GI_REQUIRE(a.ends[s] > before, "adapter_product: a slice without columns");
        before = a.ends[s];
    }
    GI_REQUIRE(before == N, "adapter_product: the slices have %d columns, the output %d", before, N);
    a.wide = reinterpret_cast<uintptr_t>(out) % 16 == 0 && ldo * (out_dtype == kF32 ? 4 : 2) % 16 == 0;
    GI_REQUIRE(dtype == kBF16 || out_dtype == kF32, "adapter_product: 32-bit weights give 32-bit output");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == kF32) return launch_f32(a, st);
    return out_dtype == kF32 ? launch_bf16<float>(a, st) : launch_bf16<__nv_bfloat16>(a, st);
}

extern "C" int gi_adapter_plan(const int* row_adapter, int T, int A, int tile_rows, int* plan, void* stream) {
    return gi::dispatch(gi_adapter_plan_impl, row_adapter, T, A, tile_rows, plan, stream);
}

extern "C" int gi_adapter_product(const void* x, long long ldx, int dtype, const void* down, const void* up, const float* scales, const int* plan, int T,
                                  int A, int used, int tile_rows, void* out, long long ldo, int out_dtype, int K, int N, int r, int S, int end0, int end1,
                                  int end2, int end3, void* stream) {
    return gi::dispatch(gi_adapter_product_impl, x, ldx, dtype, down, up, scales, plan, T, A, used, tile_rows, out, ldo, out_dtype, K, N, r, S, end0, end1,
                        end2, end3, stream);
}
