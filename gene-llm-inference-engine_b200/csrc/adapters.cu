// Low-rank adapters of many requests beside a shared projection:
//   out[t, n] += scale_a * sum_j up_a[n, j] * (sum_k x[t, k] down_a[s(n) * r + j, k]),  a = the adapter of row t (none: nothing),
// s(n) the slice of column n (q | k | v, or gate | up, stacked in one output, each with a pair of matrices of its own).
//
// The rows of a step are put in the adapters' order once (adapter_plan) and cut into tiles of one adapter each. A cluster of CTAs
// takes a tile: every CTA multiplies its share of K, the partial sums [rows, S r] are added through distributed shared
// memory, and every CTA writes its share of the columns. x, out and the weights cross memory once; the r values in between never do.
#include <climits>

#include <cooperative_groups.h>

#include "common.cuh"
#include "device_limit.h"

namespace gi {

namespace cg = cooperative_groups;

constexpr int kPlanThreads = 1024;
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
    auto adapter = [&](int t) {
        const int a = t < T ? row_adapter[t] : -1;
        return a >= 0 && a < A ? a : -1;
    };
    for (int t0 = 0; t0 < T; t0 += kPlanThreads) {
        const int a = adapter(t0 + threadIdx.x);
        const unsigned same = __match_any_sync(0xffffffffu, a);
        if (a >= 0 && lane == __ffs(same) - 1) atomicAdd(&counts[a], __popc(same));
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
    for (int t0 = 0; t0 < T; t0 += kPlanThreads) {
        const int t = t0 + threadIdx.x, a = adapter(t);
        const unsigned same = __match_any_sync(0xffffffffu, a);
        const int leader = __ffs(same) - 1;
        int place = 0;
        if (a >= 0 && lane == leader) place = atomicAdd(&counts[a], __popc(same));
        place = __shfl_sync(0xffffffffu, place, leader) + __popc(same & ((1u << lane) - 1));
        if (a >= 0) plan[1 + place] = t;
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
    int K, N, r, S, tile_rows;
    int ends[kAdapterSlicesMost];              // a slice's last column + 1
};

// ---- any type, any size: on the CUDA cores, in 32 bits ----
constexpr int kPlainThreads = 256, kPlainRows = 32, kPlainCols = 64, kPlainK = 32;

template <typename T, typename TO>
__global__ void __launch_bounds__(kPlainThreads) adapter_plain_kernel(AdapterArgs a) {
    pdl_prologue();
    extern __shared__ float h[];               // [2][kPlainRows][S r]: this CTA's partial sums, then the whole sums
    __shared__ float xs[kPlainRows][kPlainK + 1], ds[kPlainCols][kPlainK + 1];
    __shared__ int s_rows[kPlainRows];
    cg::cluster_group cluster = cg::this_cluster();
    const int part = cluster.block_rank(), parts = cluster.num_blocks();
    const int per_tile = (a.tile_rows + kPlainRows - 1) / kPlainRows;
    const int which = blockIdx.x / parts, tile = which / per_tile, piece = which % per_tile;
    if (tile >= a.plan.tiles()) return;        // (the whole cluster)
    const int* info = a.plan.tile(tile);
    const int adapter = info[0], first = info[1] + piece * kPlainRows, rows = min(kPlainRows, info[2] - piece * kPlainRows);
    if (rows <= 0) return;
    if (threadIdx.x < kPlainRows) s_rows[threadIdx.x] = threadIdx.x < rows ? a.plan.rows()[first + threadIdx.x] : -1;
    __syncthreads();
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

// CTAs of a tile's cluster: enough for two on every multiprocessor.
inline int cluster_parts(long long tiles) {
    int parts = 1;
    while (parts < kAdapterClusterMost && tiles * parts < 2LL * sm_count()) parts *= 2;
    return parts;
}

template <typename T, typename TO>
int launch_plain(const AdapterArgs& a, long long tiles, cudaStream_t st) {
    static SharedLimit limit;
    const long long pieces = tiles * ((a.tile_rows + kPlainRows - 1) / kPlainRows);
    const size_t smem = 2ull * kPlainRows * a.S * a.r * sizeof(float);
    const cudaError_t e = limit.allow(reinterpret_cast<const void*>(&adapter_plain_kernel<T, TO>), 2 * kPlainRows * kAdapterRanksMost * sizeof(float));
    GI_REQUIRE(e == cudaSuccess, "adapter_product: %s", cudaGetErrorString(e));
    launch_tile_clusters((adapter_plain_kernel<T, TO>), pieces, cluster_parts(pieces), kPlainThreads, smem, st, a);
    return check_launch("adapter_product");
}

}  // namespace gi

using namespace gi;

static int gi_adapter_plan_impl(const int* row_adapter, int T, int A, int tile_rows, int* plan, void* stream) {
    GI_REQUIRE(T >= 0 && A > 0 && tile_rows > 0, "adapter_plan: sizes must be positive (T=%d, adapters=%d, tile rows=%d)", T, A, tile_rows);
    GI_REQUIRE(A <= kPlanAdaptersMost, "adapter_plan: %d adapters exceed the limit of %d", A, kPlanAdaptersMost);
    launch_kernel((adapter_plan_kernel), dim3(1), dim3(kPlanThreads), A * sizeof(int), static_cast<cudaStream_t>(stream), row_adapter, T, A, tile_rows, plan);
    return check_launch("adapter_plan");
}

// x [T, K] with ldx values between rows; down [A, S r, K]; up [A, N, r]; out [T, N] with ldo values between rows; ends [S]: host memory, read
// during the call; tiles: the most that the plan can have.
static int gi_adapter_product_impl(const void* x, long long ldx, int dtype, const void* down, const void* up, const float* scales, const int* plan, int T,
                                   int tile_rows, int tiles, void* out, long long ldo, int out_dtype, int K, int N, int r, int S, int end0, int end1, int end2,
                                   int end3, void* stream) {
    if (T == 0 || tiles == 0) return 0;
    GI_REQUIRE(T > 0 && K > 0 && N > 0 && r > 0 && tile_rows > 0 && tiles > 0, "adapter_product: sizes must be positive (T=%d, K=%d, N=%d, rank=%d)", T, K, N, r);
    GI_REQUIRE(S >= 1 && S <= kAdapterSlicesMost, "adapter_product: %d slices (1 to %d)", S, kAdapterSlicesMost);
    GI_REQUIRE(static_cast<long long>(S) * r <= kAdapterRanksMost, "adapter_product: %d slices of rank %d exceed %d", S, r, kAdapterRanksMost);
    AdapterArgs a = {x, ldx, down, up, scales, {plan, T}, out, ldo, K, N, r, S, tile_rows, {end0, end1, end2, end3}};
    int before = 0;
    for (int s = 0; s < S; ++s) {
        GI_REQUIRE(a.ends[s] > before, "adapter_product: a slice without columns");
        before = a.ends[s];
    }
    GI_REQUIRE(before == N, "adapter_product: the slices have %d columns, the output %d", before, N);
    GI_REQUIRE(static_cast<long long>(tiles) * tile_rows <= INT_MAX / kAdapterClusterMost, "adapter_product: %d tiles exceed the grid limit", tiles);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    GI_REQUIRE(dtype == kBF16 || out_dtype == kF32, "adapter_product: 32-bit weights give 32-bit output");
    if (dtype == kF32) return launch_plain<float, float>(a, tiles, st);
    return out_dtype == kF32 ? launch_plain<__nv_bfloat16, float>(a, tiles, st) : launch_plain<__nv_bfloat16, __nv_bfloat16>(a, tiles, st);
}

extern "C" int gi_adapter_plan(const int* row_adapter, int T, int A, int tile_rows, int* plan, void* stream) {
    return gi::dispatch(gi_adapter_plan_impl, row_adapter, T, A, tile_rows, plan, stream);
}

extern "C" int gi_adapter_product(const void* x, long long ldx, int dtype, const void* down, const void* up, const float* scales, const int* plan, int T,
                                  int tile_rows, int tiles, void* out, long long ldo, int out_dtype, int K, int N, int r, int S, int end0, int end1, int end2,
                                  int end3, void* stream) {
    return gi::dispatch(gi_adapter_product_impl, x, ldx, dtype, down, up, scales, plan, T, tile_rows, tiles, out, ldo, out_dtype, K, N, r, S, end0, end1, end2,
                        end3, stream);
}
