// Matrix product in 8-bit integers on the 5th-generation tensor cores, scales for every row and channel:
//
//   out[t, n] (+)= scale_a[t] * scale_w[n] * sum over k of a[t, k] * w[n, k]
//
// tcgen05.mma kind::i8 adds the products in 32-bit integers in tensor memory. They are exact (K up to 131,056, which the host
// checks), so a result depends neither on how K is cut nor on which of the two kernels below computed it: every sum is turned
// into a float once, multiplied by the row's scale, then by the channel's, in that order everywhere (so the sum times the row's scale has to lie within the
// range of 32 bits), and what it is added to is added once, rounded to nearest, subnormals kept, by either kernel.
//
// The weights lie in tiles of 128 channels x 128 values of K, 16 KB each, [channel tile][block of K][128][128] with K padded to whole
// blocks by zeros and every row's eight 16-byte pieces permuted by piece ^ (row % 8): a tile in memory is what tcgen05.mma
// reads in shared memory (K-major, 128-byte swizzle), so a tile is one stretch of memory and both kernels read the same one copy.
// Weights of a gated pair lie gate tile, up tile, gate tile, .. (each part padded to whole tiles).
//
// Few rows (int8_few_kernel). The weights take the 128-row side and up to 128 rows of activations the narrow side. What bounds it is
// the stream of the weights: a CTA keeps its share of shared memory full of bulk copies and computes as they land. K is cut over the CTAs of
// a cluster until the SMs have work; each CTA then collects the sums of its share of the rows from the others' shared memory
// (integers, so in any order), scales and stores them.
//
// Many rows (int8_many_kernel). Pairs of CTAs (cta_group::2) on tiles of 256 rows x 256 channels, persistent, accumulators
// twice in tensor memory so that the epilogue of a tile runs beside the products of the next. Epilogues: 32-bit store or addition and
// bfloat16 store by TMA from a staging buffer (or by the lanes' loads and stores, where the output's rows are not whole 16 bytes), and act(gate) * up in
// bfloat16 for gated weights.
//
// Every wait is bounded: where a limit is hit the kernel records a code in the status word, stops issuing work, lets its own copies
// land, frees its tensor memory and returns.
#include "common.cuh"
#include "device_limit.h"
#include "tma.cuh"

namespace gi {
namespace {

constexpr int kTileRows = 128;                      // channels of a weight tile
constexpr int kRowBytes = 128;                      // values of K in a block: one swizzle row
constexpr int kTileBytes = kTileRows * kRowBytes;
constexpr unsigned long long kWaitCycles = 4000000000ull;      // about two seconds

enum Int8Error : int { kErrProducer = 41, kErrMma = 42, kErrEpilogue = 43, kErrDrain = 44 };

// ------------------------------------------------------------------------------------------ PTX
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_arrive_remote(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
template <bool CLUSTER>
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    if (CLUSTER)
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Bounded: false where the limit is hit (recorded) or another role of the CTA has given up.
template <bool CLUSTER = false>
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* gave_up, int* status, int code) {
    if (bar_try<CLUSTER>(bar, parity)) return true;
    const unsigned long long t0 = clock64();
    while (!bar_try<CLUSTER>(bar, parity)) {
        if (*gave_up) return false;
        if (clock64() - t0 > kWaitCycles) {
            *gave_up = 1;
            atomicCAS(status, 0, code);
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ uint32_t map_to(uint32_t local, uint32_t rank) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
    return remote;
}
__device__ __forceinline__ void store_cluster(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// the two halves of a barrier over the cluster's threads
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }

__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(bar) : "memory");
}
// into this CTA's shared memory, the bytes counted on a barrier of either CTA of the pair
__device__ __forceinline__ void load_tile_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(bar) : "memory");
}
__device__ __forceinline__ void load_bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar, uint64_t policy) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar), "l"(policy) : "memory");
}
__device__ __forceinline__ uint64_t read_once_policy() {
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}
__device__ __forceinline__ void store_tile(const CUtensorMap* map, uint32_t src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void add_tile(const CUtensorMap* map, uint32_t src, int c0, int c1) {
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.bulk_group [%0, {%2, %3}], [%1];"
                 ::"l"(map), "r"(src), "r"(c0), "r"(c1) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tmem_allocate(uint32_t dst, uint32_t cols) {
    if (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
    if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
template <bool PAIR>
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// arrives on the barrier once the products issued so far are done; of a pair's products on the barriers at this place in both CTAs
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mma_commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                   "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_load8(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(addr));
}
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// K-major tile in shared memory, 128-byte swizzle, groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr) {
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (1ull << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// D 32-bit integers (2 at bit 4), A and B signed 8-bit (1 at bits 7 and 10), both K-major; N / 8 at bit 17, M / 16 at bit 24
constexpr uint32_t int8_idesc(int m, int n) { return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24); }

__device__ __forceinline__ float scaled(int sum, float row, float channel) { return __fmul_rn(__fmul_rn(static_cast<float>(sum), row), channel); }

// ------------------------------------------------------------------------------------------ few rows
struct FewParams {
    const uint8_t* tiles;
    const float* a_scales;
    const float* w_scales;
    void* out;               // out[t * ldo + n]
    long long ldo;
    int T, N;                // N: channels of a part (gated weights: of gate and of up)
    int gated;
    int total_kb, kb_per_split, splits;
    int stages;
    int w_constant;          // no kernel that may still be running writes the tiles: the first ones may be asked for before the wait
    int* status;
};

enum Epilogue : int { kStoreF32 = 0, kAddF32 = 1, kStoreBF16 = 2, kGatedBF16 = 3, kAddLanesF32 = 4 };      // (the last: many rows whose outputs TMA cannot address)

// Measured on B200 in a stream of launches, weights from memory: 8 rows 4096 -> 28672 18.4 us (6.4 TB/s), 64 rows 21.2; one token 8192 -> 2048 5.4 us, 2048 ->
// 2048 3.5 (the hand-over from launch to launch, first operands and the cluster's exchange, about 3 us); 400 rows 4096 -> 4096 14.4.
// Tiles of BQ rows. Tiles of 8 have one group of four epilogue warps, larger ones two that take turns (one token through 8192 -> 2048 with 16 rows to a
// tile: 5.9 us with one group, 6.4 with two; 64 rows through 4096 -> 4096: 8.8 and 8.0).
template <int BQ>
struct FewConfig {
    static constexpr int kGroups = BQ <= 8 ? 1 : 2;
    static constexpr int kThreads = 64 + 128 * kGroups;        // producer, MMA, epilogue
    static constexpr int kKb = BQ <= 8 ? 2 : 1;                // blocks of K to a stage
    static constexpr int kBlockBytes = kTileBytes + BQ * kRowBytes;
    static constexpr int kStageBytes = kKb * kBlockBytes;
    static constexpr int kTmemCols = BQ < 32 ? 32 : BQ;
    static constexpr int kSideBytes = 256 + 4 * BQ;            // barriers, flags, the rows' scales
    // the sums that the CTAs of a cluster hand each other: equal shares of a tile's rows, the last one padded
    static constexpr int meet(int rows, int splits) { return splits > 1 ? (rows + splits - 1) / splits * splits * kTileRows * 4 : 0; }
    static constexpr int smem(int stages, int rows, int splits) { return stages * kStageBytes + meet(rows, splits) + kSideBytes; }
};

// A kernel for each epilogue, with and without a cluster: a short kernel pays for every instruction that it has to fetch.
template <int BQ, int EPI, bool CLUSTER>
__global__ void __launch_bounds__(FewConfig<BQ>::kThreads)
int8_few_kernel(const __grid_constant__ CUtensorMap map_a, const FewParams p) {
    using Cfg = FewConfig<BQ>;
    constexpr int kKb = Cfg::kKb;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int stages = p.stages, splits = CLUSTER ? p.splits : 1;
    uint8_t* behind = smem + stages * Cfg::kStageBytes;
    int* meet = reinterpret_cast<int*>(behind);                // [split][rows of a CTA's share][128]
    if (CLUSTER) behind += Cfg::meet(min(BQ, p.T), splits);
    uint64_t* bars = reinterpret_cast<uint64_t*>(behind);      // [0, 8) full, [8, 16) empty, [16] sums complete
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 17);
    volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* row_scales = reinterpret_cast<float*>(behind + 256);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile_n = blockIdx.x, tile_t = blockIdx.y, split = CLUSTER ? blockIdx.z : 0;
    const int kb_begin = split * p.kb_per_split;
    const int n_kb = min(p.total_kb, kb_begin + p.kb_per_split) - kb_begin;
    const int n_steps = (n_kb + kKb - 1) / kKb;

    if (threadIdx.x == 0) {
        timeline_record(kTlInt8ProductFew, 0);
        for (int s = 0; s < stages; ++s) {
            bar_init(smem_addr(&bars[s]), 1);
            bar_init(smem_addr(&bars[8 + s]), 1);
        }
        bar_init(smem_addr(&bars[16]), 1);
        *gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_allocate<false>(smem_addr(tmem_slot), Cfg::kTmemCols);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
    if (CLUSTER) cluster_arrive();

    if (warp == 0) {
        if (lane == 0) {
            const uint64_t policy = read_once_policy();
            const uint8_t* src = p.tiles + (static_cast<size_t>(tile_n) * p.total_kb + kb_begin) * kTileBytes;
            auto blocks_of = [&](int i) { return min(kKb, n_kb - i * kKb); };
            auto load_w = [&](int i, int s) {
                bar_expect(smem_addr(&bars[s]), blocks_of(i) * Cfg::kBlockBytes);
                load_bulk(smem_addr(smem + s * Cfg::kStageBytes), src + static_cast<size_t>(i) * kKb * kTileBytes, blocks_of(i) * kTileBytes,
                          smem_addr(&bars[s]), policy);
            };
            auto load_a = [&](int i, int s) {
                for (int j = 0; j < blocks_of(i); ++j)
                    load_tile(smem_addr(smem + s * Cfg::kStageBytes + kKb * kTileBytes + j * BQ * kRowBytes), &map_a,
                              (kb_begin + i * kKb + j) * kRowBytes, tile_t * BQ, smem_addr(&bars[s]));
            };
            // constant weights: their first tiles are asked for before the wait for the kernels ahead
            const int early = min(n_steps, stages);
            if (p.w_constant)
                for (int i = 0; i < early; ++i) load_w(i, i);
            pdl_wait();
            timeline_record(kTlInt8ProductFew, 1);
            for (int i = 0; i < early; ++i) {
                if (!p.w_constant) load_w(i, i);
                load_a(i, i);
            }
            int issued = early, s = 0, parity = 0;
            for (int i = early; i < n_steps; ++i) {      // (early == stages, where there are more steps)
                if (!bar_wait(smem_addr(&bars[8 + s]), parity, gave_up, p.status, kErrProducer)) break;
                load_w(i, s);
                load_a(i, s);
                issued = i + 1;
                if (++s == stages) { s = 0; parity ^= 1; }
            }
            if (*gave_up) {      // every copy must have landed before the CTA leaves
                for (int i = max(0, issued - stages); i < issued; ++i) {
                    const unsigned long long t0 = clock64();
                    while (!bar_try<false>(smem_addr(&bars[i % stages]), (i / stages) & 1))
                        if (clock64() - t0 > kWaitCycles) { atomicCAS(p.status, 0, kErrDrain); break; }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = int8_idesc(kTileRows, BQ);
            pdl_wait();          // the rows come with the kernels ahead: the waits' limit counts from their end, and this kernel's copies alone
            bool ok = true;
            int s = 0, parity = 0;
            for (int i = 0; i < n_steps; ++i) {
                if (!bar_wait(smem_addr(&bars[s]), parity, gave_up, p.status, kErrMma)) { ok = false; break; }
                fence_after();
                if (i == 0) timeline_record(kTlInt8ProductFew, 2);
                const uint32_t at = smem_addr(smem + s * Cfg::kStageBytes);
                const int blocks = min(kKb, n_kb - i * kKb);
#pragma unroll 1
                for (int j = 0; j < blocks; ++j) {
                    const uint64_t w = tile_desc(at + j * kTileBytes), a = tile_desc(at + kKb * kTileBytes + j * BQ * kRowBytes);
#pragma unroll
                    for (int k = 0; k < kRowBytes / 32; ++k)      // 32 values of K to an instruction
                        mma_i8<false>(tmem, w + 2 * k, a + 2 * k, idesc, (i > 0 || j > 0 || k > 0) ? 1u : 0u);
                }
                mma_commit(smem_addr(&bars[8 + s]));
                if (++s == stages) { s = 0; parity ^= 1; }
            }
            if (ok) mma_commit(smem_addr(&bars[16]));
            timeline_record(kTlInt8ProductFew, 3);
        }
    }
    __syncwarp();
    // ---------------------------------------------------------------- the sums
    const int lane_group = warp & 3;
    const int row = lane_group * 32 + lane;                                  // the channel within the tile = the tensor memory's lane
    const int rows_here = min(BQ, p.T - tile_t * BQ);
    const int part_tile = p.gated ? tile_n >> 1 : tile_n;
    const bool channel_there = part_tile * kTileRows + row < p.N;
    const int channel = (p.gated && (tile_n & 1) ? p.N : 0) + part_tile * kTileRows + row;
    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(lane_group * 32) << 16);
    const bool epilogue = warp >= 2;
    // CTA r of the cluster ends rows r * share .. of the tile (share: all of them without a cluster)
    const int share = (rows_here + splits - 1) / splits, first = split * share, n_mine = min(share, rows_here - first);
    bool ok = false;
    float w_scale = 0.f;
    constexpr int kBytes = EPI == kStoreBF16 ? 2 : 4;
    char* out = static_cast<char*>(p.out) + (static_cast<size_t>(tile_t * BQ) * p.ldo + channel) * kBytes;
    const size_t out_step = static_cast<size_t>(p.ldo) * kBytes;
    // Rows t .. t + kGroup - 1 (n of them there) of this thread's channel. All loads stand before the first store: nothing tells the compiler that they do
    // not overlap, and one load behind each store costs a row 100 cycles (128 rows one by one: 7 us).
    constexpr int kGroup = 8;
    const int group_first = Cfg::kGroups == 1 ? 0 : ((warp - 2) >> 2) * kGroup;
    auto load_old = [&](int t, int n, float* old) {
#pragma unroll
        for (int j = 0; j < kGroup; ++j) old[j] = j < n ? __ldcg(reinterpret_cast<const float*>(out + (t + j) * out_step)) : 0.f;
    };
    auto put = [&](int t, int n, const int* sum, const float* old) {
        float v[kGroup];
#pragma unroll
        for (int j = 0; j < kGroup; ++j) v[j] = scaled(sum[j], row_scales[min(t + j, BQ - 1)], w_scale);
#pragma unroll
        for (int j = 0; j < kGroup; ++j) {
            if (j >= n) continue;
            if (EPI == kStoreBF16) *reinterpret_cast<__nv_bfloat16*>(out + (t + j) * out_step) = __float2bfloat16_rn(v[j]);
            else *reinterpret_cast<float*>(out + (t + j) * out_step) = EPI == kAddF32 ? __fadd_rn(old[j], v[j]) : v[j];
        }
    };
    float old[kGroup];
    const bool adds = EPI == kAddF32 && epilogue && channel_there;
    if (epilogue) {
        pdl_wait();
        if (channel_there) w_scale = __ldcg(p.w_scales + channel);
        for (int t = threadIdx.x - 64; t < rows_here; t += 128 * Cfg::kGroups) row_scales[t] = __ldcg(p.a_scales + tile_t * BQ + t);
        if (adds) load_old(first + group_first, n_mine - group_first, old);          // while the products run
        ok = bar_wait(smem_addr(&bars[16]), 0, gave_up, p.status, kErrEpilogue);
        fence_after();
        asm volatile("bar.sync 1, %0;" ::"n"(128 * Cfg::kGroups) : "memory");
        if (threadIdx.x == 64) timeline_record(kTlInt8ProductFew, 4);
    }
    const bool whole = epilogue && __all_sync(0xffffffffu, ok);
    if constexpr (!CLUSTER) {
        if (whole) {
#pragma unroll 1
            for (int c = group_first; c < rows_here; c += Cfg::kGroups * kGroup) {
                uint32_t r[kGroup];
                tmem_load8(lane_addr + c, r);
                if (adds && c > group_first) load_old(c, rows_here - c, old);
                tmem_load_wait();
                if (channel_there) put(c, rows_here - c, reinterpret_cast<const int*>(r), old);
            }
        }
    } else {
        cluster_wait();                           // every CTA of the cluster has begun: its shared memory may be written
        if (epilogue) {
#pragma unroll 1
            for (int c = group_first; c < rows_here; c += Cfg::kGroups * kGroup) {
                uint32_t r[kGroup];
                if (whole) {
                    tmem_load8(lane_addr + c, r);
                    tmem_load_wait();
                }
                int owner = c / share, place = c - owner * share;
                uint32_t to = map_to(smem_addr(meet + (split * share) * kTileRows + row), static_cast<uint32_t>(owner));
#pragma unroll
                for (int j = 0; j < kGroup; ++j) {
                    if (c + j < rows_here) {
                        store_cluster(to + static_cast<uint32_t>(place * kTileRows * 4), whole ? r[j] : 0u);
                        if (++place == share) {
                            place = 0;
                            ++owner;
                            to = map_to(smem_addr(meet + (split * share) * kTileRows + row), static_cast<uint32_t>(min(owner, splits - 1)));
                        }
                    }
                }
            }
        }
        __syncwarp();
        cluster_sync();                           // everyone's sums have arrived; nobody's memory is written from here on
        if (threadIdx.x == 64) timeline_record(kTlInt8ProductFew, 7);
        if (epilogue && channel_there) {
#pragma unroll 1
            for (int i = group_first; i < n_mine; i += Cfg::kGroups * kGroup) {
                int sum[kGroup];
#pragma unroll
                for (int j = 0; j < kGroup; ++j) sum[j] = 0;
                if (adds && i > group_first) load_old(first + i, n_mine - i, old);
#pragma unroll 1
                for (int s = 0; s < splits; ++s) {
                    const int* from = meet + (s * share + i) * kTileRows + row;
#pragma unroll
                    for (int j = 0; j < kGroup; ++j)
                        if (i + j < n_mine) sum[j] += from[j * kTileRows];
                }
                put(first + i, n_mine - i, sum, old);
            }
        }
        if (threadIdx.x == 64) timeline_record(kTlInt8ProductFew, 5);
    }
    fence_before();
    __syncthreads();
    if (threadIdx.x == 0) timeline_record(kTlInt8ProductFew, 6);
    if (warp == 1) {
        fence_after();
        tmem_free<false>(tmem, Cfg::kTmemCols);
    }
}

// ------------------------------------------------------------------------------------------ many rows
struct ManyParams {
    const float* a_scales;
    const float* w_scales;
    const float* bias;       // gated: [2 N] or null
    void* out;
    long long ldo;
    int plain_stores;        // the output's rows do not start on or do not end with whole 16 bytes: no TMA
    int T, N;                // N: output channels
    int total_kb;
    int tiles_t, tiles_n;    // of 256 rows, of 256 channels (gated: 128 gates and their ups)
    int group_t;             // tiles of rows that are walked together
    int act;
    float limit;
    int* status;
};

// Measured on B200: 8192 x 14336 -> 4096 305 us (3,160 TOP/s), 4096 x 4096 -> 4096 48 to 52 (2,650 to 2,850: 256 tiles are 3.46 rounds of 74 pairs), 2048 x 2048 -> 2 x
// 8192 with its activation 49. A CTA takes in 32 KB and its tensor core works 512 cycles for every 128 values of K: both are near their limits.
constexpr int kManyThreads = 64 + 2 * 128;      // producer, MMA, two epilogue groups of four warps

constexpr int kTileN = 256;                                                  // channels of a tile: 128 in each CTA's shared memory
constexpr int kManyStageBytes = 2 * kTileBytes;
constexpr int kManyStages = 6;
constexpr int kStagingBytes = kTileRows * 128;                               // 128 rows x 128 bytes, one to a group
constexpr int kManySmem = kManyStages * kManyStageBytes + 2 * kStagingBytes + 256 + 4 * kTileN + 1024;      // barriers; the channels' scales of a tile
static_assert(kManySmem <= 232448, "the pipeline does not fit into an SM's shared memory");
static_assert(kTileN / 32 * kStagingBytes <= kManyStages * kManyStageBytes, "the last tile's chunks do not fit into the stages");

// act(gate) * up of 32 channels, packed to bfloat16; n0: the first one's number.
__device__ __forceinline__ void gated32(uint32_t* r, uint32_t* u, const float* gate_scales, const float* up_scales, float row_scale, int n0, const ManyParams& p,
                                        uint32_t* packed) {
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        r[j] = __float_as_uint(scaled(static_cast<int>(r[j]), row_scale, gate_scales[j]));
        u[j] = __float_as_uint(scaled(static_cast<int>(u[j]), row_scale, up_scales[j]));
    }
    if (p.bias != nullptr) {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            const float bg = n0 + j < p.N ? p.bias[n0 + j] : 0.f, bu = n0 + j < p.N ? p.bias[p.N + n0 + j] : 0.f;
            r[j] = __float_as_uint(__fadd_rn(__uint_as_float(r[j]), bg));
            u[j] = __float_as_uint(__fadd_rn(__uint_as_float(u[j]), bu));
        }
    }
    with_activation(p.act, [&](auto act) {
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
            const __nv_bfloat162 hb = __floats2bfloat162_rn(gated_value_bf16<decltype(act)::value>(__uint_as_float(r[j]), __uint_as_float(u[j]), p.limit),
                                                            gated_value_bf16<decltype(act)::value>(__uint_as_float(r[j + 1]), __uint_as_float(u[j + 1]), p.limit));
            packed[j / 2] = *reinterpret_cast<const uint32_t*>(&hb);
        }
    });
}

template <int EPI>
__global__ void __launch_bounds__(kManyThreads, 1)
int8_many_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_o,
                 const ManyParams p) {
    constexpr int kStages = kManyStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* staging = smem + kStages * kManyStageBytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(staging + 2 * kStagingBytes);
    // [0, S) full, [S, 2S) empty, [2S, 2S + 2) sums complete, [2S + 2, 2S + 4) sums read
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 4);
    volatile int* gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* decided = gave_up + 1;
    float* scales = reinterpret_cast<float*>(staging + 2 * kStagingBytes + 256);      // [256]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int worker = blockIdx.x / 2, n_workers = gridDim.x / 2;
    const int n_tiles = p.tiles_t * p.tiles_n;
    // Tiles are walked in groups of group_t tiles of rows, through all channels.
    auto tile_of = [&](int i, int& tile_t, int& tile_n) {
        const int per_group = p.group_t * p.tiles_n, g = i / per_group, in = i - g * per_group;
        const int here = min(p.group_t, p.tiles_t - g * p.group_t);
        tile_t = g * p.group_t + in % here;
        tile_n = in / here;
    };

    if (threadIdx.x == 0) {
        timeline_record(kTlInt8ProductMany, 0);
        for (int s = 0; s < kStages; ++s) {
            bar_init(smem_addr(&bars[s]), 1);
            bar_init(smem_addr(&bars[kStages + s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            bar_init(smem_addr(&bars[2 * kStages + b]), 1);
            bar_init(smem_addr(&bars[2 * kStages + 2 + b]), 2 * (kManyThreads - 64));
        }
        *gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_allocate<true>(smem_addr(tmem_slot), 2 * kTileN);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
    cluster_sync();          // both CTAs' barriers exist before either signals the other's
    pdl_wait();
    if (threadIdx.x == 0) timeline_record(kTlInt8ProductMany, 1);
    auto leader_bar = [&](int i) { return map_to(smem_addr(&bars[i]), 0u); };

    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            bool ok = true;
            for (int i = worker; i < n_tiles && ok; i += n_workers) {
                int tile_t, tile_n;
                tile_of(i, tile_t, tile_n);
                const int t0 = tile_t * 256 + static_cast<int>(rank) * kTileRows;
                const int w0 = (2 * tile_n + static_cast<int>(rank)) * p.total_kb * kTileRows;      // this CTA's tile of the channels
                for (int kb = 0; kb < p.total_kb; ++kb, ++it) {
                    const int s = it % kStages;
                    if (!bar_wait(smem_addr(&bars[kStages + s]), ((it / kStages) & 1) ^ 1, gave_up, p.status, kErrProducer)) { ok = false; break; }
                    const uint32_t stage = smem_addr(smem + s * kManyStageBytes), full = leader_bar(s);
                    if (rank == 0) bar_expect(smem_addr(&bars[s]), 2 * kManyStageBytes);
                    load_tile_pair(stage, &map_a, kb * kRowBytes, t0, full);
                    load_tile_pair(stage + kTileBytes, &map_w, 0, w0 + kb * kTileRows, full);
                }
            }
            if (*gave_up && rank == 0) {
                for (int i = max(0, it - kStages); i < it; ++i) {
                    const unsigned long long t0 = clock64();
                    while (!bar_try<false>(smem_addr(&bars[i % kStages]), (i / kStages) & 1))
                        if (clock64() - t0 > kWaitCycles) { atomicCAS(p.status, 0, kErrDrain); break; }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {      // a pair's products are issued by its first CTA
            constexpr uint32_t idesc = int8_idesc(256, kTileN);
            int it = 0, n = 0;
            bool ok = true;
            for (int i = worker; i < n_tiles && ok; i += n_workers, ++n) {
                const int buf = n & 1;
                if (!bar_wait<true>(smem_addr(&bars[2 * kStages + 2 + buf]), ((n >> 1) & 1) ^ 1, gave_up, p.status, kErrMma)) break;
                fence_after();
                const uint32_t d = tmem + buf * kTileN;
                for (int kb = 0; kb < p.total_kb; ++kb, ++it) {
                    const int s = it % kStages;
                    if (!bar_wait(smem_addr(&bars[s]), (it / kStages) & 1, gave_up, p.status, kErrMma)) { ok = false; break; }
                    fence_after();
                    if (it == 0) timeline_record(kTlInt8ProductMany, 2);
                    const uint32_t at = smem_addr(smem + s * kManyStageBytes);
                    const uint64_t a = tile_desc(at), w = tile_desc(at + kTileBytes);
#pragma unroll
                    for (int k = 0; k < kRowBytes / 32; ++k) mma_i8<true>(d, a + 2 * k, w + 2 * k, idesc, (kb > 0 || k > 0) ? 1u : 0u);
                    mma_commit_pair(smem_addr(&bars[kStages + s]));
                }
                if (ok) mma_commit_pair(smem_addr(&bars[2 * kStages + buf]));
            }
            timeline_record(kTlInt8ProductMany, 3);
        }
    } else {
        // Group 0 (warps 2..5) takes the even chunks of a tile's columns, group 1 the odd ones; each has a staging buffer, a
        // named barrier and a thread that issues its stores. A thread holds one row of the tile.
        const int group = (warp - 2) >> 2, lane_group = warp & 3;
        const int row = lane_group * 32 + lane;
        const int mine = static_cast<int>(threadIdx.x) - 64;
        const bool leader = (mine & 127) == 0;
        auto group_sync = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory"); };
        auto both_sync = [&]() { asm volatile("bar.sync 3, 256;" ::: "memory"); };
        auto sums_read = [&](int buf) {
            fence_before();
            if (rank == 0) bar_arrive(smem_addr(&bars[2 * kStages + 2 + buf]));
            else bar_arrive_remote(leader_bar(2 * kStages + 2 + buf));
        };
        // kAddLanesF32: what is added to is read by the lanes, side by side in a row, 32 rows of a chunk at once and a chunk ahead of its use. (Additions in L2, atomicAdd,
        // take 49 us for 4000 x 2000 -> 4097 and this 61; but they count values below 2^-126 as zeros, which neither the TMA form nor the kernel of few rows does.
        // Asked for into L2 a tile ahead 60.)
        constexpr bool kLanes = EPI == kAddLanesF32;
        float old[kLanes ? 32 : 1];
        auto load_old = [&](float* dst, int tile_t, int col) {
            const int first = tile_t * 256 + static_cast<int>(rank) * kTileRows + lane_group * 32, rows = p.T - first;
            const float* o = static_cast<const float*>(p.out) + static_cast<size_t>(first) * p.ldo + col + lane;
#pragma unroll
            for (int j = 0; j < (kLanes ? 32 : 0); ++j) dst[j] = col + lane < p.N && j < rows ? __ldcg(o + j * p.ldo) : 0.f;
        };
        int n = 0;
        for (int i = worker; i < n_tiles; i += n_workers, ++n) {
            int tile_t, tile_n;
            tile_of(i, tile_t, tile_n);
            const int t = tile_t * 256 + static_cast<int>(rank) * kTileRows + row;
            const int buf = n & 1;
            const float row_scale = t < p.T ? __ldcg(p.a_scales + t) : 0.f;
            // the tile's channels: column c of the sums is channel n0 + c (gated: columns 128 .. are the ups)
            const int n0 = EPI == kGatedBF16 ? tile_n * kTileRows : tile_n * kTileN;
            const bool up = EPI == kGatedBF16 && mine >= kTileRows;
            const int ch = n0 + (up ? mine - kTileRows : mine);
            const float mine_scale = ch < p.N ? __ldcg(p.w_scales + (up ? p.N : 0) + ch) : 0.f;
            if (kLanes) load_old(old, tile_t, n0 + group * 32);
            bar_wait(smem_addr(&bars[2 * kStages + buf]), (n >> 1) & 1, gave_up, p.status, kErrEpilogue);
            both_sync();                               // nobody reads the last tile's scales any more
            scales[mine] = mine_scale;
            if (mine == 0) *decided = *gave_up == 0;
            both_sync();                               // the scales are there, and one decision for all
            if (!*decided) break;
            fence_after();
            if (n == 0 && mine == 0) timeline_record(kTlInt8ProductMany, 4);
            const uint32_t d = tmem + buf * kTileN + (static_cast<uint32_t>(lane_group * 32) << 16);
            constexpr int kCols = EPI == kStoreBF16 || EPI == kGatedBF16 ? 64 : 32;      // output columns to a chunk: 128 bytes
            constexpr int kChunks = EPI == kGatedBF16 ? 2 : kTileN / kCols;
            // The pipeline's stages are free once the sums of this CTA's last tile are complete: each chunk then has a place of its own there and waits for no
            // earlier store.
            const bool free_stages = i + n_workers >= n_tiles;
            for (int c = group; c < kChunks; c += 2) {
                uint8_t* stg = free_stages ? smem + c * kStagingBytes : staging + group * kStagingBytes;
                if (!free_stages) {
                    if (leader) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // the last store has read the staging buffer
                    group_sync();
                }
                const bool last = c + 2 >= kChunks;
                const int col = n0 + c * kCols, out_row = tile_t * 256 + static_cast<int>(rank) * kTileRows;
#pragma unroll
                for (int half = 0; half < kCols / 32; ++half) {
                    const int at = c * kCols + half * 32;
                    uint32_t r[32];
                    tmem_load16(d + at, r);
                    tmem_load16(d + at + 16, r + 16);
                    if constexpr (EPI == kGatedBF16) {
                        uint32_t u[32], packed[16];
                        tmem_load16(d + kTileRows + at, u);
                        tmem_load16(d + kTileRows + at + 16, u + 16);
                        tmem_load_wait();
                        if (last && half == kCols / 32 - 1) sums_read(buf);
                        gated32(r, u, scales + at, scales + kTileRows + at, row_scale, n0 + at, p, packed);
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            *reinterpret_cast<uint4*>(stg + row * 128 + (((half * 4 + q) ^ (row & 7)) * 16)) =
                                make_uint4(packed[4 * q], packed[4 * q + 1], packed[4 * q + 2], packed[4 * q + 3]);
                    } else {
                        tmem_load_wait();
                        if (last && half == kCols / 32 - 1) sums_read(buf);
#pragma unroll
                        for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(scaled(static_cast<int>(r[j]), row_scale, scales[at + j]));
                        if constexpr (EPI == kStoreBF16) {
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                uint32_t packed[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const __nv_bfloat162 vb = __floats2bfloat162_rn(__uint_as_float(r[q * 8 + 2 * e]), __uint_as_float(r[q * 8 + 2 * e + 1]));
                                    packed[e] = *reinterpret_cast<const uint32_t*>(&vb);
                                }
                                *reinterpret_cast<uint4*>(stg + row * 128 + (((half * 4 + q) ^ (row & 7)) * 16)) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
                            }
                        } else {
#pragma unroll
                            for (int q = 0; q < 8; ++q)
                                *reinterpret_cast<uint4*>(stg + row * 128 + ((q ^ (row & 7)) * 16)) = make_uint4(r[4 * q], r[4 * q + 1], r[4 * q + 2], r[4 * q + 3]);
                        }
                    }
                }
                if constexpr (kLanes) {
                    float next[32];
                    if (c + 2 < kChunks) load_old(next, tile_t, col + 2 * kCols);
                    group_sync();
                    const int rows = min(32, p.T - (out_row + lane_group * 32));
                    float* o = static_cast<float*>(p.out) + static_cast<size_t>(out_row + lane_group * 32) * p.ldo + col + lane;
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const float v = *reinterpret_cast<const float*>(stg + (lane_group * 32 + j) * 128 + (((lane >> 2) ^ (j & 7)) * 16) + (lane & 3) * 4);
                        if (col + lane < p.N && j < rows) o[j * p.ldo] = __fadd_rn(old[j], v);
                    }
#pragma unroll
                    for (int j = 0; j < 32; ++j) old[j] = next[j];
                } else if (!p.plain_stores) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    group_sync();
                    if (leader) {
                        if (EPI == kAddF32) add_tile(&map_o, smem_addr(stg), col, out_row);
                        else store_tile(&map_o, smem_addr(stg), col, out_row);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                } else {
                    // A warp stores the rows of its quarter of the tile, the lanes side by side, eight rows at a time.
                    group_sync();
#pragma unroll 1
                    for (int r0 = lane_group * 32; r0 < lane_group * 32 + 32 && out_row + r0 < p.T; r0 += 8) {
#pragma unroll
                        for (int part = 0; part < kCols / 32; ++part) {
                            const int cc = part * 32 + lane;
                            const bool there = col + cc < p.N;
                            const size_t to = static_cast<size_t>(out_row + r0) * p.ldo + col + cc;
                            if constexpr (kCols == 64) {
                                __nv_bfloat16* o = static_cast<__nv_bfloat16*>(p.out) + to;
#pragma unroll
                                for (int j = 0; j < 8; ++j)
                                    if (there && out_row + r0 + j < p.T)
                                        o[j * p.ldo] = *reinterpret_cast<const __nv_bfloat16*>(stg + (r0 + j) * 128 + (((cc >> 3) ^ ((r0 + j) & 7)) * 16) + (cc & 7) * 2);
                            } else {
                                float* o = static_cast<float*>(p.out) + to;
                                float v[8];
#pragma unroll
                                for (int j = 0; j < 8; ++j)
                                    v[j] = *reinterpret_cast<const float*>(stg + (r0 + j) * 128 + (((cc >> 2) ^ ((r0 + j) & 7)) * 16) + (cc & 3) * 4);
#pragma unroll
                                for (int j = 0; j < 8; ++j)
                                    if (there && out_row + r0 + j < p.T) o[j * p.ldo] = v[j];
                            }
                        }
                    }
                }
            }
        }
        if (leader) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        if (mine == 0) timeline_record(kTlInt8ProductMany, 5);
        fence_before();
    }
    __syncthreads();
    if (threadIdx.x == 0) timeline_record(kTlInt8ProductMany, 6);
    cluster_sync();          // neither CTA leaves while the other may still signal it
    if (warp == 1) {
        fence_after();
        tmem_free<true>(tmem, 2 * kTileN);
    }
}

// ------------------------------------------------------------------------------------------ host side
int encode(CUtensorMap* map, CUtensorMapDataType type, const void* base, unsigned long long rows, unsigned long long cols, unsigned long long row_bytes,
           int box_rows, int box_cols, CUtensorMapSwizzle swizzle, CUtensorMapL2promotion promotion) {
    EncodeTiledFn fn = tensor_map_encoder();
    if (!fn) { set_error("int8_product: cuTensorMapEncodeTiled is not available from the driver"); return 1; }
    cuuint64_t dims[2] = {cols, rows};
    cuuint64_t strides[1] = {row_bytes};
    cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
    cuuint32_t elem[2] = {1, 1};
    const CUresult r = fn(map, type, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, promotion,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) { set_error("int8_product: cuTensorMapEncodeTiled failed with code %d", static_cast<int>(r)); return 1; }
    return 0;
}

int encode_rows(CUtensorMap* map, const void* a, int T, int width, int box_rows) {
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, a, T, width, width, box_rows, kRowBytes, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}

template <int BQ, int EPI, bool CLUSTER>
int launch_few(const CUtensorMap& map_a, const FewParams& p, dim3 grid, cudaStream_t st) {
    using Cfg = FewConfig<BQ>;
    static SharedLimit limit;
    constexpr int kMost = 232448;
    const cudaError_t le = limit.allow(reinterpret_cast<const void*>(int8_few_kernel<BQ, EPI, CLUSTER>), kMost);
    if (le != cudaSuccess) { set_error("int8_product: cannot reserve %d bytes of shared memory: %s", kMost, cudaGetErrorString(le)); return 1; }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(Cfg::kThreads);
    cfg.dynamicSmemBytes = Cfg::smem(p.stages, min(BQ, p.T), p.splits);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = g_pdl_enabled ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = p.splits;
    cfg.attrs = attr;
    cfg.numAttrs = CLUSTER ? 2 : 1;
    counted(cudaLaunchKernelEx(&cfg, int8_few_kernel<BQ, EPI, CLUSTER>, map_a, p));
    return check_launch("int8_product");
}

// Stages of the pipeline: `asked`, or as many as let two CTAs share an SM (twice the copies under way, and the CTAs of the next product fetch their first weights
// while this one ends); no more than there are steps.
template <int BQ>
int few_stages(int asked, int steps, int rows, int splits) {
    using Cfg = FewConfig<BQ>;
    constexpr int kTwoToAnSm = 233472 / 2 - 1024;
    int stages = max(1, min(asked > 0 ? min(asked, 8) : 8, steps));
    while (stages > 1 && Cfg::smem(stages, rows, splits) > (asked > 0 ? 232448 : kTwoToAnSm)) --stages;
    return stages;
}

template <int EPI>
int launch_many(const CUtensorMap& map_a, const CUtensorMap& map_w, const CUtensorMap& map_o, const ManyParams& p, cudaStream_t st) {
    static SharedLimit limit;
    const cudaError_t le = limit.allow(reinterpret_cast<const void*>(int8_many_kernel<EPI>), kManySmem);
    if (le != cudaSuccess) { set_error("int8_product: cannot reserve %d bytes of shared memory: %s", kManySmem, cudaGetErrorString(le)); return 1; }
    const long long tiles = static_cast<long long>(p.tiles_t) * p.tiles_n;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * static_cast<unsigned>(min(tiles, static_cast<long long>(max(1, sm_count() / 2)))));
    cfg.blockDim = dim3(kManyThreads);
    cfg.dynamicSmemBytes = kManySmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = g_pdl_enabled ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    counted(cudaLaunchKernelEx(&cfg, int8_many_kernel<EPI>, map_a, map_w, map_o, p));
    return check_launch("int8_product");
}

int check_operands(const void* a, int T, int width, const void* tiles, int N, const void* status) {
    GI_REQUIRE(T > 0 && N > 0 && width > 0, "int8_product: sizes must be positive (rows=%d, channels=%d, width=%d)", T, N, width);
    GI_REQUIRE(width % 16 == 0 && width <= 131056, "int8_product: a width of %d (multiples of 16, at most 131056: the sums stay within 32 bits)", width);
    GI_REQUIRE(reinterpret_cast<uintptr_t>(a) % 16 == 0 && reinterpret_cast<uintptr_t>(tiles) % 128 == 0, "int8_product: rows must be 16-byte aligned, weights 128-byte");
    GI_REQUIRE(status != nullptr, "int8_product: a status word is required");
    return 0;
}

int int8_few_impl(const void* a, const float* a_scales, int T, int width, const void* tiles, const float* w_scales, int N, int gated, void* out,
                  int out_dtype, long long ldo, int accumulate, int bq, int splits, int stages, int w_constant, void* status, void* stream) {
    if (T == 0) return 0;
    if (int bad = check_operands(a, T, width, tiles, N, status)) return bad;
    GI_REQUIRE(out_dtype == kF32 || out_dtype == kBF16, "int8_product: unsupported dtype code %d", out_dtype);
    GI_REQUIRE(!(accumulate && out_dtype != kF32), "int8_product: accumulation needs a 32-bit output");
    GI_REQUIRE(T == 1 || ldo >= (gated ? 2ll : 1ll) * N, "int8_product: rows of the output overlap");
    GI_REQUIRE(bq == 8 || bq == 32 || bq == 64 || bq == 128, "int8_product: tiles of %d rows (8, 32, 64 or 128)", bq);
    GI_REQUIRE(splits >= 1 && splits <= (bq == 128 ? 1 : 8), "int8_product: %d ranges of K with tiles of %d rows (1 to 8: one cluster; one with 128)", splits, bq);
    FewParams p{};
    p.tiles = static_cast<const uint8_t*>(tiles);
    p.a_scales = a_scales;
    p.w_scales = w_scales;
    p.out = out;
    p.ldo = ldo;
    p.T = T;
    p.N = N;
    p.gated = gated;
    p.w_constant = w_constant;
    p.total_kb = (width + kRowBytes - 1) / kRowBytes;
    p.kb_per_split = (p.total_kb + splits - 1) / splits;
    p.splits = (p.total_kb + p.kb_per_split - 1) / p.kb_per_split;      // (no range is empty)
    p.status = static_cast<int*>(status);
    const int n_tiles = (N + kTileRows - 1) / kTileRows * (gated ? 2 : 1);
    const dim3 grid(n_tiles, (T + bq - 1) / bq, p.splits);
    GI_REQUIRE(grid.y <= 65535, "int8_product: too many rows for tiles of %d", bq);
    CUtensorMap map_a;
    if (int bad = encode_rows(&map_a, a, T, width, bq)) return bad;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto go = [&](auto tile) {
        constexpr int BQ = decltype(tile)::value;
        p.stages = few_stages<BQ>(stages, (p.kb_per_split + FewConfig<BQ>::kKb - 1) / FewConfig<BQ>::kKb, min(BQ, T), p.splits);
        if constexpr (BQ <= 64) {
            if (p.splits > 1) {
                if (out_dtype == kBF16) return launch_few<BQ, kStoreBF16, true>(map_a, p, grid, st);
                return accumulate ? launch_few<BQ, kAddF32, true>(map_a, p, grid, st) : launch_few<BQ, kStoreF32, true>(map_a, p, grid, st);
            }
        }
        if (out_dtype == kBF16) return launch_few<BQ, kStoreBF16, false>(map_a, p, grid, st);
        return accumulate ? launch_few<BQ, kAddF32, false>(map_a, p, grid, st) : launch_few<BQ, kStoreF32, false>(map_a, p, grid, st);
    };
    switch (bq) {
        case 8: return go(std::integral_constant<int, 8>());
        case 32: return go(std::integral_constant<int, 32>());
        case 64: return go(std::integral_constant<int, 64>());
        default: return go(std::integral_constant<int, 128>());
    }
}

int int8_many_impl(const void* a, const float* a_scales, int T, int width, const void* tiles, const float* w_scales, int N, int gated, int act, float limit,
                   const float* bias, void* out, int out_dtype, long long ldo, int accumulate, int group_t, void* status, void* stream) {
    if (T == 0) return 0;
    if (int bad = check_operands(a, T, width, tiles, N, status)) return bad;
    GI_REQUIRE(out_dtype == kF32 || out_dtype == kBF16, "int8_product: unsupported dtype code %d", out_dtype);
    GI_REQUIRE(!(accumulate && out_dtype != kF32), "int8_product: accumulation needs a 32-bit output");
    GI_REQUIRE(T == 1 || ldo >= N, "int8_product: rows of the output overlap");
    GI_REQUIRE(!gated || out_dtype == kBF16, "int8_product: a gated product has a bfloat16 output");
    GI_REQUIRE(act >= 0 && act < kActCount, "int8_product: unknown activation %d", act);
    GI_REQUIRE(!(gated && act == kActCappedSwish && limit < 0.f), "int8_product: a bound of %g (not below zero)", limit);
    GI_REQUIRE(group_t >= 1, "int8_product: groups of %d tiles", group_t);
    ManyParams p{};
    p.a_scales = a_scales;
    p.w_scales = w_scales;
    p.bias = bias;
    p.out = out;
    p.ldo = ldo;
    p.T = T;
    p.N = N;
    p.total_kb = (width + kRowBytes - 1) / kRowBytes;
    p.tiles_t = (T + 255) / 256;
    p.tiles_n = (N + (gated ? kTileRows : kTileN) - 1) / (gated ? kTileRows : kTileN);
    p.group_t = min(group_t, p.tiles_t);
    p.act = act;
    p.limit = limit;
    p.status = static_cast<int*>(status);
    GI_REQUIRE(static_cast<long long>(p.tiles_t) * p.tiles_n < (1ll << 30), "int8_product: too many tiles");
    const int elt = out_dtype == kBF16 ? 2 : 4;
    // (a TMA store writes whole 16 bytes: it would reach into what lies behind a row's last channel. Behind a gated row there is scratch.)
    p.plain_stores = ldo * elt % 16 != 0 || reinterpret_cast<uintptr_t>(out) % 16 != 0 || (!gated && static_cast<long long>(N) * elt % 16 != 0);
    const long long weight_rows = static_cast<long long>((N + kTileRows - 1) / kTileRows) * (gated ? 2 : 1) * p.total_kb * kTileRows;
    GI_REQUIRE(weight_rows < (1ll << 31), "int8_product: the weights are too large");
    CUtensorMap map_a, map_w, map_o{};
    if (int bad = encode_rows(&map_a, a, T, width, kTileRows)) return bad;
    if (int bad = encode(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, tiles, weight_rows, kRowBytes, kRowBytes, kTileRows, kRowBytes, CU_TENSOR_MAP_SWIZZLE_NONE,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B)) return bad;
    if (!p.plain_stores) {
        if (int bad = encode(&map_o, elt == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, out, T, N, ldo * elt, kTileRows, 128 / elt,
                             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE)) return bad;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (gated) return launch_many<kGatedBF16>(map_a, map_w, map_o, p, st);
    if (elt == 2) return launch_many<kStoreBF16>(map_a, map_w, map_o, p, st);
    if (accumulate && p.plain_stores) return launch_many<kAddLanesF32>(map_a, map_w, map_o, p, st);
    return accumulate ? launch_many<kAddF32>(map_a, map_w, map_o, p, st) : launch_many<kStoreF32>(map_a, map_w, map_o, p, st);
}

}  // namespace
}  // namespace gi
GI_TIMELINE_SETTER(gi_timeline_set_int8_product)

// Few rows: tiles of bq rows of a [T, width], K in `splits` ranges (one cluster), `stages` stages of the pipeline (0: chosen). `gated`: the weights are a gated
// pair of N channels each, out [T, 2 N] = [gate; up]. out[t, n] at t * ldo + n. w_constant: no launch before this one that may still be running writes the
// tiles, so that the first ones may be asked for before the wait for them.
extern "C" int gi_int8_product_few(const void* a, const float* a_scales, int T, int width, const void* tiles, const float* w_scales, int N, int gated,
                                   void* out, int out_dtype, long long ldo, int accumulate, int bq, int splits, int stages, int w_constant, void* status,
                                   void* stream) {
    return gi::dispatch(gi::int8_few_impl, a, a_scales, T, width, tiles, w_scales, N, gated, out, out_dtype, ldo, accumulate, bq, splits, stages, w_constant,
                        status, stream);
}

// Many rows: tiles of 256 rows x 256 channels, `group_t` tiles of rows walked together. `gated`: out [T, N] = act(gate) * up, bfloat16; `bias` [2 N] or null.
extern "C" int gi_int8_product_many(const void* a, const float* a_scales, int T, int width, const void* tiles, const float* w_scales, int N, int gated,
                                    int act, float limit, const float* bias, void* out, int out_dtype, long long ldo, int accumulate, int group_t,
                                    void* status, void* stream) {
    return gi::dispatch(gi::int8_many_impl, a, a_scales, T, width, tiles, w_scales, N, gated, act, limit, bias, out, out_dtype, ldo, accumulate, group_t,
                        status, stream);
}

extern "C" int gi_rows_int8(int kind, const void* x, int x_dtype, long long ldx, const void* add, int add_dtype, const float* weight, float eps, int act,
                            float limit, void* q, int width, float* scales, int T, int D, int w_constant, void* stream);

// act(gate) * up of a gated pair of N channels each, in 8 bits: q [T, out_width] and scales [T]. Few rows (bq > 0: see gi_int8_product_few) leave [gate; up] in `work`
// as 32-bit [T, 2 N] for the activation with the rows; many (bq 0, `splits` the tiles of rows walked together) act(gate) * up as bfloat16, rows of whole 16 bytes.
extern "C" int gi_int8_gated(const void* a, const float* a_scales, int T, int width, const void* tiles, const float* w_scales, int N, int act, float limit,
                             const float* bias, void* work, void* q, int out_width, float* scales, int bq, int splits, int stages, int w_constant, void* status,
                             void* stream) {
    if (bq > 0) {
        const int code = gi_int8_product_few(a, a_scales, T, width, tiles, w_scales, N, 1, work, gi::kF32, 2ll * N, 0, bq, splits, stages, w_constant, status, stream);
        return code ? code : gi_rows_int8(2, work, gi::kF32, 2ll * N, nullptr, 0, bias, 0.f, act, limit, q, out_width, scales, T, N, 0, stream);
    }
    const long long row = (N + 7ll) / 8 * 8;
    const int code = gi_int8_product_many(a, a_scales, T, width, tiles, w_scales, N, 1, act, limit, bias, work, gi::kBF16, row, 0, splits, status, stream);
    return code ? code : gi_rows_int8(0, work, gi::kBF16, row, nullptr, 0, nullptr, 0.f, 0, 0.f, q, out_width, scales, T, N, 0, stream);
}
