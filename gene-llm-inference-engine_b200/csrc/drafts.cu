// Drafted tokens against the target's distribution, and the drafter's own probabilities.
//
// Request r brings d_r drafted tokens and d_r + 1 rows of the target's logits. With temperature T > 0 row j's distribution is
//   p_i = e_i * (float)(1 / sum e), e_i = exp((l_i - max l) / T), the sum in 64 bits  (the numbers that the sampler draws from).
// Draft x_j is kept while u_j * q_j(x_j) < p_j(x_j); the first refused one is replaced by a draw from max(p_j - q_j, 0), and with
// all of them kept one more token is drawn from the last row's p: the tokens are then distributed as if each had been drawn from
// the target alone. T <= 0: a draft is kept while it is the row's argmax, which is also what replaces it. The draw takes the first index i of
// weight w_i > 0 with w_0 + .. + w_i > v * sum(w); the random numbers u and v come from the caller.
//
// Two launches: one cluster of CTAs per row finds max and sum (a row is read once and stays in registers), one cluster per request
// finds the stop and draws. The answer is a whole number, so sums run in 64 bits: their order moves a boundary between two tokens by
// 1e-13 of the mass, where 32-bit sums would move all 128,000 of them by 1e-7, a different token in one draw of a hundred.
#include <climits>

#include <cooperative_groups.h>

#include "common.cuh"

namespace gi {

namespace cg = cooperative_groups;

constexpr int kRowThreads = 512, kRowWarps = kRowThreads / 32;
constexpr int kRowCtasMost = 8;           // CTAs of a row's cluster
constexpr int kRowUnitsMost = 10;         // groups of four values that a thread holds: vocabularies of up to 163,840 stay in registers

// (l - max) / T. With y the rounded reciprocal of T, q = l y and one correction by the exact remainder give the rounded
// quotient (P. Markstein, IBM J. Res. Dev. 34, 1990): three multiply-adds instead of the general division. Temperatures whose
// reciprocal could leave the normal range take the division. The dividend is bounded below, where exp gives 0 anyway: an infinite one has no remainder.
struct ByTemperature {
    float t, y;
    bool plain;
    __device__ explicit ByTemperature(float temp) : t(temp), y(1.0f / temp), plain(!(temp > 1e-3f && temp < 1e3f)) {}
    __device__ __forceinline__ float operator()(float a) const {
        if (plain) return a / t;
        a = fmaxf(a, -1e30f);
        const float q = __fmul_rn(a, y);
        return __fmaf_rn(__fmaf_rn(-q, t, a), y, q);
    }
};

__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// A row in groups of four neighbours on a boundary of four elements: the first and the last group may reach beyond the row.
template <typename T> struct Row {
    const T* row;
    int V, off, units, begin, end;         // begin, end: this CTA's groups
    __device__ Row(const T* p, int vocab, int part, int parts) : row(p), V(vocab) {
        off = static_cast<int>((reinterpret_cast<uintptr_t>(p) / sizeof(T)) & 3);
        units = static_cast<int>((static_cast<long long>(V) + off + 3) / 4);
        const int per = ((units + parts - 1) / parts + 31) / 32 * 32;
        begin = min(units, part * per);
        end = min(units, begin + per);
    }
    __device__ __forceinline__ int index(int unit) const { return 4 * unit - off; }
    __device__ __forceinline__ bool whole(int unit) const { return index(unit) >= 0 && index(unit) <= V - 4; }
    // the group's values, `none` beyond the row
    __device__ __forceinline__ void load(int unit, float none, float (&v)[4]) const {
        const int i = index(unit);
        if (whole(unit)) {
            if constexpr (sizeof(T) == 4) {
                const float4 x = *reinterpret_cast<const float4*>(row + i);
                v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
            } else {
                const uint2 x = *reinterpret_cast<const uint2*>(row + i);
                v[0] = __uint_as_float(x.x << 16); v[1] = __uint_as_float(x.x & 0xffff0000u);
                v[2] = __uint_as_float(x.y << 16); v[3] = __uint_as_float(x.y & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = i + e >= 0 && i + e < V ? to_float(row[i + e]) : none;
        }
    }
};

__device__ __forceinline__ double warp_total(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// What a row's pass needs of shared memory: warps' results, and one result of every CTA of the cluster.
struct RowShared {
    float warp_max[kRowWarps];
    int warp_at[kRowWarps];
    double warp_sum[kRowWarps];
    float cta_max[kRowCtasMost];
    int cta_at[kRowCtasMost];
    double cta_sum[kRowCtasMost];
};

// The largest value of the cluster's row (NaN if any value is none); every thread has it.
__device__ __forceinline__ float cluster_max(float mx, RowShared& s, cg::cluster_group& cluster, int part, int parts) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = max_or_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) s.warp_max[warp] = mx;
    __syncthreads();
    cluster.barrier_wait();                // (arrived at when the kernel began)
    if (warp == 0) {
        mx = s.warp_max[lane & (kRowWarps - 1)];
#pragma unroll
        for (int o = kRowWarps / 2; o > 0; o >>= 1) mx = max_or_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        if (lane < parts) *cluster.map_shared_rank(&s.cta_max[part], lane) = mx;
    }
    cluster.sync();
    mx = s.cta_max[0];
    for (int p = 1; p < parts; ++p) mx = max_or_nan(mx, s.cta_max[p]);
    return mx;
}

// The cluster's sum, in the order of the CTAs; every thread has it.
__device__ __forceinline__ double cluster_sum(double v, RowShared& s, cg::cluster_group& cluster, int part, int parts) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = warp_total(v);
    if (lane == 0) s.warp_sum[warp] = v;
    __syncthreads();
    if (warp == 0) {
        v = s.warp_sum[lane & (kRowWarps - 1)];
#pragma unroll
        for (int o = kRowWarps / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane < parts) *cluster.map_shared_rank(&s.cta_sum[part], lane) = v;
    }
    cluster.sync();
    v = s.cta_sum[0];
    for (int p = 1; p < parts; ++p) v += s.cta_sum[p];
    return v;
}

__device__ __forceinline__ void keep_best(float v, int i, float& best, int& at) {
    if (v > best || (v == best && i < at)) { best = v; at = i; }
}

// Index of the largest value of the cluster's row, the lowest among equals (values that are no number are passed over; 0 where there
// is no other).
template <typename Each>
__device__ __forceinline__ int cluster_argmax(const Each& each, RowShared& s, cg::cluster_group& cluster, int part, int parts) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float best = -INFINITY;
    int at = INT_MAX;
    each([&](int i, float v) { keep_best(v, i, best, at); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float v = __shfl_xor_sync(0xffffffffu, best, o);
        const int i = __shfl_xor_sync(0xffffffffu, at, o);
        keep_best(v, i, best, at);
    }
    if (lane == 0) { s.warp_max[warp] = best; s.warp_at[warp] = at; }
    __syncthreads();
    cluster.barrier_wait();                // (arrived at when the kernel began)
    if (threadIdx.x == 0) {
        for (int w = 1; w < kRowWarps; ++w) keep_best(s.warp_max[w], s.warp_at[w], best, at);
        for (int p = 0; p < parts; ++p) {
            *cluster.map_shared_rank(&s.cta_max[part], p) = best;
            *cluster.map_shared_rank(&s.cta_at[part], p) = at;
        }
    }
    cluster.sync();
    best = s.cta_max[0];
    at = s.cta_at[0];
    for (int p = 1; p < parts; ++p) keep_best(s.cta_max[p], s.cta_at[p], best, at);
    return at == INT_MAX ? 0 : at;
}

// Values of a CTA's groups: held in registers (kUnits groups of four a thread) or, kUnits = 0, read again in every pass.
template <typename T, int kUnits> struct Values {
    const Row<T>& r;
    float held[kUnits > 0 ? kUnits : 1][4];
    __device__ explicit Values(const Row<T>& row) : r(row) {
        if constexpr (kUnits > 0) {
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
                const int unit = r.begin + u * kRowThreads + threadIdx.x;
                if (unit < r.end) r.load(unit, -INFINITY, held[u]);
                else held[u][0] = held[u][1] = held[u][2] = held[u][3] = -INFINITY;
            }
        }
    }
    // f(group, values): every group of the thread, in order
    template <typename F> __device__ __forceinline__ void groups(F f) {
        if constexpr (kUnits > 0) {
#pragma unroll
            for (int u = 0; u < kUnits; ++u) f(r.begin + u * kRowThreads + static_cast<int>(threadIdx.x), held[u]);
        } else {
            for (int unit = r.begin + threadIdx.x; unit < r.end; unit += kRowThreads) {
                float v[4];
                r.load(unit, -INFINITY, v);
                f(unit, v);
            }
        }
    }
};

struct RowArgs {
    const void* logits;
    long long stride;                      // values from row to row
    int N, V;
    const float* temperature;              // per row (probabilities) or per request
    float* out;                            // probabilities [N, V]
    // verification
    const int* row_start;
    const int* drafted;
    const int* counts;
    const float* q;
    long long q_request, q_place;          // values between requests and between drafts
    const float* accept;
    const float* draw;
    int* tokens;
    int* accepted;
    float4* work;                          // per row: max, 1 / sum, kept (1) or not (0), argmax (as an integer's bits)
    int R, D;
};

// The request's drafts, or -1 where its rows do not lie in the logits.
__device__ __forceinline__ int drafts_of(const RowArgs& a, int r) {
    const int d = min(max(a.counts[r], 0), a.D), start = a.row_start[r];
    return start < 0 || start > a.N - 1 - d ? -1 : d;
}

// One cluster per row. kProbs: row i's distribution goes to out; else: row j of request r, its max and sum and whether its draft is kept.
template <typename T, int kUnits, bool kProbs>
__global__ void __launch_bounds__(kRowThreads, 2) row_softmax_kernel(RowArgs a) {
    pdl_prologue();
    __shared__ RowShared s;
    cg::cluster_group cluster = cg::this_cluster();
    const int part = cluster.block_rank(), parts = cluster.num_blocks();
    const int which = blockIdx.x / parts;
    int row = which, j = 0, d = 0, r = which;
    if constexpr (!kProbs) {
        r = which / (a.D + 1);
        j = which % (a.D + 1);
        d = drafts_of(a, r);
        if (j > d) return;                 // (the whole cluster)
        row = a.row_start[r] + j;
    }
    cluster.barrier_arrive();              // every CTA of the cluster runs before another writes into its shared memory
    const T* p = static_cast<const T*>(a.logits) + row * a.stride;
    const Row<T> span(p, a.V, part, parts);
    Values<T, kUnits> values(span);
    const float temp = a.temperature[r];
    if (!(temp > 0.f)) {
        const int best = cluster_argmax([&](auto f) {
            values.groups([&](int unit, float (&v)[4]) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (v[e] > -INFINITY || (unit < span.end && span.index(unit) + e >= 0 && span.index(unit) + e < a.V && v[e] == -INFINITY)) f(span.index(unit) + e, v[e]);
            });
        }, s, cluster, part, parts);
        if constexpr (kProbs) {
            float* out = a.out + static_cast<size_t>(row) * a.V;
            for (int unit = span.begin + threadIdx.x; unit < span.end; unit += kRowThreads)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = span.index(unit) + e;
                    if (i >= 0 && i < a.V) out[i] = i == best ? 1.0f : 0.0f;
                }
        } else if (part == 0 && threadIdx.x == 0) {
            const bool kept = j < d && a.drafted[static_cast<size_t>(r) * a.D + j] == best;
            a.work[row] = make_float4(0.f, 0.f, kept ? 1.f : 0.f, __int_as_float(best));
        }
        return;
    }
    float mx = -INFINITY;
    values.groups([&](int, float (&v)[4]) { mx = max_or_nan(max_or_nan(mx, max_or_nan(v[0], v[1])), max_or_nan(v[2], v[3])); });
    mx = cluster_max(mx, s, cluster, part, parts);
    const bool some = mx > -INFINITY && mx < INFINITY;      // else there are no probabilities (a value is none, or infinite, or all are -infinity)
    const ByTemperature by(temp);
    double sum = 0.0;
    if (some)
        values.groups([&](int, float (&v)[4]) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = expf(by(v[e] - mx));
                sum += static_cast<double>(x);
                if constexpr (kProbs) v[e] = x;
            }
        });
    sum = cluster_sum(sum, s, cluster, part, parts);
    const float inv = some ? static_cast<float>(1.0 / sum) : NAN;
    if constexpr (kProbs) {
        float* out = a.out + static_cast<size_t>(row) * a.V;
        const bool wide = (reinterpret_cast<uintptr_t>(out) / 4 & 3) == static_cast<unsigned>(span.off);
        values.groups([&](int unit, float (&v)[4]) {
            if (unit >= span.end) return;
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = __fmul_rn(kUnits > 0 ? v[e] : expf(by(v[e] - mx)), inv);
            const int i = span.index(unit);
            if (wide && span.whole(unit)) {
                *reinterpret_cast<float4*>(out + i) = make_float4(y[0], y[1], y[2], y[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + e >= 0 && i + e < a.V) out[i + e] = y[e];
            }
        });
    } else if (part == 0 && threadIdx.x == 0) {
        bool kept = false;
        if (j < d) {
            const int x = a.drafted[static_cast<size_t>(r) * a.D + j];
            if (x >= 0 && x < a.V) {
                const float q = a.q ? a.q[r * a.q_request + j * a.q_place + x] : 1.0f;
                const float px = __fmul_rn(expf(by(to_float(p[x]) - mx)), inv);
                kept = __fmul_rn(a.accept[static_cast<size_t>(r) * a.D + j], q) < px;
            }
        }
        a.work[row] = make_float4(mx, inv, kept ? 1.f : 0.f, 0.f);
    }
}

// One cluster per request: the stop among its rows, and the token there. A warp owns neighbouring groups; the row and q's row are read once, then
// once more (from the caches) by the one warp in whose piece the draw falls.
template <typename T>
__global__ void __launch_bounds__(kRowThreads, 2) draft_draw_kernel(RowArgs a) {
    pdl_prologue();
    __shared__ RowShared s;
    cg::cluster_group cluster = cg::this_cluster();
    const int part = cluster.block_rank(), parts = cluster.num_blocks();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = blockIdx.x / parts, d = drafts_of(a, r);
    int* tokens = a.tokens + static_cast<size_t>(r) * (a.D + 1);
    if (d < 0) {
        if (part == 0) {
            for (int j = threadIdx.x; j <= a.D; j += kRowThreads) tokens[j] = -1;
            if (threadIdx.x == 0) a.accepted[r] = -1;
        }
        return;
    }
    const int start = a.row_start[r];
    int stop = 0;
    while (stop < d && a.work[start + stop].z != 0.f) ++stop;
    if (part == 0) {
        for (int j = threadIdx.x; j <= a.D; j += kRowThreads)
            if (j != stop) tokens[j] = j < stop ? a.drafted[static_cast<size_t>(r) * a.D + j] : -1;
        if (threadIdx.x == 0) a.accepted[r] = stop;
    }
    const float4 stat = a.work[start + stop];
    const float temp = a.temperature[r];
    if (!(temp > 0.f) || !(stat.y == stat.y)) {             // greedy, or a row without probabilities (the last token, as the sampler has it)
        if (part == 0 && threadIdx.x == 0) tokens[stop] = temp > 0.f ? a.V - 1 : __float_as_int(stat.w);
        return;
    }
    cluster.barrier_arrive();              // every CTA of the cluster runs before another writes into its shared memory
    const Row<T> span(static_cast<const T*>(a.logits) + (start + stop) * a.stride, a.V, part, parts);
    const ByTemperature by(temp);
    const float mx = stat.x, inv = stat.y;
    const bool refused = stop < d;
    const float* q = refused && a.q ? a.q + r * a.q_request + stop * a.q_place : nullptr;
    const int without = refused && !a.q ? a.drafted[static_cast<size_t>(r) * a.D + stop] : -1;
    const bool q_wide = q != nullptr && (reinterpret_cast<uintptr_t>(q) / 4 & 3) == static_cast<unsigned>(span.off);
    bool subtract = refused;

    // what is taken off a group's probabilities
    auto taken = [&](int unit, float (&take)[4]) {
        const int i = span.index(unit);
        take[0] = take[1] = take[2] = take[3] = 0.f;
        if (q_wide && span.whole(unit)) {
            const float4 x = *reinterpret_cast<const float4*>(q + i);
            take[0] = x.x; take[1] = x.y; take[2] = x.z; take[3] = x.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e >= 0 && i + e < a.V) take[e] = q ? q[i + e] : i + e == without ? 1.0f : 0.0f;
        }
    };
    // the four weights of a group, and their sum; beyond the row none
    auto weigh = [&](const float (&take)[4], float (&w)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float pe = __fmul_rn(expf(by(w[e] - mx)), inv);
            w[e] = pe > take[e] ? __fsub_rn(pe, take[e]) : 0.f;      // (a q that is no number takes all)
        }
        return (static_cast<double>(w[0]) + static_cast<double>(w[1])) + (static_cast<double>(w[2]) + static_cast<double>(w[3]));
    };
    const int share = (((span.end - span.begin) + kRowWarps - 1) / kRowWarps + 31) / 32 * 32;
    const int begin = min(span.end, span.begin + warp * share), end = min(span.end, begin + share);
    constexpr int kBatch = 4;                               // turns whose loads are in flight together
    // f(group, weights, sum) of every turn of 32 groups, until it says stop
    auto turns = [&](auto f) {
        for (int base = begin; base < end; base += 32 * kBatch) {
            float w[kBatch][4], take[kBatch][4];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int unit = base + 32 * b + lane;
                w[b][0] = w[b][1] = w[b][2] = w[b][3] = -INFINITY;
                take[b][0] = take[b][1] = take[b][2] = take[b][3] = 0.f;
                if (unit < end) {
                    span.load(unit, -INFINITY, w[b]);
                    if (subtract) taken(unit, take[b]);
                }
            }
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const double t = weigh(take[b], w[b]);
                if (f(base + 32 * b + lane, w[b], t)) return;
            }
        }
    };

    double total;
    for (bool first = true;; first = false) {
        double mine = 0.0;
        turns([&](int, const float (&)[4], double t) { mine += t; return false; });
        mine = warp_total(mine);
        if (lane == 0) s.warp_sum[warp] = mine;
        __syncthreads();
        if (first) cluster.barrier_wait();
        if (warp == 0) {
            double t = 0.0;
            for (int w = 0; w < kRowWarps; ++w) t += s.warp_sum[w];
            if (lane < parts) *cluster.map_shared_rank(&s.cta_sum[part], lane) = t;
        }
        cluster.sync();
        total = 0.0;
        for (int c = 0; c < parts; ++c) total += s.cta_sum[c];
        if (!subtract || total > 0.0) break;
        subtract = false;                                   // nothing is left of p behind q: the draw is from p (the whole cluster takes this turn)
        cluster.sync();                                     // all have read the sums
    }
    const double target = static_cast<double>(a.draw[r]) * total;
    // The CTA, the warp, the group and the value in which the running sum passes the target, every sum taken the same way by all who
    // compare it; where rounding (or a number of 1 and more) lets none, the last that weighs anything.
    double run = 0.0, ahead = 0.0;
    int owner = -1;
    bool found = false;
    for (int c = 0; c < parts && !found; ++c) {
        const double t = s.cta_sum[c];
        if (t > 0.0) { owner = c; ahead = run; found = run + t > target; }
        run += t;
    }
    if (owner != part) return;
    run = ahead;
    owner = -1;
    found = false;
    for (int w = 0; w < kRowWarps && !found; ++w) {
        const double t = s.warp_sum[w];
        if (t > 0.0) { owner = w; ahead = run; found = run + t > target; }
        run += t;
    }
    if (owner != warp) return;
    int pick = a.V - 1;
    turns([&](int unit, const float (&w)[4], double t) {
        double cum = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double m = __shfl_up_sync(0xffffffffu, cum, o);
            if (lane >= o) cum += m;
        }
        const unsigned some = __ballot_sync(0xffffffffu, t > 0.0), over = __ballot_sync(0xffffffffu, t > 0.0 && ahead + cum > target);
        if (some) {
            const int at = over ? __ffs(over) - 1 : 31 - __clz(some);
            double c = ahead + (cum - t);
            int place = 0;
            bool passed = false;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (w[e] > 0.f && !passed) { c += static_cast<double>(w[e]); place = e; passed = c > target; }
            pick = __shfl_sync(0xffffffffu, span.index(unit) + place, at);
        }
        ahead += __shfl_sync(0xffffffffu, cum, 31);
        return over != 0;
    });
    if (lane == 0) tokens[stop] = pick;
}

template <typename... KArgs, typename... Args>
inline void launch_row_clusters(void (*kernel)(KArgs...), long long rows, int parts, cudaStream_t stream, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows * parts));
    cfg.blockDim = dim3(kRowThreads);
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

// CTAs of a row's cluster and groups a thread holds (0: read again in every pass).
struct RowPlan { int parts, units; };
inline RowPlan row_plan(int V) {
    const long long groups = (static_cast<long long>(V) + 6) / 4;         // with an edge on either side
    int parts = 1;
    while (parts < kRowCtasMost && groups > 2LL * kRowThreads * parts) parts *= 2;
    const long long per = ((groups + parts - 1) / parts + 31) / 32 * 32, units = (per + kRowThreads - 1) / kRowThreads;
    return {parts, units <= 2 ? 2 : units <= 4 ? 4 : units <= 8 ? 8 : units <= kRowUnitsMost ? kRowUnitsMost : 0};
}

template <typename T, bool kProbs>
int launch_rows(const RowArgs& a, long long rows, cudaStream_t st, const char* what) {
    const RowPlan plan = row_plan(a.V);
    GI_REQUIRE(rows <= INT_MAX / plan.parts, "%s: %lld rows exceed the grid limit", what, rows);
    switch (plan.units) {
        case 2: launch_row_clusters((row_softmax_kernel<T, 2, kProbs>), rows, plan.parts, st, a); break;
        case 4: launch_row_clusters((row_softmax_kernel<T, 4, kProbs>), rows, plan.parts, st, a); break;
        case 8: launch_row_clusters((row_softmax_kernel<T, 8, kProbs>), rows, plan.parts, st, a); break;
        case kRowUnitsMost: launch_row_clusters((row_softmax_kernel<T, kRowUnitsMost, kProbs>), rows, plan.parts, st, a); break;
        default: launch_row_clusters((row_softmax_kernel<T, 0, kProbs>), rows, plan.parts, st, a); break;
    }
    return check_launch(what);
}

template <typename T>
int launch_draw(const RowArgs& a, cudaStream_t st) {
    launch_row_clusters((draft_draw_kernel<T>), a.R, row_plan(a.V).parts, st, a);
    return check_launch("verify_drafts");
}

}  // namespace gi

using namespace gi;

static int gi_token_probabilities_impl(const void* logits, int dtype, int rows, int V, const float* temperature, float* out, void* stream) {
    if (rows == 0) return 0;
    GI_REQUIRE(rows > 0 && V > 0 && V <= INT_MAX - 8, "token_probabilities: sizes must be positive (rows=%d, V=%d)", rows, V);
    RowArgs a = {};
    a.logits = logits; a.stride = V; a.N = rows; a.V = V; a.temperature = temperature; a.out = out;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == kF32 ? launch_rows<float, true>(a, rows, st, "token_probabilities") : launch_rows<__nv_bfloat16, true>(a, rows, st, "token_probabilities");
}

// logits [N, V]; request r's rows start at row_start[r]; drafted, accept [R, D]; q (or null): q_request / q_place values between
// requests / drafts, V neighbours each; tokens [R, D + 1], accepted [R]; work: 16 bytes a row of logits, aligned to 16.
static int gi_verify_drafts_impl(const void* logits, int dtype, int N, int V, int R, int D, const int* row_start, const int* drafted, const int* counts,
                                 const float* q, long long q_request, long long q_place, const float* temperature, const float* accept, const float* draw,
                                 int* tokens, int* accepted, void* work, void* stream) {
    if (R == 0) return 0;
    GI_REQUIRE(N > 0 && V > 0 && V <= INT_MAX - 8 && R > 0 && D >= 0, "verify_drafts: sizes must be positive (N=%d, V=%d, R=%d, D=%d)", N, V, R, D);
    GI_REQUIRE(reinterpret_cast<uintptr_t>(work) % 16 == 0, "verify_drafts: the workspace must lie on a boundary of 16 bytes");
    RowArgs a = {};
    a.logits = logits; a.stride = V; a.N = N; a.V = V; a.temperature = temperature; a.row_start = row_start; a.drafted = drafted; a.counts = counts;
    a.q = q; a.q_request = q_request; a.q_place = q_place; a.accept = accept; a.draw = draw; a.tokens = tokens; a.accepted = accepted;
    a.work = static_cast<float4*>(work); a.R = R; a.D = D;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const long long rows = static_cast<long long>(R) * (D + 1);
    const int rc = dtype == kF32 ? launch_rows<float, false>(a, rows, st, "verify_drafts") : launch_rows<__nv_bfloat16, false>(a, rows, st, "verify_drafts");
    if (rc) return rc;
    return dtype == kF32 ? launch_draw<float>(a, st) : launch_draw<__nv_bfloat16>(a, st);
}

extern "C" int gi_token_probabilities(const void* logits, int dtype, int rows, int V, const float* temperature, float* out, void* stream) {
    return gi::dispatch(gi_token_probabilities_impl, logits, dtype, rows, V, temperature, out, stream);
}

extern "C" int gi_verify_drafts(const void* logits, int dtype, int N, int V, int R, int D, const int* row_start, const int* drafted, const int* counts,
                                const float* q, long long q_request, long long q_place, const float* temperature, const float* accept, const float* draw,
                                int* tokens, int* accepted, void* work, void* stream) {
    return gi::dispatch(gi_verify_drafts_impl, logits, dtype, N, V, R, D, row_start, drafted, counts, q, q_request, q_place, temperature, accept, draw,
                        tokens, accepted, work, stream);
}
