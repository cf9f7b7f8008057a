// Drafted tokens against the target's distribution, and the drafter's own probabilities.
//
// Request r brings d_r drafted tokens and d_r + 1 rows of the target's logits. With temperature T > 0 row j's distribution is
//   p_i = e_i * (float)(1 / sum e), e_i = exp((l_i - max l) / T), the sum in 64 bits  (the numbers that the sampler draws from).
// Draft x_j is kept while u_j * q_j(x_j) < p_j(x_j); the first refused one is replaced by a draw from max(p_j - q_j, 0), and with
// all of them kept one more token is drawn from the last row's p: the tokens are then distributed as if each had been drawn from
// the target alone. T <= 0: a draft is kept while it is the row's argmax, which is also what replaces it. The draw takes the first index i of
// weight w_i > 0 with w_0 + .. + w_i > v * sum(w); the random numbers u and v come from the caller.
//
// A cluster of CTAs per row finds max and sum and whether the row's draft is kept; a cluster per request finds the stop and draws there. Where there
// are more rows than the GPU holds at a time, the rows run in the order of the drafts' places, and those whose request has met a
// refusal by then are left out. The answer is a whole number, so sums run in 64 bits: their order moves a boundary between two tokens by
// 1e-13 of the mass, where 32-bit sums would move all 128,000 of them by 1e-7, a different token in one draw of a hundred.
//
// What bounds it: few rows the chain of read, exchange, exponentials, exchange (one user's five rows of 128,256: 6.5 us, the draw 9.7 us of which 4.4
// read p and q); many rows the instructions, 22 a value where the exponential and the quotient alone take 12 (128 requests, 742 rows, of which 550 are
// looked at: 119 us, 82 of them until the rows are through and 37 for the draws behind; 0.57 of the copy bandwidth for what the call cannot do without).
#include <climits>

#include <cooperative_groups.h>

#include "common.cuh"
#include "device_limit.h"

namespace gi {

namespace cg = cooperative_groups;

constexpr int kRowThreads = 512, kRowWarps = kRowThreads / 32;
constexpr int kSmallThreads = 256, kNarrowThreads = 128;        // (many rows that registers hold: row_plan)
constexpr int kRowCtasMost = 8;           // CTAs of a row's cluster
constexpr int kRowUnitsMost = 10;         // groups of four values that a thread holds: vocabularies of up to 163,840 stay in registers
constexpr int kEdge = 4;                  // places at either end of a row that may lie in no whole group

// Two 32-bit operations an instruction, each rounded as its single form.
__device__ __forceinline__ float2 add_2(float2 a, float2 b) {
    float2 d;
    asm("{.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 z, x, y;\nmov.b64 {%0, %1}, z;}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul_2(float2 a, float2 b) {
    float2 d;
    asm("{.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmul.rn.f32x2 z, x, y;\nmov.b64 {%0, %1}, z;}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 fma_2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{.reg .b64 x, y, z, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\nfma.rn.f32x2 w, x, y, z;\nmov.b64 {%0, %1}, w;}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

// exp((l - max) / T). With y the rounded reciprocal of T, q = a y and one correction by the exact remainder give the rounded
// quotient a / T (P. Markstein, IBM J. Res. Dev. 34, 1990): three multiply-adds, two values at a time, instead of the general division. Temperatures
// whose reciprocal could leave the normal range take the division. The dividend is bounded below, where exp gives 0 anyway: an infinite one
// has no remainder.
struct ByTemperature {
    float max, t, y;
    bool plain;
    __device__ ByTemperature(float mx, float temp) : max(mx), t(temp), y(1.0f / temp), plain(!(temp > 1e-3f && temp < 1e3f)) {}
    __device__ __forceinline__ float operator()(float l) const {
        float v[2] = {l, l};
        if (plain) general(v);
        else usual(v);
        return v[0];
    }
    template <int n> __device__ __forceinline__ void general(float (&v)[n]) const {
#pragma unroll
        for (int i = 0; i < n; ++i) v[i] = expf((v[i] - max) / t);
    }
    template <int n> __device__ __forceinline__ void usual(float (&v)[n]) const {
        const float2 y2 = {y, y}, t2 = {-t, -t}, m2 = {-max, -max};
#pragma unroll
        for (int i = 0; i < n; i += 2) {
            float2 a = add_2(make_float2(v[i], v[i + 1]), m2);
            a.x = fmaxf(a.x, -1e30f);
            a.y = fmaxf(a.y, -1e30f);
            const float2 q = mul_2(a, y2), x = fma_2(fma_2(q, t2, a), y2, q);
            v[i] = expf(x.x);
            v[i + 1] = expf(x.y);
        }
    }
};

__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float max_or_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// A row in groups of four neighbours on a boundary of four elements: the first and the last group may reach beyond the row.
template <typename T> struct Row {
    const T* row;
    int V, off, units, begin, end;         // begin, end: this CTA's groups
    int first_whole, end_whole;            // the groups that lie within the row
    __device__ Row(const T* p, int vocab, int part, int log_parts) : row(p), V(vocab) {
        off = static_cast<int>((reinterpret_cast<uintptr_t>(p) / sizeof(T)) & 3);
        units = (V + off + 3) / 4;             // (V leaves room for the sum)
        const int per = (((units - 1) >> log_parts) + 32) & ~31;          // the groups over the CTAs, rounded up, in whole warps
        begin = min(units, part * per);
        end = min(units, begin + per);
        first_whole = off > 0;
        end_whole = (V + off) / 4;
    }
    __device__ __forceinline__ int index(int unit) const { return 4 * unit - off; }
    // the i-th place ahead of the first whole group, or behind the last one; -1: there is none
    __device__ __forceinline__ int head(int i) const { return i < min((4 - off) & 3, V) ? i : -1; }
    __device__ __forceinline__ int tail(int i) const {
        const int at = max(min((4 - off) & 3, V), index(end_whole)) + i;
        return at < V ? at : -1;
    }
    // asks the CTA's whole groups (of this row, or of the same places of a row of 32-bit values) into L2 at once: the passes' own loads, a few a thread
    // at a time, then wait for L2 only
    __device__ __forceinline__ void ask() const { ask(row); }
    template <typename U> __device__ __forceinline__ void ask(const U* values) const {
        const int from = max(begin, first_whole), to = min(end, end_whole);
        const U* at = values + index(from);
        const int skip = static_cast<int>((16 - reinterpret_cast<uintptr_t>(at) % 16) % 16 / sizeof(U));          // (the groups need not lie on 16 bytes)
        const long long bytes = (static_cast<long long>(to - from) * 4 - skip) * sizeof(U) / 16 * 16;
        if (threadIdx.x == 0 && bytes > 0)
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" :: "l"(at + skip), "r"(static_cast<int>(bytes)) : "memory");
    }
    __device__ __forceinline__ void load_whole(int unit, float (&v)[4]) const {
        const int i = index(unit);
        if constexpr (sizeof(T) == 4) {
            const float4 x = *reinterpret_cast<const float4*>(row + i);
            v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
        } else {
            const uint2 x = *reinterpret_cast<const uint2*>(row + i);
            v[0] = __uint_as_float(x.x << 16); v[1] = __uint_as_float(x.x & 0xffff0000u);
            v[2] = __uint_as_float(x.y << 16); v[3] = __uint_as_float(x.y & 0xffff0000u);
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
    double cta_sum[3][kRowCtasMost];       // of the exponentials, of the weights, of the weights where those are nothing
};

// All threads of the cluster meet behind the remote stores of every CTA's first warp: only that warp's arrival has to wait for its stores to be seen.
__device__ __forceinline__ void meet_behind_first_warps() {
    if (threadIdx.x < 32) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    else asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The largest value of the cluster's row (NaN if any value is none); every thread has it.
template <int kThreads>
__device__ __forceinline__ float cluster_max(float mx, RowShared& s, cg::cluster_group& cluster, int part, int parts) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = max_or_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) s.warp_max[warp] = mx;
    __syncthreads();
    cluster.barrier_wait();                // (arrived at when the kernel began)
    if (warp == 0) {
        mx = s.warp_max[lane & ((kThreads / 32) - 1)];
#pragma unroll
        for (int o = (kThreads / 32) / 2; o > 0; o >>= 1) mx = max_or_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        if (lane < parts) *cluster.map_shared_rank(&s.cta_max[part], lane) = mx;
    }
    meet_behind_first_warps();
    mx = s.cta_max[0];
    for (int p = 1; p < parts; ++p) mx = max_or_nan(mx, s.cta_max[p]);
    return mx;
}

// The cluster's sum, in the order of the CTAs; every thread has it. The warps' sums stay in s.warp_sum, the CTAs' in s.cta_sum[turn].
template <int kThreads>
__device__ __forceinline__ double cluster_sum(double v, RowShared& s, int turn, cg::cluster_group& cluster, int part, int parts) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = warp_total(v);
    if (lane == 0) s.warp_sum[warp] = v;
    __syncthreads();
    if (warp == 0) {
        v = s.warp_sum[lane & ((kThreads / 32) - 1)];
#pragma unroll
        for (int o = (kThreads / 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane < parts) *cluster.map_shared_rank(&s.cta_sum[turn][part], lane) = v;
    }
    meet_behind_first_warps();
    v = s.cta_sum[turn][0];
    for (int p = 1; p < parts; ++p) v += s.cta_sum[turn][p];
    return v;
}

__device__ __forceinline__ void keep_best(float v, int i, float& best, int& at) {
    if (v > best || (v == best && i < at)) { best = v; at = i; }
}

// Index of the largest value of the cluster's row, the lowest among equals (values that are no number are passed over; 0 where there
// is no other).
template <int kThreads, typename Each>
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
        for (int w = 1; w < (kThreads / 32); ++w) keep_best(s.warp_max[w], s.warp_at[w], best, at);
        for (int p = 0; p < parts; ++p) {
            *cluster.map_shared_rank(&s.cta_max[part], p) = best;
            *cluster.map_shared_rank(&s.cta_at[part], p) = at;
        }
    }
    meet_behind_first_warps();
    best = s.cta_max[0];
    at = s.cta_at[0];
    for (int p = 1; p < parts; ++p) keep_best(s.cta_max[p], s.cta_at[p], best, at);
    return at == INT_MAX ? 0 : at;
}

// Values of a CTA's whole groups: held in registers (kUnits groups of four a thread) or, kUnits = 0, read again in every pass (the cluster's row is then
// in L2). kOrdered: a warp's groups are neighbours, as a draw wants them; else the block's threads take turns (a little faster). The places
// in no whole group: one each for the first lanes of the first CTA's first warp and of the last CTA's last warp.
template <typename T, int kUnits, bool kOrdered, int kThreads> struct Values {
    static constexpr int kWarps = kThreads / 32;
    static constexpr int kBatch = 4;       // groups whose loads are in flight together
    static constexpr int kStep = kOrdered ? 32 : kThreads;
    const Row<T>& r;
    int first, last, edge_at;
    float edge;
    float held[kUnits > 0 ? kUnits : 1][4];
    __device__ Values(const Row<T>& row, int part, int parts) : r(row) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        last = min(r.end, r.end_whole);
        if constexpr (kOrdered) {
            const int share = ((r.end - r.begin + kWarps - 1) / kWarps + 31) & ~31;
            first = r.begin + warp * share + lane;
            last = min(last, r.begin + (warp + 1) * share);
        } else {
            first = max(r.begin, r.first_whole) + threadIdx.x;
        }
        edge_at = part == 0 && warp == 0 && lane < kEdge ? r.head(lane) : part == parts - 1 && warp == kWarps - 1 && lane >= kEdge && lane < 2 * kEdge ? r.tail(lane - kEdge) : -1;
        edge = edge_at >= 0 ? to_float(r.row[edge_at]) : -INFINITY;
        if constexpr (kUnits > 0) {
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
                held[u][0] = held[u][1] = held[u][2] = held[u][3] = -INFINITY;
                if (there(first + kStep * u)) r.load_whole(first + kStep * u, held[u]);
            }
        }
    }
    __device__ __forceinline__ bool there(int unit) const { return unit < last && (!kOrdered || unit >= r.first_whole); }
    // f(group, values): every group of the thread, in order, until it says stop (kOrdered: by the warp); values of a group that is not there are -infinity
    template <typename F> __device__ __forceinline__ void groups(F f) {
        groups_with([](int, float (&)[4]) {}, [&](int unit, float (&v)[4], float (&)[4]) { return f(unit, v); });
    }
    // f(group, values, others) where more(group, others) fetches four further values of a group that is there (0 where it is not)
    template <typename G, typename F> __device__ __forceinline__ void groups_with(G more, F f) {
        if constexpr (kUnits > 0) {
            float none[4];
#pragma unroll
            for (int u = 0; u < kUnits; ++u)
                if (f(first + kStep * u, held[u], none)) return;
        } else {
            // whole batches of the warp (of the thread, where nothing hangs on the warp) without a look at what is there, then what is left
            const int lane = kOrdered ? threadIdx.x & 31 : 0;
            int unit = first;
            for (; unit + (31 - lane) * kOrdered + kStep * (kBatch - 1) < last && (!kOrdered || unit - lane >= r.first_whole); unit += kBatch * kStep) {
                float v[kBatch][4], w[kBatch][4];
#pragma unroll
                for (int u = 0; u < kBatch; ++u) { r.load_whole(unit + kStep * u, v[u]); more(unit + kStep * u, w[u]); }
#pragma unroll
                for (int u = 0; u < kBatch; ++u)
                    if (f(unit + kStep * u, v[u], w[u])) return;
            }
            for (; unit - lane < last; unit += kBatch * kStep) {
                float v[kBatch][4], w[kBatch][4];
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    v[u][0] = v[u][1] = v[u][2] = v[u][3] = -INFINITY;
                    w[u][0] = w[u][1] = w[u][2] = w[u][3] = 0.f;
                    if (there(unit + kStep * u)) { r.load_whole(unit + kStep * u, v[u]); more(unit + kStep * u, w[u]); }
                }
#pragma unroll
                for (int u = 0; u < kBatch; ++u)
                    if (unit + kStep * u - lane < last && f(unit + kStep * u, v[u], w[u])) return;
            }
        }
    }
};

struct RowArgs {
    const void* logits;
    long long stride;                      // values from row to row
    int N, V, log_parts;                   // CTAs of a row's cluster: 2^log_parts
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
    float4* work;                          // per row: max, 1 / sum, draft kept (1) or not (0), argmax of a greedy row (an integer's bits)
    int R, D, skip;                        // skip: rows behind a refusal that is known when they begin are left out
};

// The request's drafts, or -1 where its rows do not lie in the logits.
__device__ __forceinline__ int drafts_of(const RowArgs& a, int r) {
    const int d = min(max(a.counts[r], 0), a.D), start = a.row_start[r];
    return start < 0 || start > a.N - 1 - d ? -1 : d;
}

// What a draw needs of a row: q's row (or null), the token that a draft without a distribution leaves out, both for refused drafts only.
template <typename T>
__device__ __forceinline__ int draw_token(Values<T, 0, true, kRowThreads>& values, const ByTemperature& by, float inv, const float* q, int without, float number, int V,
                                          RowShared& s, cg::cluster_group& cluster, int part, int parts) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool q_wide = q != nullptr && (reinterpret_cast<uintptr_t>(q) / 4 & 3) == static_cast<unsigned>(values.r.off);
    bool subtract = q != nullptr || without >= 0;
    auto taken = [&](int unit, float (&take)[4]) {
        take[0] = take[1] = take[2] = take[3] = 0.f;
        if (q == nullptr || !subtract) return;
        const int i = values.r.index(unit);
        if (q_wide) {
            const float4 x = *reinterpret_cast<const float4*>(q + i);
            take[0] = x.x; take[1] = x.y; take[2] = x.z; take[3] = x.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) take[e] = q[i + e];
        }
    };
    // the four weights of a group in the place of its values, and their sum
    auto weigh = [&](int unit, float (&w)[4], float (&take)[4]) {
        const int i = values.r.index(unit);
        if (by.plain) by.general(w);
        else by.usual(w);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float pe = __fmul_rn(w[e], inv);
            if (i + e == without && subtract) take[e] = 1.0f;
            w[e] = pe > take[e] ? __fsub_rn(pe, take[e]) : 0.f;      // (a q that is no number takes all)
        }
        return (static_cast<double>(w[0]) + static_cast<double>(w[1])) + (static_cast<double>(w[2]) + static_cast<double>(w[3]));
    };
    auto weigh_edge = [&]() {
        if (values.edge_at < 0) return 0.f;
        const float pe = __fmul_rn(by(values.edge), inv), take = !subtract ? 0.f : q != nullptr ? q[values.edge_at] : values.edge_at == without ? 1.0f : 0.0f;
        return pe > take ? __fsub_rn(pe, take) : 0.f;
    };
    double total;
    int turn = 1;
    for (;; ++turn) {
        double mine = static_cast<double>(weigh_edge());
        values.groups_with(taken, [&](int unit, float (&w)[4], float (&take)[4]) {
            mine += weigh(unit, w, take);
            return false;
        });
        if (turn == 1) cluster.barrier_wait();              // (arrived at when the kernel began)
        total = cluster_sum<kRowThreads>(mine, s, turn, cluster, part, parts);
        if (!subtract || total > 0.0) break;
        subtract = false;                                   // nothing is left of p behind q: the draw is from p (the whole cluster takes this turn)
        __syncthreads();                                    // all have read the warps' sums
    }
    const double target = static_cast<double>(number) * total;
    // The CTA, the warp, the group and the value in which the running sum passes the target, every sum taken the same way by all who
    // compare it; where rounding (or a number of 1 and more) lets none, the last that weighs anything.
    double run = 0.0, ahead = 0.0;
    int owner = -1;
    bool found = false;
    for (int c = 0; c < parts && !found; ++c) {
        const double t = s.cta_sum[turn][c];
        if (t > 0.0) { owner = c; ahead = run; found = run + t > target; }
        run += t;
    }
    if (owner != part) return -1;
    run = ahead;
    owner = -1;
    found = false;
    for (int w = 0; w < kRowWarps && !found; ++w) {
        const double t = s.warp_sum[w];
        if (t > 0.0) { owner = w; ahead = run; found = run + t > target; }
        run += t;
    }
    if (owner != warp) return -1;
    int pick = V - 1;
    // the lanes' sums t in order: the lane that passes the target (or the last that weighs anything), and what lies ahead of it
    auto look = [&](double t, bool& over_any, double& before) {
        double cum = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double m = __shfl_up_sync(0xffffffffu, cum, o);
            if (lane >= o) cum += m;
        }
        const unsigned some = __ballot_sync(0xffffffffu, t > 0.0), over = __ballot_sync(0xffffffffu, t > 0.0 && ahead + cum > target);
        before = ahead + (cum - t);
        ahead += __shfl_sync(0xffffffffu, cum, 31);
        over_any = over != 0;
        return over ? __ffs(over) - 1 : some ? 31 - __clz(some) : -1;
    };
    bool done = false;
    double before;
    auto look_edge = [&](bool mine) {
        const float w = mine ? weigh_edge() : 0.f;
        const int at = look(static_cast<double>(w), done, before);
        if (at >= 0) pick = __shfl_sync(0xffffffffu, values.edge_at, at);
    };
    if (part == 0 && warp == 0) look_edge(lane < kEdge);
    if (!done)
        values.groups_with(taken, [&](int unit, float (&w)[4], float (&take)[4]) {
            const double t = weigh(unit, w, take);
            const int at = look(t, done, before);
            if (at >= 0) {
                int place = 0;
                bool passed = false;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (w[e] > 0.f && !passed) { before += static_cast<double>(w[e]); place = e; passed = before > target; }
                pick = __shfl_sync(0xffffffffu, values.r.index(unit) + place, at);
            }
            return done;
        });
    if (!done && part == parts - 1 && warp == kRowWarps - 1) look_edge(lane >= kEdge);
    return lane == 0 ? pick : -1;
}

// One cluster per row. kProbs: row i's distribution goes to out; else row j of request r: whether its draft is kept, and if there is none or it is not, the
// token that a draw at this row gives.
template <typename T, int kUnits, bool kProbs, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads != kSmallThreads ? 1024 / kThreads : kUnits > 8 ? 2 : 3) row_softmax_kernel(RowArgs a) {
    pdl_prologue();
    __shared__ RowShared s;
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = 1 << a.log_parts, part = blockIdx.x & (parts - 1);
    const int r = blockIdx.x >> a.log_parts;                // the row, or the request
    int row = r, j = 0, d = 0;
    if constexpr (!kProbs) {
        j = blockIdx.y;
        d = drafts_of(a, r);
        if (j > d) return;                 // (the whole cluster)
        row = a.row_start[r] + j;
        if (a.skip && j > 0) {
            // A refusal ahead that has been seen: nobody asks for this row. The cluster's CTAs must all go or all stay: who comes first decides, in the
            // place of the row's token, which belongs to this cluster alone even where requests share rows (the draw writes it afterwards).
            __shared__ int s_decided;
            if (threadIdx.x == 0) {
                int* decided = a.tokens + static_cast<size_t>(r) * (a.D + 1) + j;
                const int mine = *reinterpret_cast<volatile const int*>(a.accepted + r) < j ? 2 : 1;
                const int before = atomicCAS(decided, 0, mine);
                s_decided = before ? before : mine;
            }
            __syncthreads();
            if (s_decided == 2) return;
        }
    }
    cluster.barrier_arrive();              // every CTA of the cluster runs before another writes into its shared memory
    const T* p = static_cast<const T*>(a.logits) + row * a.stride;
    const Row<T> span(p, a.V, part, a.log_parts);
    if constexpr (kUnits == 0) span.ask();
    Values<T, kUnits, false, kThreads> values(span, part, parts);
    const float temp = a.temperature[r];
    // the draft, its logit, its probability in q and the number that decides (the same in every thread)
    int x = -1;
    float lx = 0.f, qx = 1.f, number = 0.f;
    const float* q = nullptr;
    if constexpr (!kProbs) {
        if (j < d) {
            x = a.drafted[static_cast<size_t>(r) * a.D + j];
            number = a.accept[static_cast<size_t>(r) * a.D + j];
            if (x < 0 || x >= a.V) x = -1;
            if (a.q) q = a.q + r * a.q_request + j * a.q_place;
            if (x >= 0) {
                lx = to_float(p[x]);
                if (q) qx = q[x];
            }
        }
    }
    if (!(temp > 0.f)) {
        const int best = cluster_argmax<kThreads>([&](auto f) {
            values.groups([&](int unit, float (&v)[4]) {
                if (values.there(unit))
#pragma unroll
                    for (int e = 0; e < 4; ++e) f(span.index(unit) + e, v[e]);
                return false;
            });
            if (values.edge_at >= 0) f(values.edge_at, values.edge);
        }, s, cluster, part, parts);
        if constexpr (kProbs) {
            float* out = a.out + static_cast<size_t>(row) * a.V;
            const int share = ((a.V - 1) >> a.log_parts) + 1, end = static_cast<int>(min(static_cast<long long>(a.V), static_cast<long long>(part + 1) * share));
            for (int i = part * share + threadIdx.x; i < end; i += kThreads) out[i] = i == best ? 1.0f : 0.0f;
        } else if (part == 0 && threadIdx.x == 0) {
            a.work[row] = make_float4(0.f, 0.f, x == best ? 1.f : 0.f, __int_as_float(best));
            if (a.skip && x != best && j < d) atomicMin(a.accepted + r, j);
        }
        return;
    }
    float mx = values.edge;
    values.groups([&](int, float (&v)[4]) { mx = max_or_nan(max_or_nan(mx, v[0], v[1]), v[2], v[3]); return false; });
    mx = cluster_max<kThreads>(mx, s, cluster, part, parts);
    const bool some = mx > -INFINITY && mx < INFINITY;      // else there are no probabilities (a value is none, or infinite, or all are -infinity)
    const ByTemperature by(mx, temp);
    double sum = 0.0;
    auto weigh = [&](auto exponentials, auto counts) {      // sum += exp of every value; the probabilities keep them
        values.groups([&](int unit, float (&v)[4]) {
            float y[4] = {v[0], v[1], v[2], v[3]};
            exponentials(y);
            if (counts(unit)) sum += (static_cast<double>(y[0]) + static_cast<double>(y[1])) + (static_cast<double>(y[2]) + static_cast<double>(y[3]));
            if constexpr (kProbs) { v[0] = y[0]; v[1] = y[1]; v[2] = y[2]; v[3] = y[3]; }
            return false;
        });
        if (values.edge_at >= 0) sum += static_cast<double>(by(values.edge));
    };
    // (a place that is not there holds -infinity: exp gives 0, but for an infinite temperature, by which it is no number)
    if (some && !by.plain) weigh([&](float (&y)[4]) { by.usual(y); }, [](int) { return true; });
    else if (some) weigh([&](float (&y)[4]) { by.general(y); }, [&](int unit) { return values.there(unit); });
    sum = cluster_sum<kThreads>(sum, s, 0, cluster, part, parts);
    const float inv = some ? static_cast<float>(1.0 / sum) : NAN;
    if constexpr (kProbs) {
        float* out = a.out + static_cast<size_t>(row) * a.V;
        const bool wide = (reinterpret_cast<uintptr_t>(out) / 4 & 3) == static_cast<unsigned>(span.off);
        values.groups([&](int unit, float (&v)[4]) {
            if (!values.there(unit)) return false;
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = __fmul_rn(kUnits > 0 ? v[e] : by(v[e]), inv);
            const int i = span.index(unit);
            if (wide) {
                *reinterpret_cast<float4*>(out + i) = make_float4(y[0], y[1], y[2], y[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) out[i + e] = y[e];
            }
            return false;
        });
        if (values.edge_at >= 0) out[values.edge_at] = __fmul_rn(by(values.edge), inv);
    } else {
        if (part == 0 && threadIdx.x == 0) {
            const bool kept = some && x >= 0 && __fmul_rn(number, qx) < __fmul_rn(by(lx), inv);
            a.work[row] = make_float4(mx, inv, kept ? 1.f : 0.f, 0.f);
            if (a.skip && !kept && j < d) atomicMin(a.accepted + r, j);
        }
    }
}

// Ahead of rows of which some may be left out: no refusal known, no row decided.
__global__ void __launch_bounds__(256) draft_begin_kernel(RowArgs a) {
    pdl_prologue();
    const long long places = static_cast<long long>(a.R) * (a.D + 1);
    for (long long i = blockIdx.x * 256 + threadIdx.x; i < places; i += gridDim.x * 256) {
        a.tokens[i] = 0;
        if (i < a.R) a.accepted[i] = INT_MAX;
    }
}

// One cluster per request: the stop among its rows, and the token there.
template <typename T>
__global__ void __launch_bounds__(kRowThreads, 2) draft_draw_kernel(RowArgs a) {
    pdl_prologue();
    __shared__ RowShared s;
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = 1 << a.log_parts, part = blockIdx.x & (parts - 1);
    const int r = blockIdx.x >> a.log_parts, d = drafts_of(a, r);
    int* tokens = a.tokens + static_cast<size_t>(r) * (a.D + 1);
    if (d < 0) {
        if (part == 0) {
            for (int j = threadIdx.x; j <= a.D; j += kRowThreads) tokens[j] = -1;
            if (threadIdx.x == 0) a.accepted[r] = -1;
        }
        return;
    }
    const int start = a.row_start[r];
    int stop = d;
    for (int j0 = 0; j0 < d && stop == d; j0 += 32) {       // (rows behind the first refusal may not have been written)
        const int j = j0 + (threadIdx.x & 31);
        const unsigned refused = __ballot_sync(0xffffffffu, j < d && a.work[start + j].z == 0.f);
        if (refused) stop = j0 + __ffs(refused) - 1;
    }
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
    cluster.barrier_arrive();                               // every CTA of the cluster runs before another writes into its shared memory
    const Row<T> span(static_cast<const T*>(a.logits) + (start + stop) * a.stride, a.V, part, a.log_parts);
    const float* q = stop < d && a.q ? a.q + r * a.q_request + stop * a.q_place : nullptr;
    span.ask();
    if (q) span.ask(q);
    Values<T, 0, true, kRowThreads> values(span, part, parts);
    const int without = stop < d && !a.q ? a.drafted[static_cast<size_t>(r) * a.D + stop] : -1;
    const int pick = draw_token<T>(values, ByTemperature(stat.x, temp), stat.y, q, without, a.draw[r], a.V, s, cluster, part, parts);
    if (pick >= 0) tokens[stop] = pick;
}

template <typename... KArgs, typename... Args>
inline void launch_row_clusters(void (*kernel)(KArgs...), dim3 grid, int threads, int parts, cudaStream_t stream, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
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

// CTAs of a row's cluster, groups a thread holds (0: read again in every pass, out of L2) and threads of a CTA.
// Few rows: as many CTAs as fit the GPU at once, and registers where those hold the row, for the shortest way from first read to answer.
// Many rows: as few CTAs a row as may be, since what a row costs besides its values (the exchanges within warps, block and cluster) grows with them.
// Probabilities (`keeps`) need every exponential twice and hold it: the fewest CTAs whose registers hold the row (1,000 rows of 32,000: clusters of
// two 61 us, clusters of eight, where a thread has two groups, 157 us). Verification needs them once: kSlice values a CTA and nothing held, two CTAs a
// multiprocessor (742 rows of 128,256, the call: 119 us, 159 us in registers), but for rows that one CTA holds (896 of 9,000: 34 us, 37 us).
// Rows in registers run in CTAs of 256 threads from four a multiprocessor on, whose warps have more to do between two exchanges (300 rows of 32,000:
// 22.9 us, 24.6 us with 512 threads), and of 512 threads below, whose single round is shorter (64 rows of 151,669: 28.2 us, 31.0 us with 256).
// Vocabularies of up to 5,112 run in CTAs of 128 threads, eight a multiprocessor, each with a row (2,304 rows of 5,000: 34 us, 49 us with 512).
constexpr int kSlice = 65536, kDrawSlice = 32768;
constexpr int kNarrowUnits = 10;
// The fewest CTAs a row that have at most `most` groups each (or the most there are); more while all of them still fit the GPU at once.
inline int fewest_parts(long long groups, long long rows, long long most) {
    int log_parts = 0;
    while ((1 << log_parts) < kRowCtasMost && (groups > most << log_parts || (rows << log_parts <= sm_count() && groups > (2LL * kRowThreads << log_parts)))) ++log_parts;
    return log_parts;
}
struct RowPlan { int log_parts, units, threads; };
inline RowPlan row_plan(int V, long long rows, bool keeps = false) {
    const long long groups = (static_cast<long long>(V) + 6) / 4, sms = sm_count();         // with an edge on either side
    constexpr long long kHeld = static_cast<long long>(kRowThreads) * kRowUnitsMost;        // groups that a CTA holds (of 256 threads: twice as many each)
    if (groups <= kNarrowThreads * kNarrowUnits && rows > 2 * sms) return {0, kNarrowUnits, kNarrowThreads};
    const int log_parts = fewest_parts(groups, rows, keeps ? kHeld : kSlice / 4);
    const long long per = (((groups - 1) >> log_parts) + 32) & ~31LL, ctas = rows << log_parts;
    if (per > kHeld) return {log_parts, 0, kRowThreads};
    if (ctas > 4 * sms && (keeps || log_parts == 0)) {
        const long long units = (per + kSmallThreads - 1) / kSmallThreads;
        return {log_parts, units <= 8 ? 8 : units <= 12 ? 12 : units <= 16 ? 16 : 20, kSmallThreads};
    }
    if (!keeps && ctas > 2 * sms) return {log_parts, 0, kRowThreads};
    const long long units = (per + kRowThreads - 1) / kRowThreads;
    return {log_parts, units <= 2 ? 2 : units <= 4 ? 4 : units <= 8 ? 8 : kRowUnitsMost, kRowThreads};
}

template <typename T, bool kProbs>
int launch_rows(RowArgs a, int rows, int places, cudaStream_t st, const char* what) {
    const RowPlan plan = row_plan(a.V, static_cast<long long>(rows) * places, kProbs);
    a.log_parts = plan.log_parts;
    GI_REQUIRE(rows <= INT_MAX >> plan.log_parts && places <= 65535, "%s: %d rows of %d places exceed the grid limit", what, rows, places);
    const dim3 grid(static_cast<unsigned>(rows) << plan.log_parts, places);
    auto run = [&](auto kernel) { launch_row_clusters(kernel, grid, plan.threads, 1 << plan.log_parts, st, a); };
    if (plan.threads == kNarrowThreads) {
        run(row_softmax_kernel<T, kNarrowUnits, kProbs, kNarrowThreads>);
    } else if (plan.threads == kSmallThreads) {
        switch (plan.units) {
            case 8: run(row_softmax_kernel<T, 8, kProbs, kSmallThreads>); break;
            case 12: run(row_softmax_kernel<T, 12, kProbs, kSmallThreads>); break;
            case 16: run(row_softmax_kernel<T, 16, kProbs, kSmallThreads>); break;
            default: run(row_softmax_kernel<T, 20, kProbs, kSmallThreads>); break;
        }
    } else {
        switch (plan.units) {
            case 2: run(row_softmax_kernel<T, 2, kProbs, kRowThreads>); break;
            case 4: run(row_softmax_kernel<T, 4, kProbs, kRowThreads>); break;
            case 8: run(row_softmax_kernel<T, 8, kProbs, kRowThreads>); break;
            case kRowUnitsMost: run(row_softmax_kernel<T, kRowUnitsMost, kProbs, kRowThreads>); break;
            default: run(row_softmax_kernel<T, 0, kProbs, kRowThreads>); break;
        }
    }
    return check_launch(what);
}

template <typename T>
int launch_verify(RowArgs a, cudaStream_t st) {
    // From twice the rows that the GPU holds at a time on (128 requests of six drafts, 2.8 kept: 119 us with rows left out, 135 without)
    const long long rows = static_cast<long long>(a.R) * (a.D + 1);
    a.skip = rows << row_plan(a.V, rows).log_parts > 4LL * sm_count();
    if (a.skip) {
        launch_kernel((draft_begin_kernel), dim3(16), dim3(256), 0, st, a);
        if (check_launch("verify_drafts")) return 1;
    }
    if (const int rc = launch_rows<T, false>(a, a.R, a.D + 1, st, "verify_drafts")) return rc;
    // the draw, a cluster a request (250 requests of 32,000: 66 us in one CTA each, 99 us in eight; 128 of 128,256: 119 us in four or eight, 128 us in two)
    a.log_parts = fewest_parts((static_cast<long long>(a.V) + 6) / 4, a.R, kDrawSlice / 4);
    GI_REQUIRE(a.R <= INT_MAX >> a.log_parts, "verify_drafts: %d requests exceed the grid limit", a.R);
    launch_row_clusters((draft_draw_kernel<T>), dim3(static_cast<unsigned>(a.R) << a.log_parts), kRowThreads, 1 << a.log_parts, st, a);
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
    return dtype == kF32 ? launch_rows<float, true>(a, rows, 1, st, "token_probabilities") : launch_rows<__nv_bfloat16, true>(a, rows, 1, st, "token_probabilities");
}

// logits [N, V]; request r's rows start at row_start[r]; drafted, accept [R, D]; q (or null): q_request / q_place values between
// requests / drafts, V neighbours each; tokens [R, D + 1], accepted [R]; work: 16 bytes a row of logits, aligned to 16.
static int gi_verify_drafts_impl(const void* logits, int dtype, int N, int V, int R, int D, const int* row_start, const int* drafted, const int* counts,
                                 const float* q, long long q_request, long long q_place, const float* temperature, const float* accept, const float* draw,
                                 int* tokens, int* accepted, void* work, void* stream) {
    if (R == 0) return 0;
    GI_REQUIRE(N > 0 && V > 0 && V <= INT_MAX - 8 && R > 0 && D >= 0 && D < INT_MAX, "verify_drafts: sizes must be positive (N=%d, V=%d, R=%d, D=%d)", N, V, R, D);
    GI_REQUIRE(reinterpret_cast<uintptr_t>(work) % 16 == 0, "verify_drafts: the workspace must lie on a boundary of 16 bytes");
    RowArgs a = {};
    a.logits = logits; a.stride = V; a.N = N; a.V = V; a.temperature = temperature; a.row_start = row_start; a.drafted = drafted; a.counts = counts;
    a.q = q; a.q_request = q_request; a.q_place = q_place; a.accept = accept; a.draw = draw; a.tokens = tokens; a.accepted = accepted;
    a.work = static_cast<float4*>(work); a.R = R; a.D = D;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return dtype == kF32 ? launch_verify<float>(a, st) : launch_verify<__nv_bfloat16>(a, st);
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
