// Rows in 8-bit integers: q = rint(v * (127 / m)) with m the row's largest |v|, and the row's scale in 32 bits, scale * q ~ v.
// What the 8-bit product reads (int8_product.cu). The values v come from
//   rows        v = x
//   norm        x <- x + add (optional), v = x * weight; the scale also takes the norm's factor 1 / sqrt(mean(x^2) + eps)
//   activation  v = act(g) * u of a row [g; u], rounded to bfloat16 as the bfloat16 path has it
//
// The norm's factor is the same for the whole row, so the integers do not depend on it: the sum of squares and the largest value
// are found in the same pass and meet in one exchange between the warps, and every thread keeps its values in registers. A pass
// reads the row once and writes a quarter of it (all of it again where the sum goes back): memory bound for many rows, one exchange
// and the launch for few. The integers take three operations that IEEE arithmetic fixes (a product, a quotient per row, a product), so
// they do not depend on how a row is cut over threads.
//
// What is not finite: the largest |v| is kept as the bits of its absolute value, an integer that orders infinities and NaN above
// every number, so that one of them anywhere in a row shows: such a row gets the scale NaN and zeros, and every product with it is
// NaN. A norm whose squares (or products with the weights) leave the range of 32 bits is taken again from values 2^-80 times as large.
// Rows whose largest |v| is below 2^-100 count as zero (scale 0): 127 / m would leave that range at the other end.
#include "common.cuh"

namespace gi {
namespace {

enum RowsKind : int { kRowsPlain = 0, kRowsNorm = 1, kRowsGated = 2 };

struct RowsParams {
    const void* x;          // rows of D values (gated: 2 D), ldx values apart; the norm's are 32-bit and written where add is
    const void* add;        // norm: [T, D] or null
    const float* weight;    // norm: [D]; gated: the bias [2 D] or null
    int8_t* q;              // [T, width]
    float* scales;          // [T]
    long long ldx;
    int T, D, width;        // width: D or more, a multiple of 16; zeros behind D
    int act;
    float limit, eps;
};

constexpr unsigned kInfBits = 0x7f800000u, kLeastBits = 0x0d800000u;      // 2^-100
constexpr float kDown = 8.271806125530277e-25f;                           // 2^-80

template <bool VEC>
__device__ __forceinline__ float4 load4(const float* p, int c, int D) {
    if (VEC) return c < D ? *reinterpret_cast<const float4*>(p + c) : make_float4(0.f, 0.f, 0.f, 0.f);
    return make_float4(c < D ? p[c] : 0.f, c + 1 < D ? p[c + 1] : 0.f, c + 2 < D ? p[c + 2] : 0.f, c + 3 < D ? p[c + 3] : 0.f);
}
template <bool VEC>
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p, int c, int D) {
    if (VEC) {
        if (c >= D) return make_float4(0.f, 0.f, 0.f, 0.f);
        const uint2 raw = *reinterpret_cast<const uint2*>(p + c);
        return make_float4(__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u), __uint_as_float(raw.y << 16),
                           __uint_as_float(raw.y & 0xffff0000u));
    }
    return make_float4(c < D ? to_float(p[c]) : 0.f, c + 1 < D ? to_float(p[c + 1]) : 0.f, c + 2 < D ? to_float(p[c + 2]) : 0.f,
                       c + 3 < D ? to_float(p[c + 3]) : 0.f);
}
template <bool VEC>
__device__ __forceinline__ void store4(float* p, int c, int D, const float4 v) {
    if (VEC) {
        if (c < D) *reinterpret_cast<float4*>(p + c) = v;
        return;
    }
    if (c < D) p[c] = v.x;
    if (c + 1 < D) p[c + 1] = v.y;
    if (c + 2 < D) p[c + 2] = v.z;
    if (c + 3 < D) p[c + 3] = v.w;
}

struct NoAdd {};        // a norm without an addition

__device__ __forceinline__ float gated_bf16(float g, float u, int act, float limit) {
    return __bfloat162float(__float2bfloat16_rn(gated_value(g, u, act, limit)));
}

// Columns c .. c + 3 of a row: v, and what its squares add to ss. `first`: the norm's addition is done and written back.
template <int KIND, typename TX, typename TA, bool VEC>
__device__ __forceinline__ float4 values4(const RowsParams& p, long long row, int c, const float4 w, float factor, bool first, float& ss) {
    const TX* x = static_cast<const TX*>(p.x) + row * p.ldx;
    if constexpr (KIND == kRowsGated) {
        float4 g = load4<VEC>(x, c, p.D), u = load4<VEC>(x + p.D, c, p.D);
        if (p.weight != nullptr) {
            const float4 bg = load4<VEC>(p.weight, c, p.D), bu = load4<VEC>(p.weight + p.D, c, p.D);
            g = make_float4(__fadd_rn(g.x, bg.x), __fadd_rn(g.y, bg.y), __fadd_rn(g.z, bg.z), __fadd_rn(g.w, bg.w));
            u = make_float4(__fadd_rn(u.x, bu.x), __fadd_rn(u.y, bu.y), __fadd_rn(u.z, bu.z), __fadd_rn(u.w, bu.w));
        }
        return make_float4(gated_bf16(g.x, u.x, p.act, p.limit), gated_bf16(g.y, u.y, p.act, p.limit),
                           gated_bf16(g.z, u.z, p.act, p.limit), gated_bf16(g.w, u.w, p.act, p.limit));
    } else if constexpr (KIND == kRowsNorm) {
        float4 v = load4<VEC>(x, c, p.D);
        if constexpr (!std::is_same<TA, NoAdd>::value) {
            if (first) {
                const float4 a = load4<VEC>(static_cast<const TA*>(p.add) + row * p.D, c, p.D);
                v = make_float4(__fadd_rn(v.x, a.x), __fadd_rn(v.y, a.y), __fadd_rn(v.z, a.z), __fadd_rn(v.w, a.w));
                store4<VEC>(static_cast<float*>(const_cast<void*>(p.x)) + row * p.ldx, c, p.D, v);
            }
        }
        v = make_float4(v.x * factor, v.y * factor, v.z * factor, v.w * factor);
        ss = fmaf(v.x, v.x, ss); ss = fmaf(v.y, v.y, ss); ss = fmaf(v.z, v.z, ss); ss = fmaf(v.w, v.w, ss);
        return make_float4(__fmul_rn(v.x, w.x), __fmul_rn(v.y, w.y), __fmul_rn(v.z, w.z), __fmul_rn(v.w, w.w));
    } else {
        return load4<VEC>(x, c, p.D);
    }
}

__device__ __forceinline__ unsigned top_bits(const float4 v, unsigned m) {
    m = max(m, max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu));
    return max(m, max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu));
}

__device__ __forceinline__ uint32_t four_ints(const float4 v, float inv) {
    const int a = __float2int_rn(__fmul_rn(v.x, inv)), b = __float2int_rn(__fmul_rn(v.y, inv));
    const int c = __float2int_rn(__fmul_rn(v.z, inv)), d = __float2int_rn(__fmul_rn(v.w, inv));
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// The row's largest |v| and sum of squares over the G threads that share it.
template <int G, int KIND>
__device__ __forceinline__ void meet(unsigned& m, float& ss, unsigned* part_m, float* part_s) {
    m = __reduce_max_sync(0xffffffffu, m);
    if (KIND == kRowsNorm) ss = warp_sum(ss);
    if (G > 32) {
        constexpr int kWarps = G / 32;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane == 0) { part_m[warp] = m; part_s[warp] = ss; }
        __syncthreads();
        m = lane < kWarps ? part_m[lane] : 0u;
        m = __reduce_max_sync(0xffffffffu, m);
        if (KIND == kRowsNorm) ss = warp_sum(lane < kWarps ? part_s[lane] : 0.f);
    }
}

// 127 / m and the scale of a row; a row that is not finite: 0 and NaN.
template <int KIND>
__device__ __forceinline__ float2 row_factors(unsigned m_bits, float ss, const RowsParams& p, float factor) {
    if (m_bits >= kInfBits || (KIND == kRowsNorm && !(ss < __uint_as_float(kInfBits)))) return make_float2(0.f, __uint_as_float(0x7fc00000u));
    if (m_bits < kLeastBits) return make_float2(0.f, 0.f);
    const float m = __uint_as_float(m_bits);
    float scale = __fdiv_rn(m, 127.f);
    // (of values `factor` times as large: their mean square and eps are both factor^2 times as large, and the factors cancel)
    if (KIND == kRowsNorm) scale = __fdiv_rn(scale, sqrtf(__fdiv_rn(ss, static_cast<float>(p.D)) + p.eps * factor * factor));
    return make_float2(__fdiv_rn(127.f, m), scale);
}

// G threads to a row, V groups of four values each in registers.
template <int KIND, typename TX, typename TA, int G, int V, bool VEC>
__global__ void __launch_bounds__(G < 128 ? 128 : G)
rows_int8_kernel(const RowsParams p) {
    constexpr int kRows = G < 128 ? 128 / G : 1;
    __shared__ unsigned part_m[2][32];
    __shared__ float part_s[2][32];
    const int t = threadIdx.x % G;
    const long long row = static_cast<long long>(blockIdx.x) * kRows + threadIdx.x / G;
    pdl_launch_dependents();
    float4 w[KIND == kRowsNorm ? V : 1];
    if (KIND == kRowsNorm) {      // the weights belong to no earlier kernel
#pragma unroll
        for (int k = 0; k < V; ++k) w[k] = load4<VEC>(p.weight, 4 * (t + k * G), p.D);
    }
    pdl_wait();
    if (row >= p.T) return;       // (whole warps: rows of several to a block have a warp each)
    float4 v[V];
    unsigned m = 0;
    float ss = 0.f, factor = 1.f;
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = values4<KIND, TX, TA, VEC>(p, row, 4 * (t + k * G), w[KIND == kRowsNorm ? k : 0], 1.f, true, ss);
#pragma unroll
    for (int k = 0; k < V; ++k) m = top_bits(v[k], m);
    meet<G, KIND>(m, ss, part_m[0], part_s[0]);
    if (KIND == kRowsNorm && (m >= kInfBits || !(ss < __uint_as_float(kInfBits)))) {
        factor = kDown;
        m = 0;
        ss = 0.f;
#pragma unroll 1
        for (int k = 0; k < V; ++k) {
            const float4 wk = load4<VEC>(p.weight, 4 * (t + k * G), p.D);
            m = top_bits(values4<KIND, TX, TA, VEC>(p, row, 4 * (t + k * G), wk, factor, false, ss), m);
        }
        meet<G, KIND>(m, ss, part_m[1], part_s[1]);
        float unused = 0.f;
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = values4<KIND, TX, TA, VEC>(p, row, 4 * (t + k * G), w[KIND == kRowsNorm ? k : 0], factor, false, unused);
    }
    const float2 f = row_factors<KIND>(m, ss, p, factor);
    const bool none = f.x == 0.f;        // (0 * infinity would not be 0)
    uint32_t* q = reinterpret_cast<uint32_t*>(p.q + row * p.width);
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int c = t + k * G;
        if (4 * c < p.width) q[c] = none ? 0u : four_ints(v[k], f.x);
    }
    if (t == 0) p.scales[row] = f.y;
}

// Rows wider than a block's registers: the same twice over memory.
template <int KIND, typename TX, typename TA>
__global__ void __launch_bounds__(1024)
wide_rows_int8_kernel(const RowsParams p) {
    __shared__ unsigned part_m[2][32];
    __shared__ float part_s[2][32];
    const long long row = blockIdx.x;
    pdl_prologue();
    unsigned m = 0;
    float ss = 0.f, factor = 1.f;
    auto weight = [&](int c) { return KIND == kRowsNorm ? load4<false>(p.weight, c, p.D) : make_float4(0.f, 0.f, 0.f, 0.f); };
    for (int c = 4 * threadIdx.x; c < p.D; c += 4096) m = top_bits(values4<KIND, TX, TA, false>(p, row, c, weight(c), 1.f, true, ss), m);
    meet<1024, KIND>(m, ss, part_m[0], part_s[0]);
    if (KIND == kRowsNorm && (m >= kInfBits || !(ss < __uint_as_float(kInfBits)))) {
        factor = kDown;
        m = 0;
        ss = 0.f;
        for (int c = 4 * threadIdx.x; c < p.D; c += 4096) m = top_bits(values4<KIND, TX, TA, false>(p, row, c, weight(c), factor, false, ss), m);
        meet<1024, KIND>(m, ss, part_m[1], part_s[1]);
    }
    const float2 f = row_factors<KIND>(m, ss, p, factor);
    const bool none = f.x == 0.f;
    uint32_t* q = reinterpret_cast<uint32_t*>(p.q + row * p.width);
    float unused = 0.f;
    for (int c = 4 * threadIdx.x; c < p.width; c += 4096)
        q[c / 4] = none ? 0u : four_ints(values4<KIND, TX, TA, false>(p, row, c, weight(c), factor, false, unused), f.x);
    if (threadIdx.x == 0) p.scales[row] = f.y;
}

template <int KIND, typename TX, typename TA, bool VEC>
void launch_rows(const RowsParams& p, cudaStream_t st) {
    auto go = [&](auto* kernel, int threads, int rows) {
        launch_kernel(kernel, dim3(static_cast<unsigned>((static_cast<long long>(p.T) + rows - 1) / rows)), dim3(threads), 0, st, p);
    };
    if (p.width <= 512) go(rows_int8_kernel<KIND, TX, TA, 32, 4, VEC>, 128, 4);
    else if (p.width <= 2048) go(rows_int8_kernel<KIND, TX, TA, 128, 4, VEC>, 128, 1);
    else if (p.width <= 4096) go(rows_int8_kernel<KIND, TX, TA, 256, 4, VEC>, 256, 1);
    else if (p.width <= 8192) go(rows_int8_kernel<KIND, TX, TA, 512, 4, VEC>, 512, 1);
    else if (p.width <= 16384) go(rows_int8_kernel<KIND, TX, TA, 512, 8, VEC>, 512, 1);
    else if (p.width <= 32768) go(rows_int8_kernel<KIND, TX, TA, 1024, 8, VEC>, 1024, 1);
    else go(wide_rows_int8_kernel<KIND, TX, TA>, 1024, 1);
}

template <int KIND, typename TX, typename TA>
int run_rows(const RowsParams& p, bool vec, cudaStream_t st) {
    if (vec) launch_rows<KIND, TX, TA, true>(p, st);
    else launch_rows<KIND, TX, TA, false>(p, st);
    return check_launch("rows_int8");
}

// 16 bytes of 32-bit values, 8 of bfloat16: whole groups of four
bool aligned4(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype == kF32 ? 16 : 8) == 0; }

int rows_int8_impl(int kind, const void* x, int x_dtype, long long ldx, const void* add, int add_dtype, const float* weight, float eps, int act,
                   float limit, void* q, int width, float* scales, int T, int D, void* stream) {
    if (T == 0) return 0;
    GI_REQUIRE(T > 0 && D > 0, "rows_int8: sizes must be positive (rows=%d, D=%d)", T, D);
    GI_REQUIRE(D <= (1 << 30), "rows_int8: rows of %d values (at most 2^30)", D);
    GI_REQUIRE(width % 16 == 0 && width >= D && width - D < 16, "rows_int8: the output's width %d must be the multiple of 16 that follows %d", width, D);
    GI_REQUIRE(x_dtype == kF32 || x_dtype == kBF16, "rows_int8: unsupported dtype code %d", x_dtype);
    GI_REQUIRE(reinterpret_cast<uintptr_t>(q) % 16 == 0, "rows_int8: the output must be 16-byte aligned");
    GI_REQUIRE(act >= 0 && act < kActCount, "rows_int8: unknown activation %d", act);
    GI_REQUIRE(ldx >= (kind == kRowsGated ? 2ll : 1ll) * D || T == 1, "rows_int8: rows of x overlap");
    const RowsParams p{x, add, weight, static_cast<int8_t*>(q), scales, ldx, T, D, width, act, limit, eps};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    bool vec = D % 4 == 0 && (ldx % 4 == 0 || T == 1) && aligned4(x, x_dtype) && (weight == nullptr || aligned4(weight, kF32));
    if (kind == kRowsNorm) {
        GI_REQUIRE(x_dtype == kF32 && weight != nullptr, "rows_int8: a norm takes 32-bit rows and weights");
        if (add == nullptr) return run_rows<kRowsNorm, float, NoAdd>(p, vec, st);
        GI_REQUIRE(add_dtype == kF32 || add_dtype == kBF16, "rows_int8: unsupported dtype code %d", add_dtype);
        vec = vec && aligned4(add, add_dtype);
        return add_dtype == kF32 ? run_rows<kRowsNorm, float, float>(p, vec, st) : run_rows<kRowsNorm, float, __nv_bfloat16>(p, vec, st);
    }
    if (kind == kRowsGated)
        return x_dtype == kF32 ? run_rows<kRowsGated, float, NoAdd>(p, vec, st) : run_rows<kRowsGated, __nv_bfloat16, NoAdd>(p, vec, st);
    GI_REQUIRE(kind == kRowsPlain, "rows_int8: unknown kind %d", kind);
    return x_dtype == kF32 ? run_rows<kRowsPlain, float, NoAdd>(p, vec, st) : run_rows<kRowsPlain, __nv_bfloat16, NoAdd>(p, vec, st);
}

}  // namespace
}  // namespace gi

// q [T, width] and scales [T] of T rows: kind 0 of x [T, D], 1 of the norm of x (32-bit; x += add [T, D] first where add is given), 2 of
// act(g) * u with x [T, 2 D] = [g; u] and `weight` its bias (may be null). Rows of x lie ldx values apart.
extern "C" int gi_rows_int8(int kind, const void* x, int x_dtype, long long ldx, const void* add, int add_dtype, const float* weight, float eps,
                            int act, float limit, void* q, int width, float* scales, int T, int D, void* stream) {
    return gi::dispatch(gi::rows_int8_impl, kind, x, x_dtype, ldx, add, add_dtype, weight, eps, act, limit, q, width, scales, T, D, stream);
}
