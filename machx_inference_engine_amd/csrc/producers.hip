// producers.hip — normalisation and gated-activation kernels that emit the block_q8_1x activation stream of the
// int-dot GEMVs together with their fp16 output, so that no separate quantize launch is needed
// (src/ops/elementwise.cpp:136-191, src/ops/deltanet.cpp:73-130).  The quantizer sees the
// ROUNDED fp16 outputs: the stream is bit-identical to quantize_q8_1 run on y afterwards.
#include "mxq_device.h"
#include "mxq_host.h"

namespace mxq {

constexpr int kNormThreads = 256;

// sum over the workgroup; every thread gets the result
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = group_sum<64>(v);
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    if (lane == 63) red[wave] = v;
    __syncthreads();
    float t = 0.f;
    for (uint32_t w = 0; w < (blockDim.x + 63) / 64; ++w) t += red[w];
    __syncthreads();
    return t;
}

// GATED = false: y = half((x * r) * w),            x fp16, w fp32      (rms_norm_f32w_q8)
// GATED = true : y = half((w * (x * r)) * silu(z)), x fp32, w, z fp16   (gated_rms_norm_q8)
// r = rsqrt(mean(x^2) + eps).  One workgroup per row; thread t of pass p owns the 4 elements
// 4 (256 p + t) .. +3, so 8 consecutive threads own one 32-element block.
template <bool GATED, class XT, class WT>
__global__ __launch_bounds__(kNormThreads) void norm_q8_kernel(const XT* x, const half_t* z, const WT* w, half_t* y, uint8_t* q8, uint32_t hidden, float eps) {
    __shared__ float red[kNormThreads / 64];
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const XT* xr = x + (size_t)row * hidden;
    float sum = 0.f;
    for (uint32_t i = tid * 4; i < hidden; i += kNormThreads * 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float v = load_act(xr + i + j);
            sum += v * v;
        }
    }
    sum = block_sum(sum, red);
    const float r = rsqrtf(sum / (float)hidden + eps);
    half_t* yr = y + (size_t)row * hidden;
    uint8_t* qr = q8 + (size_t)row * (hidden / 32) * kQ81xBytes;
    const uint32_t n_pass = (hidden + kNormThreads * 4 - 1) / (kNormThreads * 4);
    for (uint32_t p = 0; p < n_pass; ++p) {
        const uint32_t i = (p * kNormThreads + tid) * 4;
        const bool live = i < hidden;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (live) {
            float o[4];
            half_t h4[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (GATED) {
                    const float xn = load_act(xr + i + j) * r;
                    const float gz = (float)z[(size_t)row * hidden + i + j];
                    o[j] = ((float)w[i + j] * xn) * (gz / (1.f + __expf(-gz)));
                } else {
                    o[j] = (load_act(xr + i + j) * r) * (float)w[i + j];
                }
            }
            // the stream goes by what is stored: without this the compiler rounds a product to fp32 and then to fp16 for the row, at once to fp16 for the stream
            asm("" : "+v"(o[0]), "+v"(o[1]), "+v"(o[2]), "+v"(o[3]));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                h4[j] = (half_t)o[j];
                v[j] = (float)h4[j];
            }
            *reinterpret_cast<uint2*>(yr + i) = *reinterpret_cast<const uint2*>(h4);
        }
        emit_q8_1x(v, tid & 7u, live, qr + (size_t)(i / 32) * kQ81xBytes);
    }
}

// The residual's addition, the norm of the rounded sum and the 8-bit stream of the rounded norm.  A thread owns 8 consecutive elements, those of threads 2 u and 2 u + 1 of norm_q8_kernel<false>: their
// squares are summed apart and in that kernel's order, so that rows normalised here have the bits of those normalised there.
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
struct SumArgs {
    const half_t *x, *residual;
    const float* w;
    half_t *total, *y;
    uint8_t* q8;
    uint32_t n_rows, hidden;
    float eps;
};
__device__ __forceinline__ half8 added(const SumArgs& a, size_t at) {
    const half8 x = *reinterpret_cast<const half8*>(a.x + at), r = *reinterpret_cast<const half8*>(a.residual + at);
    half8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = f32_to_f16_rne((float)x[j] + (float)r[j]);
    *reinterpret_cast<half8*>(a.total + at) = v;
    return v;
}
__device__ __forceinline__ void square(const half8& v, float& even, float& odd) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        even = fmaf((float)v[j], (float)v[j], even);
        odd = fmaf((float)v[j + 4], (float)v[j + 4], odd);
    }
}
struct Weights {
    float4 lo, hi;
};
__device__ __forceinline__ Weights weights_at(const SumArgs& a, uint32_t i) { return {*reinterpret_cast<const float4*>(a.w + i), *reinterpret_cast<const float4*>(a.w + i + 4)}; }
// All threads call (four share a block of 32); those that are not live store nothing.
template <bool HALVES>
__device__ __forceinline__ void normed(const SumArgs& a, size_t at, const half8& v, const Weights& w, float r, bool live) {
    const float ww[8] = {w.lo.x, w.lo.y, w.lo.z, w.lo.w, w.hi.x, w.hi.y, w.hi.z, w.hi.w};
    float f[8];
    half8 o = {};
    if (live) {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = (half_t)(((float)v[j] * r) * ww[j]);
        // the stream goes by what is stored: without this the compiler may round a product twice over, to fp16 at once for the one and by way of fp32 for the other
        typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));
        uint4_t bits = __builtin_bit_cast(uint4_t, o);
        asm("" : "+v"(bits));
        o = __builtin_bit_cast(half8, bits);
        if (a.y) *reinterpret_cast<half8*>(a.y + at) = o;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (float)o[j];
    emit_q8_wide<HALVES>(f, threadIdx.x & 3u, live, a.q8 + at / 32 * (HALVES ? kQ81sBytes : kQ81xBytes));
}

// A workgroup takes a row, 128 threads each 1024 elements of it (a pass), up to eight passes at once; they meet in LDS (FAR, for rows beyond it: in the sum that they wrote), where 128 threads sum
// the squares in the order above, lane by lane of half as many as block_sum has.
// Bound by memory, 8 bytes and the stream's 1.25 or 1.5 an element: 8192 x 4096 53 us, 5.8 TB/s; one row of 4096 2.7 us.  With 128 threads for the whole row, which keep it in registers, the least of
// 21 launches: 61.9 for 51.6 and 3.6 for 2.5; 2048 x 16384 68 for 56, 333 x 2880 5.6 for 4.8.
constexpr uint32_t kSumThreads = 128, kSumPasses = 8, kSumLds = 32768;      // elements that LDS holds
template <bool HALVES, bool FAR>
__global__ __launch_bounds__(kSumThreads * kSumPasses) void add_norm_kernel(SumArgs a) {
    extern __shared__ char sums[];
    __shared__ float red[kSumThreads / 32];
    const uint32_t tid = threadIdx.x, threads = blockDim.x, last = (a.hidden + kSumThreads * 8 - 1) / (kSumThreads * 8) * kSumThreads;
    const size_t row = (size_t)blockIdx.x * a.hidden;
    half8* const rows = reinterpret_cast<half8*>(sums);      // [passes][128]
    auto sum_at = [&](uint32_t i) { return !FAR ? rows[i] : i * 8 < a.hidden ? *reinterpret_cast<const half8*>(a.total + row + i * 8) : half8{}; };
    Weights w;
    if (tid * 8 < a.hidden) w = weights_at(a, tid * 8);
    for (uint32_t i = tid; i < last; i += threads) {
        const half8 v = i * 8 < a.hidden ? added(a, row + i * 8) : half8{};
        if (!FAR) rows[i] = v;
    }
    __syncthreads();
    if (tid < kSumThreads) {
        float even = 0.f, odd = 0.f;
        for (uint32_t i = tid; i < last; i += kSumThreads) square(sum_at(i), even, odd);
        const float part = group_sum<32>(even + odd);
        if ((tid & 31u) == 31) red[tid >> 5] = part;
    }
    __syncthreads();
    const float r = rsqrtf((((red[0] + red[1]) + red[2]) + red[3]) / (float)a.hidden + a.eps);
    for (uint32_t i = tid; i < last; i += threads) {
        const bool live = i * 8 < a.hidden;
        if (live && i != tid) w = weights_at(a, i * 8);
        normed<HALVES>(a, row + i * 8, sum_at(i), w, r, live);
    }
}

// Short rows: LANES lanes take one, up to 8 LANES elements; no barrier: 100000 x 128 19 us, where a workgroup a row takes 53.
template <int LANES, bool HALVES>
__global__ __launch_bounds__(256) void add_norm_short_kernel(SumArgs a) {
    const uint32_t lane = threadIdx.x % LANES, n = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const bool live = n < a.n_rows && lane * 8 < a.hidden;
    const size_t at = (size_t)n * a.hidden + lane * 8;
    half8 v = {};
    Weights w;
    if (live) {
        v = added(a, at);
        w = weights_at(a, lane * 8);
    }
    float even = 0.f, odd = 0.f;
    square(v, even, odd);
    float sum;
    if constexpr (LANES <= 16) {
        sum = group_sum<LANES>(even + odd);
    } else {                 // the halves of a wave
        const float part = group_sum<32>(even + odd), low = u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(part), 31)), high = u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(part), 63));
        sum = LANES == 64 ? low + high : (threadIdx.x & 32u) ? high : low;
    }
    const float r = rsqrtf(sum / (float)a.hidden + a.eps);
    normed<HALVES>(a, at, v, w, r, live);
}

// y = half(silu(gate) * up) (swiglu, src/ops/elementwise.cpp:449-467) or, OAI = true, the clamped
// gpt-oss form x = min(gate, limit), z = clamp(up, -limit, limit), y = half(x * sigmoid(alpha x) * (z + 1))
// (swiglu_oai, :469-492), written as fp16 (when y != NULL) and as the block_q8_1x stream of the rounded
// values: the down projection's int-dot input without a quantize launch.
// E = 8 elements per thread, from kActWideFrom elements on and where gate, up and y lie on 16-byte boundaries: 58.7 M elements 87.2 ->
// 77.3 us (5.4 TB/s, memory-bound), 7.3 M 12.8 -> 11.4 us, 524288 2.5 -> 2.4 us; fewer leave too few waves: 229376 2.12 -> 2.24 us.
constexpr uint64_t kActWideFrom = 524288;
template <bool OAI, int E>
__global__ __launch_bounds__(256) void act_q8_kernel(const half_t* gate, const half_t* up, half_t* y, uint8_t* q8, uint64_t n, float alpha, float limit) {
    typedef _Float16 vec_t __attribute__((ext_vector_type(E)));
    const uint64_t i = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) * E;
    const bool live = i < n;
    float v[E];
#pragma unroll
    for (int j = 0; j < E; ++j) v[j] = 0.f;
    if (live) {
        const vec_t gv = *reinterpret_cast<const vec_t*>(gate + i), uv = *reinterpret_cast<const vec_t*>(up + i);
        vec_t hv;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            float o;
            if (OAI) {
                const float x = fminf((float)gv[j], limit), z = fmaxf(fminf((float)uv[j], limit), -limit);
                o = (x / (1.f + __expf(alpha * (-x)))) * (z + 1.f);
            } else {
                const float g = (float)gv[j];
                o = (g / (1.f + __expf(-g))) * (float)uv[j];
            }
            hv[j] = (half_t)o;
            v[j] = (float)hv[j];
        }
        if (y) *reinterpret_cast<vec_t*>(y + i) = hv;
    }
    uint8_t* blk = q8 + (i / 32) * kQ81xBytes;
    if constexpr (E == 8) emit_q8_wide<false>(v, threadIdx.x & 3u, live, blk);
    else emit_q8_1x(v, threadIdx.x & 7u, live, blk);
}

template <bool OAI>
static int act_q8(mx_stream_t s, const uint16_t* gate, const uint16_t* up, uint16_t* y, void* q8_out, uint64_t n, float alpha, float limit) {
    MX_REQUIRE_PTR(gate); MX_REQUIRE_PTR(up); MX_REQUIRE_PTR(q8_out);
    MX_REQUIRE_SHAPE(n > 0 && n % 32 == 0 && (n / 4 + 255) / 256 <= 0x7FFFFFFFull);
    MX_REQUIRE_ALIGN(gate, 8); MX_REQUIRE_ALIGN(up, 8); MX_REQUIRE_ALIGN(y, 8); MX_REQUIRE_ALIGN(q8_out, 8);
    const half_t *g = reinterpret_cast<const half_t*>(gate), *u = reinterpret_cast<const half_t*>(up);
    half_t* yh = reinterpret_cast<half_t*>(y);
    uint8_t* q = static_cast<uint8_t*>(q8_out);
    if (n >= kActWideFrom && aligned(gate, 16) && aligned(up, 16) && aligned(y, 16))
        hipLaunchKernelGGL((act_q8_kernel<OAI, 8>), dim3((uint32_t)((n / 8 + 255) / 256)), dim3(256), 0, as_stream(s), g, u, yh, q, n, alpha, limit);
    else
        hipLaunchKernelGGL((act_q8_kernel<OAI, 4>), dim3((uint32_t)((n / 4 + 255) / 256)), dim3(256), 0, as_stream(s), g, u, yh, q, n, alpha, limit);
    return launch_status();
}

template <bool B>
struct Bool {
    static constexpr bool value = B;
};

static int check_norm(const void* x, const void* w, const void* y, const void* q8, uint32_t n_rows, uint32_t hidden) {
    MX_REQUIRE_PTR(x); MX_REQUIRE_PTR(w); MX_REQUIRE_PTR(y); MX_REQUIRE_PTR(q8);
    MX_REQUIRE_SHAPE(n_rows > 0 && hidden > 0 && hidden % 32 == 0);
    MX_REQUIRE_ALIGN(y, 8); MX_REQUIRE_ALIGN(q8, 8);
    return MX_OK;
}

}  // namespace mxq

using namespace mxq;

extern "C" {

int mx_rms_norm_f32w_q8(mx_stream_t s, const uint16_t* x, const float* w, uint16_t* y, void* q8_out, uint32_t n_rows, uint32_t hidden, float eps) {
    if (int rc = check_norm(x, w, y, q8_out, n_rows, hidden)) return rc;
    hipLaunchKernelGGL((norm_q8_kernel<false, half_t, float>), dim3(n_rows), dim3(kNormThreads), 0, as_stream(s), reinterpret_cast<const half_t*>(x),
                       (const half_t*)nullptr, w, reinterpret_cast<half_t*>(y), static_cast<uint8_t*>(q8_out), hidden, eps);
    return launch_status();
}

int mx_gated_rms_norm_q8(mx_stream_t s, const float* x, const uint16_t* z, const uint16_t* weight, uint16_t* y, void* q8_out, uint32_t n_rows,
                         uint32_t hidden, float eps) {
    if (int rc = check_norm(x, weight, y, q8_out, n_rows, hidden)) return rc;
    MX_REQUIRE_PTR(z);
    hipLaunchKernelGGL((norm_q8_kernel<true, float, half_t>), dim3(n_rows), dim3(kNormThreads), 0, as_stream(s), x, reinterpret_cast<const half_t*>(z),
                       reinterpret_cast<const half_t*>(weight), reinterpret_cast<half_t*>(y), static_cast<uint8_t*>(q8_out), hidden, eps);
    return launch_status();
}

int mx_add_rms_norm_f32w_q8(mx_stream_t s, const uint16_t* x, const uint16_t* residual, const float* w, uint16_t* sum, uint16_t* y, void* q8_out, uint32_t n_rows,
                            uint32_t hidden, float eps, int halves) {
    MX_REQUIRE_PTR(x); MX_REQUIRE_PTR(residual); MX_REQUIRE_PTR(w); MX_REQUIRE_PTR(sum); MX_REQUIRE_PTR(q8_out);
    MX_REQUIRE_SHAPE(n_rows > 0 && hidden > 0 && hidden % 32 == 0);
    const uint32_t passes = (hidden + kSumThreads * 8 - 1) / (kSumThreads * 8), at_once = passes < kSumPasses ? passes : kSumPasses;
    MX_REQUIRE_SHAPE((uint64_t)n_rows * at_once < (1u << 25));       // a launch holds fewer than 2^32 threads
    MX_REQUIRE_ALIGN(x, 16); MX_REQUIRE_ALIGN(residual, 16); MX_REQUIRE_ALIGN(w, 16); MX_REQUIRE_ALIGN(sum, 16); MX_REQUIRE_ALIGN(y, 16);
    MX_REQUIRE_ALIGN(q8_out, halves ? 16 : 8);
    const SumArgs a = {reinterpret_cast<const half_t*>(x), reinterpret_cast<const half_t*>(residual), w, reinterpret_cast<half_t*>(sum), reinterpret_cast<half_t*>(y), static_cast<uint8_t*>(q8_out),
                       n_rows, hidden, eps};
    auto launch = [&](auto kernel, uint32_t workgroups, uint32_t threads, uint32_t lds) {
        hipLaunchKernelGGL(kernel, dim3(workgroups), dim3(threads), lds, as_stream(s), a);
        return launch_status();
    };
    auto form = [&](auto h) {
        constexpr bool H = decltype(h)::value;
        if (hidden <= 128) return launch(add_norm_short_kernel<16, H>, (n_rows + 15) / 16, 256, 0);
        if (hidden <= 256) return launch(add_norm_short_kernel<32, H>, (n_rows + 7) / 8, 256, 0);
        if (hidden <= 512) return launch(add_norm_short_kernel<64, H>, (n_rows + 3) / 4, 256, 0);
        const uint32_t threads = kSumThreads * at_once;
        if (hidden > kSumLds) return launch(add_norm_kernel<H, true>, n_rows, threads, 0);
        static LdsLimit limit;
        const uint32_t lds = passes * kSumThreads * 16;
        if (lds + kSumThreads / 32 * sizeof(float) > kLdsDefaultLimit)       // with the kernel's own
            if (int rc = raise_lds_limit(reinterpret_cast<const void*>(add_norm_kernel<H, false>), limit, lds)) return rc;
        return launch(add_norm_kernel<H, false>, n_rows, threads, lds);
    };
    return halves ? form(Bool<true>()) : form(Bool<false>());
}

int mx_swiglu_q8(mx_stream_t s, const uint16_t* gate, const uint16_t* up, uint16_t* y, void* q8_out, uint64_t n) {
    return act_q8<false>(s, gate, up, y, q8_out, n, 0.f, 0.f);
}
int mx_swiglu_oai_q8(mx_stream_t s, const uint16_t* gate, const uint16_t* up, uint16_t* y, void* q8_out, uint64_t n, float alpha, float limit) {
    return act_q8<true>(s, gate, up, y, q8_out, n, alpha, limit);
}

}  // extern "C"
