// Residual addition, RMSNorm and int8 rows with scales in one pass: the input
// of the int4 products, for rows that do not come from a product's own
// residual epilogue.
//
//   s = x + delta;  y = s / sqrt(mean(s^2) + eps) * weight;  m = max(max|y|, 1e-5)
//   q = rint(y * (127 / m)), scale = m / 127, sum = sum of q
//
// x and delta are fp32, fp16 or bf16 each; s is fp32 and rounded to x's type
// only where it is stored (y is formed of the unrounded s). The orders are
// those of batch_rmsnorm_quant_kernel (thread p sums the groups of 8 values p,
// p + 256, ..., warps by butterfly, their totals in order), so fp32 rows give
// the bits of h4b_rmsnorm and h4b_quantize_rows.

namespace h4b {

// Eight consecutive values, 16-byte aligned, as fp32.
__device__ __forceinline__ void load_eight(const float* p, float (&v)[8]) { load8(p, v); }
template <typename T>
__device__ __forceinline__ void load_eight(const T* p, float (&v)[8]) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const float2 a = Pair<T>::unpack(w.x), b = Pair<T>::unpack(w.y), c = Pair<T>::unpack(w.z), d = Pair<T>::unpack(w.w);
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
}
__device__ __forceinline__ void store_eight(float* p, const float (&v)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
template <typename T>
__device__ __forceinline__ void store_eight(T* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(Pair<T>::pack(v[0], v[1]), Pair<T>::pack(v[2], v[3]),
                                              Pair<T>::pack(v[4], v[5]), Pair<T>::pack(v[6], v[7]));
}

struct NormRowsArgs {
    const void *x, *delta;  // delta may be null
    void* out;              // where s goes (null: nowhere)
    long long x_stride, delta_stride, out_stride;
    const float* weight;
    float eps;
    int width;
    int8_t* x8;
    float* scales;
    int32_t* sums;
};

// One CTA a row. kG groups of 8 a thread stay in registers; kG = 0: rows too
// wide for that are read in each of three passes (a thread its own values, so
// `out` may be x).
template <typename X, typename DT, int kG>
__global__ void __launch_bounds__(256) norm_rows_kernel(const NormRowsArgs a) {
    __shared__ float red[32];
    __shared__ int ired[8];
    const long long row = blockIdx.x;
    const int tid = threadIdx.x, groups = a.width >> 3;
    const X* x = static_cast<const X*>(a.x) + row * a.x_stride;
    const DT* delta = a.delta ? static_cast<const DT*>(a.delta) + row * a.delta_stride : nullptr;
    X* out = a.out ? static_cast<X*>(a.out) + row * a.out_stride : nullptr;
    int8_t* x8 = a.x8 + row * a.width;
    auto load = [&](int g, float (&v)[8]) {
        load_eight(x + 8 * g, v);
        if (delta) {
            float d[8];
            load_eight(delta + 8 * g, d);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = __fadd_rn(v[e], d[e]);
        }
    };
    auto normed = [&](int g, float inv, float (&v)[8]) {
        float gm[8];
        load8(a.weight + 8 * g, gm);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __fmul_rn(__fmul_rn(v[e], inv), gm[e]);
    };
    auto quantize = [&](int g, float qs, const float (&v)[8]) {
        uint32_t w[2] = {0u, 0u};
        int sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int q = quantize_one(v[e], qs);
            sum += q;
            w[e >> 2] |= static_cast<uint32_t>(q & 0xFF) << (8 * (e & 3));
        }
        *reinterpret_cast<uint2*>(x8 + 8 * g) = make_uint2(w[0], w[1]);
        return sum;
    };
    constexpr int kHeld = kG > 0 ? kG : 1;
    float v[kHeld][8];
    float ss = 0.f;
    if constexpr (kG > 0) {
#pragma unroll
        for (int k = 0; k < kG; ++k) {
            const int g = tid + 256 * k;
            if (g >= groups) continue;
            load(g, v[k]);
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = __fmaf_rn(v[k][e], v[k][e], ss);
        }
    } else {
        for (int g = tid; g < groups; g += 256) {
            load(g, v[0]);
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = __fmaf_rn(v[0][e], v[0][e], ss);
        }
    }
    ss = group_sum(ss, red, 8, 1);
    const float mean = __fdiv_rn(ss, static_cast<float>(a.width));
    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(mean, a.eps)));
    float local = 0.f;
    if constexpr (kG > 0) {
#pragma unroll
        for (int k = 0; k < kG; ++k) {
            const int g = tid + 256 * k;
            if (g >= groups) continue;
            if (out) store_eight(out + 8 * g, v[k]);
            normed(g, inv, v[k]);
#pragma unroll
            for (int e = 0; e < 8; ++e) local = fmaxf(local, fabsf(v[k][e]));
        }
    } else {
        for (int g = tid; g < groups; g += 256) {
            load(g, v[0]);
            normed(g, inv, v[0]);
#pragma unroll
            for (int e = 0; e < 8; ++e) local = fmaxf(local, fabsf(v[0][e]));
        }
    }
    const float m = group_max(local, red, 8, 1);
    const float qs = quant_multiplier(m);
    int sum = 0;
    if constexpr (kG > 0) {
#pragma unroll
        for (int k = 0; k < kG; ++k)
            if (tid + 256 * k < groups) sum += quantize(tid + 256 * k, qs, v[k]);
    } else {
        for (int g = tid; g < groups; g += 256) {
            load(g, v[0]);
            if (out) store_eight(out + 8 * g, v[0]);
            normed(g, inv, v[0]);
            sum += quantize(g, qs, v[0]);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((tid & 31) == 0) ired[tid >> 5] = sum;
    __syncthreads();
    if (tid == 0) {
        int t = 0;
        for (int w = 0; w < 8; ++w) t += ired[w];
        a.sums[row] = t;
        a.scales[row] = dequant_scale(m);
    }
}

template <typename X, typename DT>
static int launch_norm_rows(const NormRowsArgs& a, int rows, cudaStream_t stream) {
    const int per = (a.width / 8 + 255) / 256;
    if (per <= 1)
        norm_rows_kernel<X, DT, 1><<<rows, 256, 0, stream>>>(a);
    else if (per <= 2)
        norm_rows_kernel<X, DT, 2><<<rows, 256, 0, stream>>>(a);
    else if (per <= 5)
        norm_rows_kernel<X, DT, 5><<<rows, 256, 0, stream>>>(a);
    else
        norm_rows_kernel<X, DT, 0><<<rows, 256, 0, stream>>>(a);
    H4B_CUDA_TRY(cudaGetLastError());
    return 0;
}

template <typename X>
static int launch_norm_rows_delta(const NormRowsArgs& a, int delta_dtype, int rows, cudaStream_t stream) {
    if (a.delta == nullptr || delta_dtype == H4B_FP32) return launch_norm_rows<X, float>(a, rows, stream);
    if (delta_dtype == H4B_FP16) return launch_norm_rows<X, __half>(a, rows, stream);
    return launch_norm_rows<X, __nv_bfloat16>(a, rows, stream);
}

}  // namespace h4b

extern "C" int h4b_rmsnorm_quantize_rows(const void* x, int x_dtype, long long x_stride, const void* delta, int delta_dtype,
                                         long long delta_stride, void* out, long long out_stride, const float* weight,
                                         float eps, int8_t* x8, float* scales, int32_t* sums, int rows, int width,
                                         void* stream) {
    using namespace h4b;
    const auto known = [](int t) { return t == H4B_FP32 || t == H4B_FP16 || t == H4B_BF16; };
    if (rows < 0 || width < 8 || (width & 7)) return H4B_EINVAL;
    if (!known(x_dtype) || (delta != nullptr && !known(delta_dtype))) return H4B_EUNSUPPORTED;
    if (rows == 0) return 0;
    if (!x || !weight || !x8 || !scales || !sums || (delta != nullptr && out == nullptr)) return H4B_EINVAL;
    if (x_stride < width || (x_stride & 7) || (delta && (delta_stride < width || (delta_stride & 7))) ||
        (out && (out_stride < width || (out_stride & 7))))
        return H4B_EINVAL;
    if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(delta) | reinterpret_cast<uintptr_t>(out) |
          reinterpret_cast<uintptr_t>(weight)) & 15) || (reinterpret_cast<uintptr_t>(x8) & 7))
        return H4B_EINVAL;
    const NormRowsArgs a{x, delta, delta ? out : nullptr, x_stride, delta_stride, out_stride, weight, eps, width, x8, scales, sums};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (x_dtype == H4B_FP32) return launch_norm_rows_delta<float>(a, delta_dtype, rows, s);
    if (x_dtype == H4B_FP16) return launch_norm_rows_delta<__half>(a, delta_dtype, rows, s);
    return launch_norm_rows_delta<__nv_bfloat16>(a, delta_dtype, rows, s);
}
