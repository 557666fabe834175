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
    int rows, width;
    int8_t* x8;
    float* scales;
    int32_t* sums;
};

// Eight quantised values; their sum.
__device__ __forceinline__ int quantize_eight(int8_t* x8, const float (&v)[8], float qs) {
    uint32_t w[2] = {0u, 0u};
    int sum = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int q = quantize_one(v[e], qs);
        sum += q;
        w[e >> 2] |= static_cast<uint32_t>(q & 0xFF) << (8 * (e & 3));
    }
    *reinterpret_cast<uint2*>(x8) = make_uint2(w[0], w[1]);
    return sum;
}
__device__ __forceinline__ float inverse_rms(float ss, const NormRowsArgs& a) {
    const float mean = __fdiv_rn(ss, static_cast<float>(a.width));
    return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(mean, a.eps)));
}
__device__ __forceinline__ void scale_eight(float (&v)[8], float inv, const float (&gm)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __fmul_rn(__fmul_rn(v[e], inv), gm[e]);
}
__device__ __forceinline__ float largest_of(float most, const float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]));
    return most;
}
// The row's sum of codes over the CTA, and its two numbers out. `ired` may be
// written again after the CTA's next two barriers.
__device__ __forceinline__ void finish_row(const NormRowsArgs& a, long long row, float m, int sum, int* ired) {
    const int tid = threadIdx.x;
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

// One CTA a row. kG groups of 8 a thread stay in registers; kG = 0: rows too
// wide for that are read in each of three passes (a thread its own values, so
// `out` may be x), the second and third from L2 (4096 rows of 16384 in bf16 with delta
// 99 us, 4.7 TB/s of the bytes of one pass).
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
        scale_eight(v, inv, gm);
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
    const float inv = inverse_rms(group_sum(ss, red, 8, 1), a);
    float local = 0.f;
    if constexpr (kG > 0) {
#pragma unroll
        for (int k = 0; k < kG; ++k) {
            const int g = tid + 256 * k;
            if (g >= groups) continue;
            if (out) store_eight(out + 8 * g, v[k]);
            normed(g, inv, v[k]);
            local = largest_of(local, v[k]);
        }
    } else {
        for (int g = tid; g < groups; g += 256) {
            load(g, v[0]);
            normed(g, inv, v[0]);
            local = largest_of(local, v[0]);
        }
    }
    const float m = group_max(local, red, 8, 1);
    const float qs = quant_multiplier(m);
    int sum = 0;
    if constexpr (kG > 0) {
#pragma unroll
        for (int k = 0; k < kG; ++k)
            if (tid + 256 * k < groups) sum += quantize_eight(x8 + 8 * (tid + 256 * k), v[k], qs);
    } else {
        for (int g = tid; g < groups; g += 256) {
            load(g, v[0]);
            if (out) store_eight(out + 8 * g, v[0]);
            normed(g, inv, v[0]);
            sum += quantize_eight(x8 + 8 * g, v[0], qs);
        }
    }
    finish_row(a, row, m, sum, ired);
}

// Rows of up to 128 groups: a warp a row, without a barrier. Its lane l stands for the
// lanes l of the first kWarps warps above (the others' sums are zeros), whose sums it
// forms one after the other in the same order (16384 rows of 512 in bf16 with delta 33 ->
// 13.6 us, 4.3 TB/s, without 11.2; 10000 of 1000 in fp32 without delta 21 -> 14.0, 3.6
// TB/s, with it 29, 4.5; 16384 of 2048 in bf16 49, a warp a row 68).
template <typename X, typename DT, int kWarps>
__global__ void __launch_bounds__(256) norm_rows_warp_kernel(const NormRowsArgs a) {
    const long long row = blockIdx.x * 8ll + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, groups = a.width >> 3;
    if (row >= a.rows) return;
    const X* x = static_cast<const X*>(a.x) + row * a.x_stride;
    const DT* delta = a.delta ? static_cast<const DT*>(a.delta) + row * a.delta_stride : nullptr;
    X* out = a.out ? static_cast<X*>(a.out) + row * a.out_stride : nullptr;
    int8_t* x8 = a.x8 + row * a.width;
    float v[kWarps][8], ss[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const int g = 32 * w + lane;
        ss[w] = 0.f;
        if (g >= groups) continue;
        load_eight(x + 8 * g, v[w]);
        if (delta) {
            float d[8];
            load_eight(delta + 8 * g, d);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[w][e] = __fadd_rn(v[w][e], d[e]);
        }
    }
    float total = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (32 * w + lane < groups) {
#pragma unroll
            for (int e = 0; e < 8; ++e) ss[w] = __fmaf_rn(v[w][e], v[w][e], ss[w]);
        }
        total += warp_sum(ss[w]);
    }
    const float inv = inverse_rms(total, a);
    float m = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const int g = 32 * w + lane;
        if (g >= groups) continue;
        if (out) store_eight(out + 8 * g, v[w]);
        float gm[8];
        load8(a.weight + 8 * g, gm);
        scale_eight(v[w], inv, gm);
        m = largest_of(m, v[w]);
    }
    m = warp_max(m);
    const float qs = quant_multiplier(m);
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
        if (32 * w + lane < groups) sum += quantize_eight(x8 + 8 * (32 * w + lane), v[w], qs);
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (lane == 0) {
        a.sums[row] = sum;
        a.scales[row] = dequant_scale(m);
    }
}

// Many wider rows: every CTA takes each gridDim.x-th one. Bulk copies bring the next
// rows into shared memory (two of them, x and delta behind each other) while this one
// is normed and stored, and the weights stay in registers: with a CTA a row a thread's
// loads, the two reductions and the stores followed each other, and the weights came
// from the caches once a row (8192 rows of 9728 in bf16 112 -> 89 us, 6.3 TB/s; of
// 2560 in fp32 51 -> 50; three stages leave room for one CTA an SM: 132). A row's
// values are in registers before its first reduction, so its room is free at once.
constexpr int kNormStages = 2;

template <typename X, typename DT, int kG>
__global__ void __launch_bounds__(256) norm_rows_stream_kernel(const NormRowsArgs a) {
    extern __shared__ __align__(128) uint8_t norm_smem[];
    __shared__ float red[32];
    __shared__ int ired[8];
    __shared__ uint64_t full[kNormStages];
    const int tid = threadIdx.x, groups = a.width >> 3, grid = gridDim.x;
    const uint32_t x_bytes = a.width * sizeof(X), delta_bytes = a.delta ? a.width * sizeof(DT) : 0;
    auto stage_of = [&](int s) { return norm_smem + s * (x_bytes + delta_bytes); };
    auto fetch = [&](long long row, int s) {  // by one thread
        mbar_arrive_expect_tx(&full[s], x_bytes + delta_bytes);
        bulk_g2s(stage_of(s), static_cast<const X*>(a.x) + row * a.x_stride, x_bytes, &full[s]);
        if (delta_bytes)
            bulk_g2s(stage_of(s) + x_bytes, static_cast<const DT*>(a.delta) + row * a.delta_stride, delta_bytes, &full[s]);
    };
    if (tid == 0) {
        for (int s = 0; s < kNormStages; ++s) mbar_init(&full[s], 1);
        fence_mbar_init();
    }
    __syncthreads();
    if (tid == 0)
        for (int s = 0; s < kNormStages; ++s)
            if (blockIdx.x + static_cast<long long>(s) * grid < a.rows) fetch(blockIdx.x + static_cast<long long>(s) * grid, s);
    float gm[kG][8];
#pragma unroll
    for (int k = 0; k < kG; ++k)
        if (tid + 256 * k < groups) load8(a.weight + 8 * (tid + 256 * k), gm[k]);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    long long row = blockIdx.x;
    for (; row < a.rows; row += grid) {
        ok = __syncthreads_and(mbar_wait(&full[stage], phase)) != 0;
        if (!ok) break;
        const X* x = reinterpret_cast<const X*>(stage_of(stage));
        const DT* delta = reinterpret_cast<const DT*>(stage_of(stage) + x_bytes);
        float v[kG][8], ss = 0.f;
#pragma unroll
        for (int k = 0; k < kG; ++k) {
            const int g = tid + 256 * k;
            if (g >= groups) continue;
            load_eight(x + 8 * g, v[k]);
            if (delta_bytes) {
                float d[8];
                load_eight(delta + 8 * g, d);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[k][e] = __fadd_rn(v[k][e], d[e]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = __fmaf_rn(v[k][e], v[k][e], ss);
        }
        const float inv = inverse_rms(group_sum(ss, red, 8, 1), a);  // (all have read the row)
        if (tid == 0 && row + static_cast<long long>(kNormStages) * grid < a.rows)
            fetch(row + static_cast<long long>(kNormStages) * grid, stage);
        X* out = a.out ? static_cast<X*>(a.out) + row * a.out_stride : nullptr;
        float local = 0.f;
#pragma unroll
        for (int k = 0; k < kG; ++k) {
            const int g = tid + 256 * k;
            if (g >= groups) continue;
            if (out) store_eight(out + 8 * g, v[k]);
            scale_eight(v[k], inv, gm[k]);
            local = largest_of(local, v[k]);
        }
        const float m = group_max(local, red, 8, 1);
        const float qs = quant_multiplier(m);
        int8_t* x8 = a.x8 + row * a.width;
        int sum = 0;
#pragma unroll
        for (int k = 0; k < kG; ++k)
            if (tid + 256 * k < groups) sum += quantize_eight(x8 + 8 * (tid + 256 * k), v[k], qs);
        finish_row(a, row, m, sum, ired);
        if (++stage == kNormStages) stage = 0, phase ^= 1u;
    }
    if (!ok && tid == 0)  // the copies issued must land before the CTA may exit
        for (int s = 0; s < kNormStages; ++s, row += grid) {
            if (row < a.rows) mbar_wait(&full[stage], phase);
            if (++stage == kNormStages) stage = 0, phase ^= 1u;
        }
}

template <typename X, typename DT, int kG>
static int launch_norm_rows_held(const NormRowsArgs& a, cudaStream_t stream) {
    // CTAs an SM by the registers (weights and values) and by the room of the rows. One
    // alone is slower than a CTA a row (8192 fp32 rows of 9728: 189 and 178 us), and so is
    // a start without a second row to hide (1024 rows of 2560: 7.7 and 8.5 us, 600: 4.9 and
    // 4.4).
    constexpr int kMost = kG == 1 ? 6 : kG == 2 ? 4 : 2;
    const long long smem = static_cast<long long>(kNormStages) * a.width * (sizeof(X) + (a.delta ? sizeof(DT) : 0));
    const int ctas = static_cast<int>(std::min<long long>(kMost, 232448 / (smem + 1280)));
    int sms = 0;
    if (const int rc = paged_sm_count(&sms)) return rc;
    if (ctas < 2 || 2ll * a.rows < 3ll * ctas * sms) {
        norm_rows_kernel<X, DT, kG><<<a.rows, 256, 0, stream>>>(a);
    } else {
        static std::atomic<bool> opted_in[kMaxDevices];
        int dev = 0;
        H4B_CUDA_TRY(cudaGetDevice(&dev));
        if (!opted_in[dev].load(std::memory_order_acquire)) {
            H4B_CUDA_TRY(cudaFuncSetAttribute(norm_rows_stream_kernel<X, DT, kG>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                              232448 - 1024));
            opted_in[dev].store(true, std::memory_order_release);
        }
        norm_rows_stream_kernel<X, DT, kG><<<ctas * sms, 256, static_cast<size_t>(smem), stream>>>(a);
    }
    H4B_CUDA_TRY(cudaGetLastError());
    return 0;
}

template <typename X, typename DT>
static int launch_norm_rows(const NormRowsArgs& a, cudaStream_t stream) {
    const int groups = a.width / 8, per = (groups + 255) / 256;
    if (groups <= 128) {
        const unsigned grid = (static_cast<unsigned>(a.rows) + 7) / 8;
        if (groups <= 64)
            norm_rows_warp_kernel<X, DT, 2><<<grid, 256, 0, stream>>>(a);
        else
            norm_rows_warp_kernel<X, DT, 4><<<grid, 256, 0, stream>>>(a);
        H4B_CUDA_TRY(cudaGetLastError());
        return 0;
    }
    if (per <= 1) return launch_norm_rows_held<X, DT, 1>(a, stream);
    if (per <= 2) return launch_norm_rows_held<X, DT, 2>(a, stream);
    if (per <= 5) return launch_norm_rows_held<X, DT, 5>(a, stream);
    norm_rows_kernel<X, DT, 0><<<a.rows, 256, 0, stream>>>(a);
    H4B_CUDA_TRY(cudaGetLastError());
    return 0;
}

template <typename X>
static int launch_norm_rows_delta(const NormRowsArgs& a, int delta_dtype, cudaStream_t stream) {
    if (a.delta == nullptr || delta_dtype == H4B_FP32) return launch_norm_rows<X, float>(a, stream);
    if (delta_dtype == H4B_FP16) return launch_norm_rows<X, __half>(a, stream);
    return launch_norm_rows<X, __nv_bfloat16>(a, stream);
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
    const NormRowsArgs a{x,      delta, delta ? out : nullptr, x_stride, delta_stride, out_stride, weight, eps,
                         rows,   width, x8,                    scales,   sums};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (x_dtype == H4B_FP32) return launch_norm_rows_delta<float>(a, delta_dtype, s);
    if (x_dtype == H4B_FP16) return launch_norm_rows_delta<__half>(a, delta_dtype, s);
    return launch_norm_rows_delta<__nv_bfloat16>(a, delta_dtype, s);
}
