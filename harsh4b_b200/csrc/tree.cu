// Drafted token trees after the model has run their nodes: which branch agrees
// with the model (accept), and its K and V moved behind the context (keep).
// The batch's tables are those of paged.cu: sequence b's nodes are rows
// q_offsets[b] .. q_offsets[b + 1] - 1, at most kTreeNodes of them, and
// parents[row] is a node's parent within its sequence.

namespace h4b {

// ---- acceptance ---------------------------------------------------------------
// target[i] is the model's greedy token after node i: the first maximum of its
// logits, a NaN counting as the largest (numpy's and torch's rule). Node 0 is
// the token that was decided already; the branch goes on with the first child
// whose token is its parent's target, as long as there is one.
// One CTA reads a part of a row's logits; the one that is last of its sequence
// follows the branch. Which that is changes nothing: the parts' maxima are
// joined by value and index.
// Bound by HBM: the logits are read once (64 trees, 790 rows of 151936 in fp32: 75 us,
// 6.4 TB/s; 6 rows: 10.8, of which the parts' reads are 1: the chain from the tables
// over the last part's arrival to the branch is the rest).
constexpr int kAcceptThreads = 256;
static_assert(kAcceptThreads >= kTreeNodes, "a thread a node");
constexpr int kAcceptPart = 16384;  // bytes of a part, at least

struct AcceptArgs {
    const void* logits;
    long long logits_stride;
    int vocab, splits, part;          // parts of a row, values of a part (a multiple of 16 bytes' worth)
    const int32_t *tokens, *parents, *q_offsets;
    int sequences, rows, max_path;
    int32_t *targets, *path, *counts, *next_tokens;
    unsigned long long* keys;         // [rows][splits], the parts' maxima
    unsigned int* arrived;            // [sequences], parts that are done
};

// Larger value first, then the smaller index; no -0, and any NaN above all.
__device__ __forceinline__ unsigned long long accept_key(float v, uint32_t index) {
    uint32_t b = __float_as_uint(v + 0.f);
    b = v != v ? 0xFFFFFFFFu : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return (static_cast<unsigned long long>(b) << 32) | (0xFFFFFFFFu - index);
}

template <typename S>
struct Logits16B;  // 16 bytes of logits
template <>
struct Logits16B<float> {
    static constexpr int kCount = 4;
    __device__ static void unpack(uint4 w, float (&v)[4]) {
        v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
    }
    __device__ static float value(float x) { return x; }
};
template <typename T>
struct Logits16B {
    static constexpr int kCount = 8;
    __device__ static void unpack(uint4 w, float (&v)[8]) {
        const float2 a = Pair<T>::unpack(w.x), b = Pair<T>::unpack(w.y), c = Pair<T>::unpack(w.z), d = Pair<T>::unpack(w.w);
        v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
    }
    __device__ static float value(T x) { return static_cast<float>(x); }
};

// Whether the offsets ascend within the rows: else the batch holds no sequence.
// By the whole CTA.
__device__ __forceinline__ bool offsets_ascend(const AcceptArgs& a) {
    bool good = true;
    for (int j = threadIdx.x; j < a.sequences; j += kAcceptThreads)
        good = good && a.q_offsets[j] >= 0 && a.q_offsets[j] <= a.q_offsets[j + 1] && a.q_offsets[j + 1] <= a.rows;
    return __syncthreads_and(good) != 0;
}

__device__ __forceinline__ void no_branch(const AcceptArgs& a, int b) {
    for (int i = 0; i < a.max_path; ++i) a.path[static_cast<long long>(b) * a.max_path + i] = -1;
    a.counts[b] = 0;
    a.next_tokens[b] = -1;
}

// The branch of sequence b, whose `count` targets stand in `target`. By the
// whole CTA, which has written them and not yet met.
__device__ __forceinline__ void follow_branch(const AcceptArgs& a, int b, int first, int count, const int32_t* target) {
    __shared__ int child[kTreeNodes];  // the first child that agrees with its parent's target
    const int i = threadIdx.x;
    if (i < count) child[i] = INT_MAX;
    __syncthreads();
    if (i < count) {
        const int p = checked_parent(a.parents[first + i], i);
        if (p >= 0 && a.tokens[first + i] == target[p]) atomicMin(&child[p], i);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int32_t* path = a.path + static_cast<long long>(b) * a.max_path;
        int node = 0, n = 1;
        path[0] = 0;
        while (n < a.max_path && child[node] != INT_MAX) {
            node = child[node];
            path[n++] = node;
        }
        a.counts[b] = n;
        a.next_tokens[b] = target[node];
        for (; n < a.max_path; ++n) path[n] = -1;
    }
}

template <typename S>
__global__ void __launch_bounds__(kAcceptThreads) accept_logits_kernel(const AcceptArgs a) {
    using V = Logits16B<S>;
    __shared__ unsigned long long warp_keys[kAcceptThreads / 32];
    __shared__ int32_t target[kTreeNodes];
    __shared__ bool last;
    const int tid = threadIdx.x;
    const bool good = offsets_ascend(a);
    const int row = static_cast<int>(blockIdx.x / static_cast<unsigned>(a.splits)), split = blockIdx.x % a.splits;
    if (row >= a.rows) {  // the last CTA: sequences without a branch
        if (!good && tid == 0) report(kStatusBadPage);
        for (int b = tid; b < a.sequences; b += kAcceptThreads) {
            const int n = good ? a.q_offsets[b + 1] - a.q_offsets[b] : 0;
            if (n > kTreeNodes) report(kStatusBadPage);
            if (n == 0 || n > kTreeNodes) no_branch(a, b);
        }
        return;
    }
    if (!good) return;
    int b = -1;  // the row's sequence: the last whose offset is not past it
    for (int j = 0; j < a.sequences; j += kAcceptThreads)
        b += __syncthreads_count(j + tid < a.sequences && a.q_offsets[j + tid] <= row);
    if (b < 0) return;
    const int first = a.q_offsets[b], count = a.q_offsets[b + 1] - first;
    if (row >= first + count || count > kTreeNodes) return;

    const S* values = static_cast<const S*>(a.logits) + row * a.logits_stride;
    const int from = split * a.part, to = min(from + a.part, a.vocab);
    float best = -INFINITY;
    int at = INT_MAX;
    auto look = [&](float v, int i) {
        if (at == INT_MAX || v > best || (v != v && best == best)) best = v, at = i;
    };
    // 16 bytes at a time from the first aligned value on
    const uintptr_t start = reinterpret_cast<uintptr_t>(values + from);
    const int shift = static_cast<int>((16u - (start & 15u)) & 15u) / static_cast<int>(sizeof(S));
    const int head = min(from + shift, to), units = (to - head) / V::kCount;
    if (tid < head - from) look(V::value(values[from + tid]), from + tid);
    const uint4* wide = reinterpret_cast<const uint4*>(values + head);
    for (int u = tid; u < units; u += kAcceptThreads) {
        float v[V::kCount];
        V::unpack(__ldcs(wide + u), v);
#pragma unroll
        for (int e = 0; e < V::kCount; ++e) look(v[e], head + u * V::kCount + e);
    }
    const int tail = head + units * V::kCount + tid;
    if (tail < to) look(V::value(values[tail]), tail);

    unsigned long long key = at == INT_MAX ? 0ull : accept_key(best, static_cast<uint32_t>(at));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
    if ((tid & 31) == 0) warp_keys[tid >> 5] = key;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kAcceptThreads / 32; ++w) key = max(key, warp_keys[w]);
        __stcg(a.keys + static_cast<long long>(row) * a.splits + split, key);
        __threadfence();
        last = atom_acq_rel_add(a.arrived + b, 1u) == static_cast<unsigned>(count * a.splits - 1);
        if (last) a.arrived[b] = 0u;  // for the next call
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    if (tid < count) {
        // (all of the workspace is zero between calls, so that the next may be of any size)
        unsigned long long *keys = a.keys + static_cast<long long>(first + tid) * a.splits, most = 0ull;
        for (int k = 0; k < a.splits; ++k) {
            most = max(most, __ldcg(keys + k));
            keys[k] = 0ull;
        }
        target[tid] = static_cast<int32_t>(0xFFFFFFFFu - static_cast<uint32_t>(most & 0xFFFFFFFFull));
        a.targets[first + tid] = target[tid];
    }
    follow_branch(a, b, first, count, target);
}

// The same for targets that the caller chose, a CTA a sequence: the latency of a launch
// and a chain of small loads (2.3 us, one tree of 8 nodes as 64 of up to 16).
__global__ void __launch_bounds__(kAcceptThreads) accept_targets_kernel(const AcceptArgs a) {
    __shared__ int32_t target[kTreeNodes];
    const int b = blockIdx.x, first = a.q_offsets[b], end = a.q_offsets[b + 1], count = end - first;
    if (first < 0 || end < first || end > a.rows || count > kTreeNodes || count == 0) {
        if (threadIdx.x == 0) {
            if (!(first >= 0 && end == first && end <= a.rows)) report(kStatusBadPage);
            no_branch(a, b);
        }
        return;
    }
    if (threadIdx.x < count) target[threadIdx.x] = a.targets[first + threadIdx.x];
    follow_branch(a, b, first, count, target);
}

// Parts of a row: enough CTAs for the device, none of less than kAcceptPart bytes.
constexpr int kAcceptCtas = 592;
static int accept_splits(int rows, long long row_bytes) {
    const long long most = (row_bytes + kAcceptPart - 1) / kAcceptPart, wanted = (kAcceptCtas + rows - 1) / rows;
    return static_cast<int>(wanted < most ? wanted : most);
}

// ---- keeping the accepted tokens --------------------------------------------------
// Slot context + path[i] -> slot context + i of every layer's K and V. A thread
// moves 16 bytes of a head for all the path's nodes, in their order: path
// ascends, so what a store overwrites (slot i) was read by an earlier step
// (a later step j > i reads path[j] >= j). kKeepBatch loads are in flight at a time: the
// stores of a batch lie below all later reads.
// Bound by HBM: twice the bytes of the nodes that move (64 branches of up to 6 nodes in
// 36 layers of 8 heads of 128: 8.6 us, 3.1 TB/s: few bytes a CTA behind the chain of
// counts, path, page and row; one branch: 2.3). Path and pages are checked at once by as
// many threads, before anything moves: 10 and 2.6 us with the pages checked at each token.
constexpr int kKeepThreads = 128, kKeepBatch = 4;

struct KeepArgs {
    PagedView p;
    uint8_t *k_pages, *v_pages;
    long long layer_bytes;   // of K, and of V
    int head_bytes;          // of one token's head
    const int32_t *path, *counts;
    int max_path;
    int32_t* lengths;
};

__global__ void __launch_bounds__(kKeepThreads) keep_tokens_kernel(const KeepArgs a) {
    const int b = blockIdx.x, count = a.counts[b];
    const SequenceSpan s = sequence_span(a.p, b);
    const int32_t* path = a.path + static_cast<long long>(b) * a.max_path;
    const int32_t* table = a.p.table + static_cast<long long>(b) * a.p.table_stride;
    auto page_of = [&](int slot) { return table[slot >> a.p.page_shift]; };
    // checked before anything moves: the path, and the pages of its nodes' places, old and new
    bool good = s.base >= 0 && count >= 0 && count <= min(s.count, a.max_path);
    if (good)
        for (int i = threadIdx.x; i < count; i += kKeepThreads) {
            const int node = path[i];
            good = node >= i && node < s.count && (i == 0 || node > path[i - 1]);
            if (!good) break;
            const int from = page_of(s.base + node), to = page_of(s.base + i);
            good = min(from, to) >= 0 && max(from, to) < a.p.pages;
            if (!good) break;
        }
    good = __syncthreads_and(good) != 0;
    if (blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0) {
        if (!good) report(kStatusBadPage);
        a.lengths[b] = good ? s.base + count : a.p.kv_lens[b];
    }
    if (!good) return;
    uint8_t* pages = (blockIdx.z ? a.v_pages : a.k_pages) + blockIdx.y * a.layer_bytes;
    const int chunks = a.head_bytes / 16, mask = (1 << a.p.page_shift) - 1;
    for (int unit = threadIdx.x; unit < a.p.kv_heads * chunks; unit += kKeepThreads) {
        const int h = unit / chunks, c = unit - h * chunks;
        auto place = [&](int slot) -> uint4* {
            const long long row = ((static_cast<long long>(page_of(slot)) * a.p.kv_heads + h) << a.p.page_shift) + (slot & mask);
            return reinterpret_cast<uint4*>(pages + row * a.head_bytes) + c;
        };
        for (int i0 = 0; i0 < count; i0 += kKeepBatch) {
            uint4 v[kKeepBatch];
            uint4* to[kKeepBatch];
#pragma unroll
            for (int k = 0; k < kKeepBatch; ++k) {
                to[k] = nullptr;
                const int i = i0 + k;
                if (i >= count || path[i] == i) continue;
                v[k] = *place(s.base + path[i]);
                to[k] = place(s.base + i);
            }
#pragma unroll
            for (int k = 0; k < kKeepBatch; ++k)
                if (to[k] != nullptr) *to[k] = v[k];
        }
    }
}

}  // namespace h4b

extern "C" long long h4b_tree_accept_workspace_bytes(int rows, int sequences) {
    if (rows < 0 || sequences < 0) return H4B_EINVAL;
    // a row has so many parts at most that all rows' are kAcceptCtas + rows
    return (4ll * sequences + 15) / 16 * 16 + 8ll * (h4b::kAcceptCtas + rows);
}

extern "C" int h4b_tree_accept(const void* logits, int logits_dtype, long long logits_stride, int vocab,
                               const int32_t* tokens, const int32_t* parents, const int32_t* q_offsets, int rows,
                               int sequences, int max_path, int32_t* targets, int32_t* path, int32_t* counts,
                               int32_t* next_tokens, void* workspace, long long workspace_bytes, void* stream) {
    using namespace h4b;
    if (rows < 0 || sequences < 0 || max_path < 1) return H4B_EINVAL;
    if (sequences == 0) return 0;
    if (!q_offsets || !path || !counts || !next_tokens || (rows > 0 && (!tokens || !parents || !targets))) return H4B_EINVAL;
    AcceptArgs a{};
    a.tokens = tokens, a.parents = parents, a.q_offsets = q_offsets, a.sequences = sequences, a.rows = rows;
    a.max_path = max_path, a.targets = targets, a.path = path, a.counts = counts, a.next_tokens = next_tokens;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (logits == nullptr) {
        accept_targets_kernel<<<sequences, kAcceptThreads, 0, s>>>(a);
        H4B_CUDA_TRY(cudaGetLastError());
        return 0;
    }
    if (logits_dtype != H4B_FP32 && logits_dtype != H4B_FP16 && logits_dtype != H4B_BF16) return H4B_EUNSUPPORTED;
    const int size = logits_dtype == H4B_FP32 ? 4 : 2;
    if (vocab < 1 || logits_stride < vocab || (reinterpret_cast<uintptr_t>(logits) & (size - 1))) return H4B_EINVAL;
    // (the parts' ends, rounded up to 16 values each, and a thread's place behind them fit 32 bits)
    if (vocab > INT_MAX - 16 * kAcceptCtas - kAcceptThreads) return H4B_EUNSUPPORTED;
    if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
        workspace_bytes < h4b_tree_accept_workspace_bytes(rows, sequences))
        return H4B_EINVAL;
    a.logits = logits, a.logits_stride = logits_stride, a.vocab = vocab;
    a.splits = rows > 0 ? accept_splits(rows, static_cast<long long>(vocab) * size) : 1;
    a.part = ((vocab + a.splits - 1) / a.splits + 15) / 16 * 16;
    a.arrived = static_cast<unsigned int*>(workspace);
    a.keys = reinterpret_cast<unsigned long long*>(static_cast<uint8_t*>(workspace) + (4ll * sequences + 15) / 16 * 16);
    if (static_cast<long long>(rows) * a.splits + 1 > INT_MAX) return H4B_EUNSUPPORTED;
    const unsigned grid = static_cast<unsigned>(rows) * a.splits + 1;
    if (logits_dtype == H4B_FP32)
        accept_logits_kernel<float><<<grid, kAcceptThreads, 0, s>>>(a);
    else if (logits_dtype == H4B_FP16)
        accept_logits_kernel<__half><<<grid, kAcceptThreads, 0, s>>>(a);
    else
        accept_logits_kernel<__nv_bfloat16><<<grid, kAcceptThreads, 0, s>>>(a);
    H4B_CUDA_TRY(cudaGetLastError());
    return 0;
}

extern "C" int h4b_tree_keep(const h4b_paged_kv* kv, int layers, long long layer_bytes, const int32_t* path, int max_path,
                             const int32_t* counts, int32_t* lengths, void* stream) {
    using namespace h4b;
    KeepArgs a{};
    if (!paged_view(kv, &a.p) || layers < 1 || max_path < 1) return H4B_EINVAL;
    if (!paged_shape_supported(kv, 0) || layers > 65535) return H4B_EUNSUPPORTED;
    const long long need = static_cast<long long>(kv->pages) * kv->kv_heads * kv->page_size * kv->head_dim * 2;
    if (layers > 1 && (layer_bytes < need || (layer_bytes & 15))) return H4B_EINVAL;
    if (kv->sequences == 0) return 0;
    if (path == nullptr || counts == nullptr || lengths == nullptr) return H4B_EINVAL;
    // (what all CTAs of a sequence read, while one of them writes lengths)
    const long long n = kv->sequences;
    const struct {
        const int32_t* at;
        long long count;
    } read[] = {{kv->kv_lens, n}, {counts, n}, {kv->q_offsets, n + 1}, {path, n * max_path}, {kv->page_table, n * kv->table_stride}};
    const uintptr_t to = reinterpret_cast<uintptr_t>(lengths);
    for (const auto& r : read) {
        const uintptr_t from = reinterpret_cast<uintptr_t>(r.at);
        if (to < from + 4ull * r.count && from < to + 4ull * n) return H4B_EINVAL;
    }
    a.k_pages = static_cast<uint8_t*>(kv->k_pages), a.v_pages = static_cast<uint8_t*>(kv->v_pages);
    a.layer_bytes = layer_bytes, a.head_bytes = kv->head_dim * 2;
    a.path = path, a.counts = counts, a.max_path = max_path, a.lengths = lengths;
    keep_tokens_kernel<<<dim3(kv->sequences, layers, 2), kKeepThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    H4B_CUDA_TRY(cudaGetLastError());
    return 0;
}
