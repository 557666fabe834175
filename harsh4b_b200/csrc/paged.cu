// Paged K/V cache: the append of new tokens, page copies, and the attention
// of few query rows a sequence (decode, short chunks). paged_tc.cu holds the
// attention of long chunks, paged_tree.cu that of drafted trees, which are here too
// where their rows are few (TREE).
//
// A layer's pages are [pages][kv_heads][page_size][head_dim] of fp16 or bf16,
// one buffer for K and one for V. Sequence b's token j lives in page
// page_table[b][j / page_size], slot j % page_size. Its new tokens are rows
// q_offsets[b] .. q_offsets[b + 1] - 1 of the batch, at positions
// kv_lens[b] - n_b + i (n_b new tokens): a token sees the keys j <= its own
// position p, with a window w only j > p - w or j < sinks.
//
// Every table is read on the device, so a captured graph follows its contents.
// Nothing a table says makes a kernel read or write out of bounds: a page id,
// an offset or a length out of range sets status bit 8 (kStatusBadPage), a
// page that is needed and out of range reads as zeros and is not written, a
// sequence with such an offset or length counts as empty.
#include <cuda_bf16.h>

#include <climits>
#include <cmath>

namespace h4b {

constexpr int kStatusBadPage = 8;  // page id, row offset or length out of range

template <typename T>
struct Pair;  // two 16-bit values of a 32-bit word
template <>
struct Pair<__half> {
    static constexpr bool kBf16 = false;
    static constexpr uint32_t kExponent = 0x7C007C00u, kExponentOne = 0x04000400u;
    __device__ static uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    __device__ static float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
};
template <>
struct Pair<__nv_bfloat16> {
    static constexpr bool kBf16 = true;
    static constexpr uint32_t kExponent = 0x7F807F80u, kExponentOne = 0x00800080u;
    __device__ static uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    __device__ static float2 unpack(uint32_t w) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    }
};

// Nonzero where one of a word's two values is an infinity or a NaN: its
// exponent, all ones, carries into the value's top bit.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    return ((w & Pair<T>::kExponent) + Pair<T>::kExponentOne) & 0x80008000u;
}

// All bits of the values that not_finite marks.
__device__ __forceinline__ uint32_t halves_of(uint32_t marks) { return (marks >> 15) * 0xffffu; }

// The batch as the kernels see it (h4b_paged_kv without its pointers' types).
struct PagedView {
    int pages, page_shift, kv_heads, sequences, table_stride, tokens;
    const int32_t* table;
    const int32_t* q_offsets;
    const int32_t* kv_lens;
};

// Rows and lengths of one sequence: as the tables have them (a load whose
// values nothing waits for yet), and made safe.
struct RawSpan {
    int first, end, len;
};
__device__ __forceinline__ RawSpan raw_span(const PagedView& p, int b) {
    return RawSpan{p.q_offsets[b], p.q_offsets[b + 1], p.kv_lens[b]};
}
constexpr int kMaxLength = 1 << 30;  // keeps position - window in 32 bits
struct SequenceSpan {
    int first, count, base;  // first row, new tokens, position of the first one
};
// Nodes of a drafted tree, at most (a row's ancestors are kept as bits). A
// sequence with more, or with more than its length, counts as out of range.
constexpr int kTreeNodes = H4B_TREE_NODES, kTreeWords = kTreeNodes / 32;
template <bool TREE = false>
__device__ __forceinline__ SequenceSpan checked_span(const PagedView& p, const RawSpan& r) {
    bool good = r.first >= 0 && r.end >= r.first && r.end <= p.tokens && r.len >= 0 &&
                r.len <= kMaxLength && r.len <= static_cast<long long>(p.table_stride) << p.page_shift;
    if constexpr (TREE) good = good && r.end - r.first <= min(kTreeNodes, r.len);
    if (!good) {
        report(kStatusBadPage);
        // its rows, as far as they exist, still get an (empty) answer
        const int lo = min(max(r.first, 0), p.tokens), hi = min(max(r.end, 0), p.tokens);
        return SequenceSpan{lo, max(hi - lo, 0), -kMaxLength};
    }
    return SequenceSpan{r.first, r.end - r.first, r.len - (r.end - r.first)};
}
template <bool TREE = false>
__device__ __forceinline__ SequenceSpan sequence_span(const PagedView& p, int b) {
    return checked_span<TREE>(p, raw_span(p, b));
}

// A drafted tree: parents[first + i] is node i's parent within its sequence,
// -1 where the node follows the tokens before the tree, and less than i. One
// that is not counts as -1 and sets status bit 8, so every walk ends.
__device__ __forceinline__ int checked_parent(int parent, int node) {
    if (parent >= -1 && parent < node) return parent;
    report(kStatusBadPage);
    return -1;
}
// Parent by parent up to the root: node `i`'s depth, and in `sight` (kTreeWords
// words) the nodes that it sees, itself among them: with a window those less than
// `window` above it, or at positions below `sinks`.
__device__ __forceinline__ int walk_tree(const int32_t* parents, int i, int base, int window, int sinks, uint32_t* sight) {
    int depth = 0;
    for (int j = checked_parent(parents[i], i); j >= 0; j = checked_parent(parents[j], j)) ++depth;
#pragma unroll
    for (int w = 0; w < kTreeWords; ++w) sight[w] = 0u;
    int up = 0;
    for (int j = i; j >= 0; j = checked_parent(parents[j], j), ++up)
        if (window <= 0 || up < window || base + depth - up < sinks) sight[j >> 5] |= 1u << (j & 31);
    return depth;
}
// By a whole warp, for 32 consecutive nodes from `first` on (parent: this lane's, of
// node first + lane, -1 past the last): the nodes of these that the lane's node
// descends from, as bits, and the parent of the topmost of them (an earlier node,
// or -1). By doubling the step: a node's set joins that of the node its step leads
// to, so a chain takes no longer than a bush.
__device__ __forceinline__ uint32_t descent(int parent, int first, int* above) {
    const int lane = threadIdx.x & 31;
    uint32_t set = 1u << lane;
    int to = parent >= first ? parent & 31 : lane;  // where the step leads: itself at the top
#pragma unroll
    for (int r = 0; r < 5; ++r) {
        set |= __shfl_sync(0xffffffffu, set, to);
        to = __shfl_sync(0xffffffffu, to, to);
    }
    *above = __shfl_sync(0xffffffffu, parent, to);
    return set;
}
// Node `i`'s depth, by a whole warp.
__device__ __forceinline__ int node_depth(const int32_t* parents, int i) {
    const int lane = threadIdx.x & 31;
    int depth = -1;
    while (i >= 0) {
        const int first = i & ~31, j = first + lane;
        int above;
        const uint32_t set = descent(j <= i ? checked_parent(parents[j], j) : -1, first, &above);
        depth += __popc(__shfl_sync(0xffffffffu, set, i & 31));
        i = __shfl_sync(0xffffffffu, above, i & 31);
    }
    return depth;
}

// ---- append ---------------------------------------------------------------
// One warp per (token, head) in steps: q and k heads are divided by their
// root mean square and scaled (norm weights), then rotated (cos/sin rows of
// the token's position, halves d and d + D/2 paired); v passes through. One
// rounding to 16 bits at the end, everything before in fp32. A head takes D/8
// lanes: lane i holds dims 4i .. 4i + 3 and their partners D/2 further, so the
// rotation needs no exchange.
// Bound by HBM: (heads + 2 kv_heads) D (source + 2) bytes a token (8192 tokens
// of 48 heads of 128 from fp32: 52 to 55 us, 5.6 to 5.9 TB/s; from fp16 45);
// a decode step by its chain of lookups (64 tokens: 3 us).
// A tree's node (TREE) goes to its place and is rotated by its depth (6200 nodes of 48
// heads of 128 from fp32: 43 us, 5.3 TB/s).
struct AppendArgs {
    PagedView p;
    const void* qkv;
    long long qkv_stride;   // values from token to token
    const float *norm_q, *norm_k, *cos, *sin;
    int max_pos, heads;
    unsigned parts;         // warps that share a token
    float eps;
    void *q_out, *k_pages, *v_pages;
    long long q_stride;
    const int32_t* parents;  // of a tree's nodes, or null
};

// Warps that share a token of a long chunk, and turns a warp has in flight
// (8192 tokens, 48 heads of 128, fp32: 8 and 1 58 us, 4 and 2 53, 2 and 3 52;
// 10 heads 16, 18 and 15).
constexpr int kAppendWarps = 8, kAppendShare = 2, kAppendTurns = 3;

// Four consecutive values, of 2 or 4 bytes, as they come.
template <typename S>
struct RawQuad {
    using type = uint2;
    __device__ static float4 value(uint2 w) {
        const float2 a = Pair<S>::unpack(w.x), b = Pair<S>::unpack(w.y);
        return make_float4(a.x, a.y, b.x, b.y);
    }
};
template <>
struct RawQuad<float> {
    using type = float4;
    __device__ static float4 value(float4 w) { return w; }
};
__device__ __forceinline__ float4 scaled(const float4& v, float f, const float4& w) {
    return make_float4(v.x * f * w.x, v.y * f * w.y, v.z * f * w.z, v.w * f * w.w);
}
// a c + b s, four at a time.
__device__ __forceinline__ float4 turned(const float4& a, const float4& c, const float4& b, const float4& s) {
    return make_float4(a.x * c.x + b.x * s.x, a.y * c.y + b.y * s.y, a.z * c.z + b.z * s.z, a.w * c.w + b.w * s.w);
}

template <typename S, typename T, int D, bool TREE>
__global__ void __launch_bounds__(32 * kAppendWarps) paged_append_kernel(const AppendArgs a) {
    using Raw = typename RawQuad<S>::type;
    constexpr int kLanes = D / 8, kPerWarp = 32 / kLanes;  // heads a warp holds in its lanes
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int page_size = 1 << a.p.page_shift;
    const int i = lane % kLanes, sub = lane / kLanes;
    // warp `part` of the `parts` that share a token
    const unsigned place = blockIdx.x * kAppendWarps + warp;
    const int token = static_cast<int>(place / a.parts), part = static_cast<int>(place % a.parts);
    if (token >= a.p.tokens) return;
    const int total = a.heads + 2 * a.p.kv_heads, stride = a.parts * kPerWarp;
    const S* row = static_cast<const S*>(a.qkv) + token * a.qkv_stride + 4 * i;
    T* q_row = static_cast<T*>(a.q_out) + token * a.q_stride + 4 * i;

    // the first heads are on their way while the token's place is looked up
    int h0 = part * kPerWarp + sub;
    Raw x[kAppendTurns], y[kAppendTurns];
    auto load = [&]() {
#pragma unroll
        for (int k = 0; k < kAppendTurns; ++k) {
            const int h = min(h0 + k * stride, total - 1);  // (a head too many is read and not used)
            x[k] = __ldcs(reinterpret_cast<const Raw*>(row + h * D));
            y[k] = __ldcs(reinterpret_cast<const Raw*>(row + h * D + D / 2));
        }
    };
    load();

    // the token's sequence: the last b whose offset is not past the token
    int b = -1;
    for (int j = 0; j < a.p.sequences; j += 32) {
        const bool before = j + lane < a.p.sequences && a.p.q_offsets[j + lane] <= token;
        b += __popc(__ballot_sync(0xffffffffu, before));
    }
    T *k_row = nullptr, *v_row = nullptr;  // of the token, kv head 0
    int position = -1;  // its place in the cache, and below its position
    int depth = -1;     // of a tree's node, less its index
    if (b >= 0) {
        const SequenceSpan s = sequence_span<TREE>(a.p, b);
        position = token < s.first + s.count ? s.base + token - s.first : -1;
        if constexpr (TREE)
            if (position >= 0) depth = node_depth(a.parents + s.first, token - s.first) - (token - s.first);
        if (position >= 0) {
            const int page = a.p.table[static_cast<long long>(b) * a.p.table_stride + (position >> a.p.page_shift)];
            if (page >= 0 && page < a.p.pages) {
                const long long at = ((static_cast<long long>(page) * a.p.kv_heads << a.p.page_shift) +
                                      (position & (page_size - 1))) * D + 4 * i;
                k_row = static_cast<T*>(a.k_pages) + at;
                v_row = static_cast<T*>(a.v_pages) + at;
            } else if (lane == 0) {
                report(kStatusBadPage);
            }
        }
    }
    if constexpr (TREE) position = position >= 0 ? position + depth : -1;
    // (not by an angle of zero where there is none: that would add 0 times the
    // partner, which need not be finite)
    float4 cos{}, sin{};
    const bool rotated = a.cos != nullptr && position >= 0 && position < a.max_pos;
    if (a.cos != nullptr && position >= 0) {
        if (rotated) {
            cos = __ldg(reinterpret_cast<const float4*>(a.cos + static_cast<long long>(position) * (D / 2)) + i);
            sin = __ldg(reinterpret_cast<const float4*>(a.sin + static_cast<long long>(position) * (D / 2)) + i);
        } else if (lane == 0) {
            report(kStatusBadPosition);
        }
    }
    const float4 minus = make_float4(-sin.x, -sin.y, -sin.z, -sin.w);
    const bool normed = a.norm_q != nullptr;
    while (true) {  // (the same number of turns in every lane)
#pragma unroll
        for (int k = 0; k < kAppendTurns; ++k) {
            const int h = h0 + k * stride;
            const bool is_v = h >= a.heads + a.p.kv_heads, is_q = h < a.heads;
            float4 u = RawQuad<S>::value(x[k]), w = RawQuad<S>::value(y[k]);
            if (normed) {
                float sum = (u.x * u.x + u.y * u.y) + (u.z * u.z + u.w * u.w) + (w.x * w.x + w.y * w.y) +
                            (w.z * w.z + w.w * w.w);
#pragma unroll
                for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (!is_v) {
                    const float inv = rsqrtf(sum * (1.0f / D) + a.eps);  // to 2 ulp; the result has 16 bits
                    const float4* weight = reinterpret_cast<const float4*>(is_q ? a.norm_q : a.norm_k) + i;
                    u = scaled(u, inv, __ldg(weight));
                    w = scaled(w, inv, __ldg(weight + kLanes));
                }
            }
            if (!is_v && rotated) {
                const float4 t = u;
                u = turned(t, cos, w, minus);
                w = turned(w, cos, t, sin);
            }
            T* dst = nullptr;
            if (is_q)
                dst = q_row + h * D;
            else if (k_row != nullptr && h < total)
                dst = is_v ? v_row + ((h - a.heads - a.p.kv_heads) << a.p.page_shift) * D
                           : k_row + ((h - a.heads) << a.p.page_shift) * D;
            if (dst != nullptr) {
                *reinterpret_cast<uint2*>(dst) = make_uint2(Pair<T>::pack(u.x, u.y), Pair<T>::pack(u.z, u.w));
                *reinterpret_cast<uint2*>(dst + D / 2) = make_uint2(Pair<T>::pack(w.x, w.y), Pair<T>::pack(w.z, w.w));
            }
        }
        h0 += kAppendTurns * stride;
        if (h0 - sub >= total) break;
        load();
    }
}

// ---- page copies ------------------------------------------------------------
// Page dst[i] <- page src[i] in every layer, K and V: one CTA moves up to
// kCopyBytes of one (layer, K or V, move), every thread with all its 16-byte
// loads in flight before its first store. Bound by HBM: twice the page bytes
// (400 pages of 32 KB in 36 layers, K and V: 286 us, 6.6 TB/s).
constexpr int kCopyThreads = 256, kCopyUnroll = 8, kCopyBytes = kCopyThreads * kCopyUnroll * 16;

__global__ void __launch_bounds__(kCopyThreads)
    pages_copy_kernel(uint8_t* k_pages, uint8_t* v_pages, int pages, long long page_bytes, int parts,
                      const int32_t* src, const int32_t* dst) {
    const int move = blockIdx.x / parts, part = blockIdx.x % parts;
    const int from = src[move], to = dst[move];
    if (from < 0 || from >= pages || to < 0 || to >= pages) {
        if (threadIdx.x == 0) report(kStatusBadPage);
        return;
    }
    uint8_t* base = (blockIdx.z ? v_pages : k_pages) + static_cast<long long>(blockIdx.y) * pages * page_bytes;
    const uint4* s = reinterpret_cast<const uint4*>(base + from * page_bytes);
    uint4* d = reinterpret_cast<uint4*>(base + to * page_bytes);
    const long long words = page_bytes / 16, first = static_cast<long long>(part) * (kCopyBytes / 16) + threadIdx.x;
    uint4 v[kCopyUnroll];
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
        if (first + u * kCopyThreads < words) v[u] = __ldcs(s + first + u * kCopyThreads);
#pragma unroll
    for (int u = 0; u < kCopyUnroll; ++u)
        if (first + u * kCopyThreads < words) __stcs(d + first + u * kCopyThreads, v[u]);
}

// ---- attention: the split of the work ------------------------------------------
// An item is (sequence, tile of ROWS / group new tokens, kv head): its query
// rows r = (token i, q head j of the group), r = i * group + j, share the
// item's keys. A unit is one block of KEYS keys of an item, from the blocks
// that some row of it sees: the sink blocks [0, sink_blocks) and then
// [low, high); an item has one unit at least, so that every row is answered.
// All items in order (sequence, tile, kv head) are laid out on a line, `extra`
// places for what an item costs beside its units and then one place a unit,
// and the line is cut into one equal contiguous range per CTA, whatever the
// lengths. A cut among an item's first places counts as one before its first
// unit. An item that lies across CTAs leaves one partial result (o, m, l) in
// each; they are joined in the order of the CTAs, by the CTA that finishes last
// (few rows) or by a kernel of its own (long chunks), so the same bits come out
// every time.
struct AttendArgs {
    PagedView p;
    int fewest, most;         // sequences with so many new tokens are this kernel's
    int extra;                // places of an item beside its units
    int least;                // places of a CTA's range, where there are few
    const void *q, *k_pages, *v_pages;
    void* out;
    float* lse;               // may be null
    long long q_stride, out_stride;
    int heads, group, window, sinks;
    float scale;              // of a score in base-2 units: scale * log2(e)
    float* partials;          // [2 * CTAs][ROWS * (D + 2)]: a CTA's first and last item
    unsigned int* counters;   // [CTAs], zero between calls (few-row kernel)
    int4* entries;            // [CTAs] the item that begins last in each (chunk kernel)
    int half_tokens;          // new tokens of each of an item's tiles (chunk kernel: two, tree kernel: one or two)
    const int32_t* parents;   // of a tree's nodes (TREE)
    bool whole;               // items are not cut: one is the CTA's whose range holds its first unit (TREE)
};

// A sequence as this kernel's share of the batch has it: without new tokens if
// it is another kernel's.
template <bool TREE>
__device__ __forceinline__ SequenceSpan own_span(const AttendArgs& a, const RawSpan& r) {
    SequenceSpan s = checked_span<TREE>(a.p, r);
    if (s.count < a.fewest || s.count > a.most) s.count = 0;
    return s;
}

// Of a tree (TREE) the new tokens lie at base .. base + count - 1 too, but a
// row sees of these its ancestors and itself only, and stands at its depth.
struct Tile {  // one tile of new tokens of a sequence
    int first, tokens;        // first row (token index in the batch), tokens
    int p0, p1;               // positions of its first and last token (TREE: base, place of its last node)
    int low, high, sink_blocks;
    __device__ __forceinline__ int units() const { return high - low + sink_blocks; }
    __device__ __forceinline__ int block(int unit) const {
        return unit < sink_blocks ? unit : low + unit - sink_blocks;
    }
};

template <int KEYS, bool TREE>
__device__ __forceinline__ Tile make_tile(const SequenceSpan& s, int t, int tile_tokens, int window, int sinks) {
    Tile x;
    x.first = s.first + t * tile_tokens;
    x.tokens = min(tile_tokens, s.count - t * tile_tokens);
    x.p0 = TREE ? s.base : s.base + t * tile_tokens;
    x.p1 = s.base + t * tile_tokens + x.tokens - 1;
    const int end = max(x.p1 + 1, 0);
    const int from = window > 0 ? max(x.p0 - window + 1, 0) : 0;
    x.high = max((end + KEYS - 1) / KEYS, 1);
    x.low = min(from / KEYS, x.high - 1);
    x.sink_blocks = window > 0 ? min((min(sinks, end) + KEYS - 1) / KEYS, x.low) : 0;
    return x;
}

template <int KEYS, bool TREE>
__device__ __forceinline__ int item_places(const AttendArgs& a, const SequenceSpan& s, int t, int tile_tokens) {
    return a.extra + make_tile<KEYS, TREE>(s, t, tile_tokens, a.window, a.sinks).units();
}

// Places of one kv head of every lane's sequence. The whole warp takes part: a
// lane sums a few tiles by itself, a long chunk's are summed by all lanes.
template <int KEYS, bool TREE>
__device__ __forceinline__ long long warp_places(const AttendArgs& a, const SequenceSpan& s, int tile_tokens) {
    const int lane = threadIdx.x & 31;
    long long n = 0;
    const bool is_long = s.count > 4 * tile_tokens;
    if (!is_long)
        for (int t = 0; t * tile_tokens < s.count; ++t) n += item_places<KEYS, TREE>(a, s, t, tile_tokens);
    for (unsigned todo = __ballot_sync(0xffffffffu, is_long); todo; todo &= todo - 1) {
        const int who = __ffs(todo) - 1;
        const SequenceSpan x{__shfl_sync(0xffffffffu, s.first, who), __shfl_sync(0xffffffffu, s.count, who),
                             __shfl_sync(0xffffffffu, s.base, who)};
        long long sum = 0;
        for (int t = lane; static_cast<long long>(t) * tile_tokens < x.count; t += 32)
            sum += item_places<KEYS, TREE>(a, x, t, tile_tokens);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == who) n = sum;
    }
    return n;
}

// The CTA's range of places and where it starts.
struct Range {
    long long begin, end, total;  // [begin, end) of total
    long long skip;               // places of its sequence before `begin`
    int sequence;                 // of place `begin`
    int ctas;                     // that have a range: every one of them has a place at least
    SequenceSpan span;            // of that sequence (trees only: the others look it up)
};
// n / d of numbers that are not negative, with SHORT in 32 bits where they fit: a
// 64-bit division is a long piece of code, and what runs once a launch runs cold (a
// tree's items take many roles' warps to their start).
template <bool SHORT>
__device__ __forceinline__ long long quotient(long long n, long long d) {
    if (SHORT && ((n | d) >> 32) == 0) return static_cast<uint32_t>(n) / static_cast<uint32_t>(d);
    return n / d;
}
template <bool SHORT>
__device__ __forceinline__ long long range_begin(long long total, int cta, int ctas) { return quotient<SHORT>(total * cta, ctas); }
// The CTA that holds a place: the largest c with range_begin(c) <= place.
template <bool SHORT>
__device__ __forceinline__ int range_owner(long long total, long long place, int ctas) {
    return static_cast<int>(quotient<SHORT>((place + 1) * ctas - 1, total));
}

// Every thread of the CTA takes part; `shared` holds THREADS / 32 long longs
// and a Range. Each thread has a share of the sequences, a prefix sum over
// the threads follows, and the thread whose sequences hold place `begin`
// finds it.
template <int THREADS, int KEYS, bool TREE = false>
__device__ __forceinline__ Range find_range(const AttendArgs& a, int tile_tokens, void* shared) {
    long long* warp_sums = static_cast<long long*>(shared);
    Range* found = reinterpret_cast<Range*>(warp_sums + THREADS / 32);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int each = (a.p.sequences + THREADS - 1) / THREADS, b0 = threadIdx.x * each;
    SequenceSpan s{0, 0, 0};
    auto places_of = [&](int e) {  // of the thread's e-th sequence, all kv heads
        s = SequenceSpan{0, 0, 0};
        if (b0 + e < a.p.sequences) s = own_span<TREE>(a, raw_span(a.p, b0 + e));
        return a.p.kv_heads * warp_places<KEYS, TREE>(a, s, tile_tokens);
    };
    long long mine = 0;
    for (int e = 0; e < each; ++e) mine += places_of(e);
    long long before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += up;
    }
    if (lane == 31) warp_sums[warp] = before;
    __syncthreads();
    long long total = 0;
    before -= mine;
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += warp_sums[w];
        total += warp_sums[w];
    }
    Range r;
    r.total = total;
    r.ctas = static_cast<int>(min(static_cast<long long>(gridDim.x), (total + a.least - 1) / a.least));
    r.begin = r.end = 0;
    if (static_cast<int>(blockIdx.x) < r.ctas) {
        r.begin = range_begin<TREE>(total, blockIdx.x, r.ctas);
        r.end = range_begin<TREE>(total, blockIdx.x + 1, r.ctas);
    }
    const bool here = r.begin < r.end && r.begin >= before && r.begin < before + mine;
    if (__any_sync(0xffffffffu, here)) {
        long long at = before;
        bool open = here;
        for (int e = 0; e < each; ++e) {
            const long long n = each == 1 ? mine : places_of(e);
            if (open && r.begin < at + n) {
                found->sequence = b0 + e;
                found->skip = r.begin - at;
                if constexpr (TREE) found->span = s;
                open = false;
            }
            at += n;
        }
    }
    __syncthreads();
    if (r.begin < r.end) {
        r.sequence = found->sequence;
        r.skip = found->skip;
        if constexpr (TREE) r.span = found->span;
    }
    return r;
}

// A walk over the CTA's units, item by item.
template <int KEYS, bool TREE = false>
struct Walk {
    SequenceSpan span;
    RawSpan following;        // of sequence b + 1, requested when b was entered
    Tile tile;
    int b, t, h, unit;        // unit within the item
    int left;                 // places of the range from this unit on (of a whole item, its units at least)

    __device__ __forceinline__ void request(const AttendArgs& a) {
        if (b + 1 < a.p.sequences) following = raw_span(a.p, b + 1);
    }
    // By whole warps: the lanes look for the tile together, 32 at a time.
    // False when the range holds no unit.
    __device__ __forceinline__ bool start(const AttendArgs& a, const Range& r, int tile_tokens) {
        const int lane = threadIdx.x & 31;
        b = r.sequence;
        left = static_cast<int>(min(r.end - r.begin, static_cast<long long>(INT_MAX)));
        if constexpr (TREE)
            span = r.span;
        else
            span = own_span<TREE>(a, raw_span(a.p, b));
        request(a);
        long long skip = r.skip;
        for (int t0 = 0;; t0 += 32) {
            long long n = 0;
            if (static_cast<long long>(t0 + lane) * tile_tokens < span.count)
                n = item_places<KEYS, TREE>(a, span, t0 + lane, tile_tokens) * static_cast<long long>(a.p.kv_heads);
            long long upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long up = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += up;
            }
            const unsigned past = __ballot_sync(0xffffffffu, skip < upto);
            if (past) {
                const int who = __ffs(past) - 1;
                t = t0 + who;
                skip -= __shfl_sync(0xffffffffu, upto - n, who);
                break;
            }
            skip -= __shfl_sync(0xffffffffu, upto, 31);
        }
        tile = make_tile<KEYS, TREE>(span, t, tile_tokens, a.window, a.sinks);
        const int places = a.extra + tile.units();
        h = static_cast<int>(quotient<TREE>(skip, places));
        unit = static_cast<int>(skip - static_cast<long long>(h) * places) - a.extra;
        if (unit < 0) {
            left += unit;
            unit = 0;
        }
        if (TREE && a.whole && unit > 0) {  // begun in an earlier range
            left -= tile.units() - unit + a.extra;
            if (left <= 0) return false;
            next_item(a, tile_tokens);
        }
        const bool any = left > 0;
        if (TREE && a.whole) left = max(left, tile.units());
        return any;
    }
    // Past the item's last unit: to the next item that has any.
    __device__ __forceinline__ void next_item(const AttendArgs& a, int tile_tokens) {
        unit = 0;
        if (++h < a.p.kv_heads) return;
        h = 0;
        ++t;
        while (t * tile_tokens >= span.count) {
            t = 0;
            ++b;
            span = own_span<TREE>(a, following);
            request(a);
        }
        tile = make_tile<KEYS, TREE>(span, t, tile_tokens, a.window, a.sinks);
    }
    __device__ __forceinline__ bool item_ends() const { return unit + 1 >= tile.units(); }
    // Whether this unit is the last of the range.
    __device__ __forceinline__ bool range_ends(const AttendArgs& a) const { return left <= (item_ends() ? 1 + a.extra : 1); }
    // Whether this unit is the last of the item in this range, or of all.
    __device__ __forceinline__ bool part_ends() const { return item_ends() || left <= 1; }
    // To the next unit; false past the range's end.
    __device__ __forceinline__ bool next(const AttendArgs& a, int tile_tokens) {
        const bool over = item_ends();
        left -= over ? 1 + a.extra : 1;
        if (left <= 0) return false;
        if (over) {
            next_item(a, tile_tokens);
            if (TREE && a.whole) left = max(left, tile.units());
        } else {
            ++unit;
        }
        return true;
    }
};

// The CTAs that hold units of an item, given one of its units (walk state of
// the CTA of `range`): from its first unit's to its last's.
template <int KEYS, bool TREE>
__device__ __forceinline__ int2 item_owners(const Range& range, const Walk<KEYS, TREE>& w) {
    const long long first = range.end - w.left - w.unit;
    return make_int2(range_owner<TREE>(range.total, first, range.ctas),
                     range_owner<TREE>(range.total, first + w.tile.units() - 1, range.ctas));
}

// Whether some row of the tile sees key j.
__device__ __forceinline__ bool tile_sees(const Tile& t, int window, int sinks, int j) {
    return j <= t.p1 && (window <= 0 || j > t.p0 - window || j < sinks);
}

// ---- attention of few rows -----------------------------------------------------
// For decode and short chunks the keys are read once and each takes part in
// few products, so HBM is the bound: 4 D kv_heads bytes a key (32 sequences of
// 32768 tokens, 8 kv heads of 128: 615 to 646 us, 6.6 to 7.0 TB/s; 64 ragged ones
// up to 2100: 64 us, 5.3 TB/s, of which 6 pass before the first keys arrive). The products
// run on mma.sync (m16n8k16): its 16 rows hold the item's rows, and its
// operands come from shared memory without the tensor-memory allocation, the
// MMA-issuing thread and the 128-row tiles that tcgen05 asks for.
//
// A CTA has four warps, a unit is 64 keys: each warp takes 16 of them, a
// 16-key piece of one page (page sizes are multiples of 16), with a ring of
// its own in shared memory fed by its own 16-byte asynchronous copies. So no
// barrier is needed between the loads and the products: a warp waits for its
// own copies only, and the ring runs on over the item boundaries. Each warp
// keeps its own (o, m, l); at an item's end (or the range's) the warps join
// theirs through shared memory.
// Softmax in base 2: p = 2^(s - m) with m 8 below a score that was the largest
// (so that small p keep clear of fp16's subnormals); m moves only when a score
// passes it by 15 (2^15 fits fp16). Where a score's unit is more than 1, m is
// the score itself: 8 less might round to more than 15 less.
// l is summed from the fp32 p, which is rounded to 16 bits for the p v
// products only: the tensor cores take both operands in the cache's type, and a
// second product for the rest of p costs 3 to 4 % (646 -> 674 us for the 32 x
// 32768 tokens, 64.6 -> 66.3 for the 64 ragged ones: the instruction count shows
// under the power cap). The rounding is to 2^-12 of a weight (bf16 2^-9), independent
// from key to key, so its part of a sum is below the result's own rounding: the
// error against 64 bits is 2.2 to 2.9e-4 in fp16, 2.2 to 2.3e-3 in bf16, with
// fp32 weights 2.1e-4 and 1.7e-3. (Trees of 2 nodes: 64 ragged ones 52.5 -> 53.6 us, 16
// over 32768 tokens 328 -> 346 under the cap, one over 1000 the same.) Keys that no row sees are zero-filled by the copy, so what
// such a slot holds cannot reach a sum. Keys that some rows see have weight 0
// in the others, and 0 times an infinity or NaN would reach those: a piece
// with such a key is searched for them (only where a tile has several tokens,
// at their own positions and at the window's edge); those found are added to
// the rows that see them and taken out of the piece before its product.
constexpr int kFewWarps = 4, kFewThreads = 32 * kFewWarps, kFewKeys = 64;
constexpr int kFewExtra = 2;  // an item's start and join, in units (1: up to 5 % slower, 3 and 4: within 3 %)
constexpr int kFewLeast = 1;  // a part is 4 KB beside 32 KB of keys
constexpr float kMostExponent = 15.f;
__device__ __forceinline__ float softmax_reference(float top) { return fabsf(top) < 16777216.f ? top - 8.f : top; }

template <int D, int ROWS>
struct FewCfg {
    static constexpr int kTiles = ROWS <= 16 ? 1 : ROWS / 16;  // m16 tiles
    static constexpr int kHalves = ROWS == 8 ? 1 : 2;          // 8-row halves of an m16 tile in use
    static constexpr int kPiece = 16 * D * 2;                  // bytes of 16 keys, K or V
    static constexpr int kStages = (ROWS <= 16 ? 3 : 2) * (128 / D);
    static constexpr int kRing = kFewWarps * kStages * 2 * kPiece;
    static constexpr int kJoin = (ROWS < 16 ? 16 : ROWS) * D * 4;  // one warp's o
    static constexpr int kJoinOff = kRing;
    static constexpr int kStatOff = kJoinOff + 2 * kJoin;
    static constexpr int kSmem = kStatOff + 2 * (ROWS < 16 ? 16 : ROWS) * 2 * 4 + 256;
    // of a tree's tile: the nodes that each of its nodes sees, and its position
    static constexpr int kSightOff = kStatOff + 2 * (ROWS < 16 ? 16 : ROWS) * 2 * 4;
    static constexpr int kTreeSmem = kSightOff + ROWS * (kTreeWords + 1) * 4;
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 bytes global -> shared; with `fill` zeros instead and no read.
__device__ __forceinline__ void async_copy16_or_zero(uint32_t dst, const void* src, bool fill) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(fill ? 0 : 16)
                 : "memory");
}

__device__ __forceinline__ void async_copy16_l2(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Byte of 16-byte chunk c of row r in a 16-row piece: the chunks of eight
// consecutive rows lie in distinct banks.
template <int D>
__device__ __forceinline__ uint32_t piece_at(int r, int c) {
    return static_cast<uint32_t>(r * (D * 2) + ((c ^ (r & 7)) * 16));
}

template <typename T, int D, int ROWS, bool TREE>
__global__ void __launch_bounds__(kFewThreads, 2) paged_attention_few_kernel(const AttendArgs a) {
    using C = FewCfg<D, ROWS>;
    constexpr int kSteps = D / 16, kCols = D / 8;
    extern __shared__ __align__(128) uint8_t few_smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tile_tokens = ROWS / a.group;
    const Range range = find_range<kFewThreads, kFewKeys, TREE>(a, tile_tokens, few_smem + C::kStatOff);
    if (range.begin >= range.end) return;
    __syncthreads();  // the range's scratch is reused below

    const uint32_t ring = smem_addr(few_smem) + warp * C::kStages * 2 * C::kPiece;
    const long long head_rows = 1ll << a.p.page_shift;  // rows of one head of a page
    const int page_mask = (1 << a.p.page_shift) - 1;

    // Page of the walk's piece: -1 when no row sees any key of it.
    auto page_of = [&](const Walk<kFewKeys, TREE>& w) -> int {
        const int key = w.tile.block(w.unit) * kFewKeys + warp * 16;
        const Tile& t = w.tile;
        const bool seen = key <= t.p1 && (a.window <= 0 || key + 15 > t.p0 - a.window || key < a.sinks);
        if (!seen) return -1;
        const int page = a.p.table[static_cast<long long>(w.b) * a.p.table_stride + (key >> a.p.page_shift)];
        if (page < 0 || page >= a.p.pages) {
            if (lane == 0) report(kStatusBadPage);
            return -2;  // needed, but nowhere: reads as zeros
        }
        return page;
    };
    // A lane copies chunk c of rows r0, r0 + kRowsStep, ..: byte `to` of row r0,
    // the others by constants (piece_at's exclusive or is linear in the row).
    constexpr int kChunks = D / 8, kRowsStep = 32 / kChunks;  // 16-byte chunks a row, rows a pass
    const int r0 = lane / kChunks;
    const uint32_t from = r0 * D + (lane % kChunks) * 8, to = piece_at<D>(r0, lane % kChunks);
    auto load = [&](const Walk<kFewKeys, TREE>& w, int page, int stage) {
        if (page == -1) return;
        const int key = w.tile.block(w.unit) * kFewKeys + warp * 16;
        const long long row = (static_cast<long long>(max(page, 0)) * a.p.kv_heads + w.h) * head_rows + (key & page_mask);
        const uint32_t dst = ring + stage * 2 * C::kPiece;
        const T* k = static_cast<const T*>(a.k_pages) + row * D + from;
        const T* v = static_cast<const T*>(a.v_pages) + row * D + from;
        if (page >= 0 && key + 15 <= w.tile.p1 &&
            (a.window <= 0 || key > w.tile.p0 - a.window || key + 15 < a.sinks)) {  // the usual: some row sees every key
#pragma unroll
            for (int r = 0; r < 16; r += kRowsStep) {
                const uint32_t at = dst + (to ^ ((r & 7) << 4)) + r * (D * 2);
                async_copy16_l2(at, k + r * D);
                async_copy16_l2(at + C::kPiece, v + r * D);
            }
        } else {
#pragma unroll 1
            for (int r = 0; r < 16; r += kRowsStep) {
                const bool fill = page < 0 || !tile_sees(w.tile, a.window, a.sinks, key + r + r0);
                const uint32_t at = dst + (to ^ ((r & 7) << 4)) + r * (D * 2);
                async_copy16_or_zero(at, k + r * D, fill);
                async_copy16_or_zero(at + C::kPiece, v + r * D, fill);
            }
        }
    };
    // ldmatrix addresses within a piece, for the first 16 dims (K), 16 dims (V):
    // K keys 0-7 and 8-15 of two chunks; V the same keys, transposed
    const uint32_t k_at = piece_at<D>((lane >> 4) * 8 + (lane & 7), (lane >> 3) & 1);
    const uint32_t v_at = piece_at<D>(((lane >> 3) & 1) * 8 + (lane & 7), lane >> 4);

    Walk<kFewKeys, TREE> now, ahead;
    if (!now.start(a, range, tile_tokens)) return;
    ahead = now;
    // the ring's first stages; `page` belongs to the piece `ahead` stands at, and
    // `live` says which of the ring's pieces, from the current one on, some row sees
    int page = page_of(ahead);
    bool more = true;
    uint32_t live = 0;
#pragma unroll 1
    for (int s = 0; s < C::kStages - 1; ++s) {
        if (more) {
            load(ahead, page, s);
            live |= (page != -1 ? 1u : 0u) << s;
            more = ahead.next(a, tile_tokens);
            if (more) page = page_of(ahead);
        }
        async_copy_commit();
    }

    uint32_t qf[C::kTiles][kSteps][4];
    float o[C::kTiles][kCols][4];
    float m[C::kTiles][2], l[C::kTiles][2];
    int pos[C::kTiles][2];
    int stage = 0;
    bool begun = now.unit == 0;  // the item's first unit is in this range
    bool fresh = true;
    uint32_t* sight = reinterpret_cast<uint32_t*>(few_smem + C::kSightOff);  // [tile tokens][kTreeWords], then positions
    int sight_b = -1, sight_t = 0;  // the tile that it holds
    while (true) {
        if (fresh) {  // a new item: its q fragments and empty sums
            fresh = false;
            if constexpr (TREE) {
                if (now.b != sight_b || now.t != sight_t) {  // (the same for every kv head; all warps are at the same item)
                    sight_b = now.b, sight_t = now.t;
                    const int i = threadIdx.x;
                    if (i < now.tile.tokens) {
                        const int node = now.tile.first - now.span.first + i;
                        const bool some = now.span.base >= 0;  // else the sequence counts as empty
                        const int depth = some ? walk_tree(a.parents + now.span.first, node, now.span.base, a.window, a.sinks,
                                                           sight + i * kTreeWords)
                                               : 0;
                        sight[ROWS * kTreeWords + i] = some ? now.span.base + depth : -1;
                    }
                    __syncthreads();
                }
            }
#pragma unroll
            for (int mt = 0; mt < C::kTiles; ++mt) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int r = mt * 16 + half * 8 + lane / 4;
                    const int i = r / a.group;
                    const bool valid = (half < C::kHalves) && i < now.tile.tokens;
                    if constexpr (TREE)
                        pos[mt][half] = valid ? static_cast<int>(sight[ROWS * kTreeWords + i]) : -1;
                    else
                        pos[mt][half] = valid ? now.tile.p0 + i : -1;
                    m[mt][half] = -INFINITY;
                    l[mt][half] = 0.f;
                    const T* q = static_cast<const T*>(a.q) + (now.tile.first + (valid ? i : 0)) * a.q_stride +
                                 (now.h * a.group + (valid ? r - i * a.group : 0)) * D + (lane & 3) * 2;
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        qf[mt][k][half] = valid ? *reinterpret_cast<const uint32_t*>(q + k * 16) : 0u;
                        qf[mt][k][2 + half] = valid ? *reinterpret_cast<const uint32_t*>(q + k * 16 + 8) : 0u;
                    }
                }
#pragma unroll
                for (int n = 0; n < kCols; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[mt][n][e] = 0.f;
            }
        }
        // Whether the row of m16 tile mt, half `half` sees key j (of those up to the tile's last).
        auto sees = [&](int mt, int half, int j) {
            const int p = pos[mt][half];
            if constexpr (TREE) {
                const int node = j - now.tile.p0;
                if (node >= 0) {
                    const int i = (mt * 16 + half * 8 + lane / 4) / a.group;
                    return p >= 0 && j <= now.tile.p1 && ((sight[i * kTreeWords + (node >> 5)] >> (node & 31)) & 1u) != 0u;
                }
            }
            return !(j > p || (a.window > 0 && j <= p - a.window && j >= a.sinks));
        };
        async_copy_wait_prior<C::kStages - 2>();
        __syncwarp();
        if (live & 1u) {
            const uint32_t kbase = ring + stage * 2 * C::kPiece, vbase = kbase + C::kPiece;
            float s[C::kTiles][2][4];
#pragma unroll
            for (int mt = 0; mt < C::kTiles; ++mt)
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[mt][n][e] = 0.f;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t b[4];  // keys 0-7 and 8-15, dims 16k..16k+15
                ldmatrix4(b, kbase + (k_at ^ (k << 5)));
#pragma unroll
                for (int mt = 0; mt < C::kTiles; ++mt) {
                    mma_16816<T>(s[mt][0], qf[mt][k], b[0], b[1]);
                    mma_16816<T>(s[mt][1], qf[mt][k], b[2], b[3]);
                }
            }
            const int key = now.tile.block(now.unit) * kFewKeys + warp * 16;
            const Tile& t = now.tile;
            const bool all = key + 15 <= t.p0 - (TREE ? 1 : 0) &&
                             (a.window <= 0 || key > t.p1 - a.window || key + 15 < a.sinks);
            if (!all) {
#pragma unroll
                for (int mt = 0; mt < C::kTiles; ++mt)
#pragma unroll
                    for (int half = 0; half < C::kHalves; ++half)
#pragma unroll
                        for (int n = 0; n < 2; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                if (!sees(mt, half, key + n * 8 + (lane & 3) * 2 + e)) s[mt][n][half * 2 + e] = -INFINITY;
                            }
            }
            // (scaled on their own: s - m is then exact near m, whatever their size)
#pragma unroll
            for (int mt = 0; mt < C::kTiles; ++mt)
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2 * C::kHalves; ++e) s[mt][n][e] = __fmul_rn(s[mt][n][e], a.scale);
            bool grow = false;
#pragma unroll
            for (int mt = 0; mt < C::kTiles; ++mt)
#pragma unroll
                for (int half = 0; half < C::kHalves; ++half)
                    grow |= fmaxf(fmaxf(s[mt][0][half * 2], s[mt][0][half * 2 + 1]),
                                  fmaxf(s[mt][1][half * 2], s[mt][1][half * 2 + 1])) - m[mt][half] > kMostExponent;
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int mt = 0; mt < C::kTiles; ++mt)
#pragma unroll
                    for (int half = 0; half < C::kHalves; ++half) {
                        float top = fmaxf(fmaxf(s[mt][0][half * 2], s[mt][0][half * 2 + 1]),
                                          fmaxf(s[mt][1][half * 2], s[mt][1][half * 2 + 1]));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                        top = softmax_reference(top);
                        if (top > m[mt][half]) {
                            const float f = ex2_approx(m[mt][half] - top);  // 0 for the first keys
                            m[mt][half] = top;
                            l[mt][half] *= f;
#pragma unroll
                            for (int n = 0; n < kCols; ++n) {
                                o[mt][n][half * 2] *= f;
                                o[mt][n][half * 2 + 1] *= f;
                            }
                        }
                    }
            }
            uint32_t pf[C::kTiles][4];
#pragma unroll
            for (int mt = 0; mt < C::kTiles; ++mt) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    if (half >= C::kHalves) {
                        pf[mt][half] = pf[mt][2 + half] = 0u;
                        continue;
                    }
                    const float base = m[mt][half] == -INFINITY ? 0.f : m[mt][half];
                    float p[4];
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) p[n * 2 + e] = ex2_approx(__fsub_rn(s[mt][n][half * 2 + e], base));
                    l[mt][half] += (p[0] + p[1]) + (p[2] + p[3]);
                    pf[mt][half] = Pair<T>::pack(p[0], p[1]);
                    pf[mt][2 + half] = Pair<T>::pack(p[2], p[3]);
                }
            }
            if (!all && (TREE || t.tokens > 1)) {
                uint8_t* piece = few_smem + (vbase - smem_addr(few_smem));
                uint4* v = reinterpret_cast<uint4*>(piece) + lane;
                uint32_t bad = 0;
#pragma unroll
                for (int c = 0; c < C::kPiece / 16; c += 32)
                    bad |= not_finite<T>(v[c].x) | not_finite<T>(v[c].y) | not_finite<T>(v[c].z) | not_finite<T>(v[c].w);
                if (__any_sync(0xffffffffu, bad != 0)) {
#pragma unroll 1
                    for (int j = 0; j < 16; ++j) {
#pragma unroll
                        for (int n = 0; n < kCols; ++n) {
                            const uint32_t w = *reinterpret_cast<const uint32_t*>(piece + piece_at<D>(j, n) + (lane & 3) * 4);
                            const uint32_t which = not_finite<T>(w);
                            if (which == 0) continue;
                            const float2 x = Pair<T>::unpack(w & halves_of(which));
#pragma unroll
                            for (int mt = 0; mt < C::kTiles; ++mt)
#pragma unroll
                                for (int half = 0; half < C::kHalves; ++half) {
                                    if (!sees(mt, half, key + j)) continue;
                                    o[mt][n][half * 2] += x.x;
                                    o[mt][n][half * 2 + 1] += x.y;
                                }
                        }
                    }
                    __syncwarp();
#pragma unroll 1
                    for (int c = 0; c < C::kPiece / 16; c += 32) {
                        uint4 x = v[c];
                        x.x &= ~halves_of(not_finite<T>(x.x)), x.y &= ~halves_of(not_finite<T>(x.y));
                        x.z &= ~halves_of(not_finite<T>(x.z)), x.w &= ~halves_of(not_finite<T>(x.w));
                        v[c] = x;
                    }
                    __syncwarp();
                }
            }
#pragma unroll
            for (int n = 0; n < kCols; n += 2) {
                uint32_t b[4];  // dims 8n..8n+7 (keys 0-7, 8-15), then the next eight
                ldmatrix4_trans(b, vbase + (v_at ^ (n << 4)));
#pragma unroll
                for (int mt = 0; mt < C::kTiles; ++mt) {
                    mma_16816<T>(o[mt][n], pf[mt], b[0], b[1]);
                    mma_16816<T>(o[mt][n + 1], pf[mt], b[2], b[3]);
                }
            }
        }
        // refill the stage freed one step ago
        __syncwarp();
        live >>= 1;
        if (more) {
            load(ahead, page, (stage + C::kStages - 1) % C::kStages);
            live |= (page != -1 ? 1u : 0u) << (C::kStages - 2);
            more = ahead.next(a, tile_tokens);
            if (more) page = page_of(ahead);
        }
        async_copy_commit();
        stage = (stage + 1) % C::kStages;

        const bool item_done = now.item_ends();
        if (!now.part_ends()) {
            now.next(a, tile_tokens);
            continue;
        }

        // ---- the warps join their sums: 2, 3 into 0, 1, then 1 into 0 --------
        float* stat = reinterpret_cast<float*>(few_smem + C::kStatOff);
        constexpr int kAll = 16 * C::kTiles;
#pragma unroll
        for (int mt = 0; mt < C::kTiles; ++mt)
#pragma unroll
            for (int half = 0; half < C::kHalves; ++half) {
                l[mt][half] += __shfl_xor_sync(0xffffffffu, l[mt][half], 1);
                l[mt][half] += __shfl_xor_sync(0xffffffffu, l[mt][half], 2);
            }
#pragma unroll
        for (int round = 2; round >= 1; round >>= 1) {
            if (warp >= round && warp < 2 * round) {
                float* dst = reinterpret_cast<float*>(few_smem + C::kJoinOff + (warp - round) * C::kJoin);
                float* st = stat + (warp - round) * 2 * kAll;
#pragma unroll
                for (int mt = 0; mt < C::kTiles; ++mt)
#pragma unroll
                    for (int half = 0; half < C::kHalves; ++half) {
                        const int r = mt * 16 + half * 8 + lane / 4;
                        if ((lane & 3) == 0) {
                            st[r] = m[mt][half];
                            st[kAll + r] = l[mt][half];
                        }
#pragma unroll
                        for (int n = 0; n < kCols; ++n)
                            *reinterpret_cast<float2*>(dst + r * D + ((n ^ (r & 7)) * 8) + (lane & 3) * 2) =
                                make_float2(o[mt][n][half * 2], o[mt][n][half * 2 + 1]);
                    }
            }
            __syncthreads();
            if (warp < round) {
                const float* src = reinterpret_cast<const float*>(few_smem + C::kJoinOff + warp * C::kJoin);
                const float* st = stat + warp * 2 * kAll;
#pragma unroll
                for (int mt = 0; mt < C::kTiles; ++mt)
#pragma unroll
                    for (int half = 0; half < C::kHalves; ++half) {
                        const int r = mt * 16 + half * 8 + lane / 4;
                        const float mo = st[r], top = fmaxf(m[mt][half], mo);
                        const float f = m[mt][half] == -INFINITY ? 0.f : ex2_approx(m[mt][half] - top);
                        const float g = mo == -INFINITY ? 0.f : ex2_approx(mo - top);
                        m[mt][half] = top;
                        l[mt][half] = l[mt][half] * f + st[kAll + r] * g;
#pragma unroll
                        for (int n = 0; n < kCols; ++n) {
                            const float2 x = *reinterpret_cast<const float2*>(src + r * D + ((n ^ (r & 7)) * 8) +
                                                                              (lane & 3) * 2);
                            o[mt][n][half * 2] = o[mt][n][half * 2] * f + x.x * g;
                            o[mt][n][half * 2 + 1] = o[mt][n][half * 2 + 1] * f + x.y * g;
                        }
                    }
            }
            __syncthreads();
        }

        // ---- the item's result, or this CTA's part of it --------------------
        const bool whole = begun && item_done;
        float* part = a.partials + static_cast<long long>(2 * blockIdx.x + (begun ? 1 : 0)) * ROWS * (D + 2);
        if (warp == 0) {
#pragma unroll
            for (int mt = 0; mt < C::kTiles; ++mt)
#pragma unroll
                for (int half = 0; half < C::kHalves; ++half) {
                    const int r = mt * 16 + half * 8 + lane / 4, i = r / a.group;
                    if (i >= now.tile.tokens) continue;
                    if (whole) {
                        const float inv = l[mt][half] > 0.f || isnan(l[mt][half]) ? 1.0f / l[mt][half] : 0.f;
                        const int head = now.h * a.group + r - i * a.group;
                        T* out = static_cast<T*>(a.out) + (now.tile.first + i) * a.out_stride + head * D + (lane & 3) * 2;
#pragma unroll
                        for (int n = 0; n < kCols; ++n)
                            *reinterpret_cast<uint32_t*>(out + n * 8) =
                                Pair<T>::pack(o[mt][n][half * 2] * inv, o[mt][n][half * 2 + 1] * inv);
                        if (a.lse != nullptr && (lane & 3) == 0)
                            a.lse[static_cast<long long>(now.tile.first + i) * a.heads + head] =
                                l[mt][half] == 0.f
                                    ? -INFINITY
                                    : m[mt][half] * 0.6931471805599453f + logf(l[mt][half]);
                    } else {
                        if ((lane & 3) == 0) {
                            __stcg(part + ROWS * D + 2 * r, m[mt][half]);
                            __stcg(part + ROWS * D + 2 * r + 1, l[mt][half]);
                        }
#pragma unroll
                        for (int n = 0; n < kCols; ++n)
                            __stcg(reinterpret_cast<float2*>(part + r * D + n * 8 + (lane & 3) * 2),
                                   make_float2(o[mt][n][half * 2], o[mt][n][half * 2 + 1]));
                    }
                }
        }
        if (!whole) {
            const int2 owners = item_owners(range, now);
            const int c0 = owners.x, c1 = owners.y;
            int* flag = reinterpret_cast<int*>(few_smem + C::kStatOff);
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                const unsigned seen = atom_acq_rel_add(a.counters + c0, 1u);
                *flag = seen == static_cast<unsigned>(c1 - c0);
                if (*flag) a.counters[c0] = 0u;  // zero for the next call
            }
            __syncthreads();
            if (*flag) {
                __threadfence();
                const int rows = now.tile.tokens * a.group;
                for (int x = threadIdx.x; x < rows * (D / 4); x += kFewThreads) {
                    const int r = x / (D / 4), c = x % (D / 4), i = r / a.group;
                    float top = -INFINITY;
#pragma unroll 8
                    for (int cta = c0; cta <= c1; ++cta)
                        top = fmaxf(top, __ldcg(a.partials + static_cast<long long>(2 * cta + (cta == c0)) * ROWS * (D + 2) +
                                                ROWS * D + 2 * r));
                    float sum = 0.f;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                    for (int cta = c0; cta <= c1; ++cta) {
                        const float* q = a.partials + static_cast<long long>(2 * cta + (cta == c0)) * ROWS * (D + 2);
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(q + ROWS * D + 2 * r));
                        const float4 y = __ldcg(reinterpret_cast<const float4*>(q + r * D) + c);
                        const float f = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - top);
                        sum += ml.y * f;
                        v.x += y.x * f, v.y += y.y * f, v.z += y.z * f, v.w += y.w * f;
                    }
                    const float inv = sum > 0.f || isnan(sum) ? 1.0f / sum : 0.f;
                    const int head = now.h * a.group + r - i * a.group;
                    T* out = static_cast<T*>(a.out) + (now.tile.first + i) * a.out_stride + head * D;
                    *(reinterpret_cast<uint2*>(out) + c) =
                        make_uint2(Pair<T>::pack(v.x * inv, v.y * inv), Pair<T>::pack(v.z * inv, v.w * inv));
                    if (a.lse != nullptr && c == 0)
                        a.lse[static_cast<long long>(now.tile.first + i) * a.heads + head] =
                            sum == 0.f ? -INFINITY : top * 0.6931471805599453f + logf(sum);
                }
            }
            __syncthreads();
        }
        if (!now.next(a, tile_tokens)) break;
        begun = true;
        fresh = true;
    }
    async_copy_wait_all();
}

}  // namespace h4b

#include "paged_tc.cu"
#include "paged_tree.cu"

namespace h4b {

// ---- host side -----------------------------------------------------------------

static bool paged_view(const h4b_paged_kv* kv, PagedView* out) {
    if (kv == nullptr || kv->pages < 1 || kv->kv_heads < 1 || kv->sequences < 0 || kv->table_stride < 0 || kv->tokens < 0)
        return false;
    if (kv->page_size < 16 || kv->page_size > 1024 || (kv->page_size & (kv->page_size - 1))) return false;
    if (kv->k_pages == nullptr || kv->v_pages == nullptr ||
        ((reinterpret_cast<uintptr_t>(kv->k_pages) | reinterpret_cast<uintptr_t>(kv->v_pages)) & 15))
        return false;
    if (kv->sequences > 0 && (kv->q_offsets == nullptr || kv->kv_lens == nullptr ||
                              (kv->page_table == nullptr && kv->table_stride > 0)))
        return false;
    int shift = 0;
    while ((1 << shift) < kv->page_size) ++shift;
    *out = PagedView{kv->pages, shift, kv->kv_heads, kv->sequences, kv->table_stride, kv->tokens, kv->page_table,
                     kv->q_offsets, kv->kv_lens};
    return true;
}

// The kernels count the values of a page and of a row (of row_heads heads) in 32 bits.
static bool paged_shape_supported(const h4b_paged_kv* kv, long long row_heads) {
    return (kv->dtype == H4B_FP16 || kv->dtype == H4B_BF16) && (kv->head_dim == 64 || kv->head_dim == 128) &&
           static_cast<long long>(kv->kv_heads) * kv->page_size <= INT_MAX / kv->head_dim &&
           row_heads <= INT_MAX / kv->head_dim;
}

static int paged_sm_count(int* sms) {
    static std::atomic<int> known[kMaxDevices];
    int dev = 0;
    H4B_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= kMaxDevices) return H4B_EUNSUPPORTED;
    int n = known[dev].load(std::memory_order_acquire);
    if (n == 0) {
        H4B_CUDA_TRY(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
        known[dev].store(n, std::memory_order_release);
    }
    *sms = n;
    return 0;
}

// The few-row kernel's CTAs an SM and largest tile; as many q heads may share a
// kv head (a token's group stays in one tile of either kernel).
constexpr int kFewCtasPerSm = 2, kFewMaxRows = 32;
constexpr long long kCounterBytes = 4096, kEntryBytes = 4096;
constexpr long long kTreeEntryBytes = 8192;  // (the tree kernel may have two CTAs an SM)

template <typename S, typename T, int D, bool TREE>
static int launch_append(AppendArgs a, cudaStream_t stream) {
    // Few tokens: a token's heads are spread over as many warps as it takes;
    // many: kAppendShare warps walk them, which look up the token's place once
    // each.
    const int total = a.heads + 2 * a.p.kv_heads, most = (total * D + 255) / 256;
    a.parts = a.p.tokens >= 1024 && most > kAppendShare ? kAppendShare : most;
    const long long ctas = (static_cast<long long>(a.p.tokens) * a.parts + kAppendWarps - 1) / kAppendWarps;
    if (ctas > INT_MAX / kAppendWarps) return H4B_EUNSUPPORTED;
    paged_append_kernel<S, T, D, TREE><<<static_cast<unsigned>(ctas), 32 * kAppendWarps, 0, stream>>>(a);
    H4B_CUDA_TRY(cudaGetLastError());
    return 0;
}

template <typename T, int D, int ROWS, bool TREE = false>
static int launch_few(AttendArgs a, int sms, cudaStream_t stream) {
    using C = FewCfg<D, ROWS>;
    constexpr int kSmem = TREE ? C::kTreeSmem : C::kSmem;
    a.extra = kFewExtra;
    a.least = kFewLeast;
    static std::atomic<bool> opted_in[kMaxDevices];
    int dev = 0;
    H4B_CUDA_TRY(cudaGetDevice(&dev));
    if (!opted_in[dev].load(std::memory_order_acquire)) {
        H4B_CUDA_TRY(cudaFuncSetAttribute(paged_attention_few_kernel<T, D, ROWS, TREE>,
                                          cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
        opted_in[dev].store(true, std::memory_order_release);
    }
    paged_attention_few_kernel<T, D, ROWS, TREE><<<kFewCtasPerSm * sms, kFewThreads, kSmem, stream>>>(a);
    H4B_CUDA_TRY(cudaGetLastError());
    return 0;
}

template <typename T, int D>
static int launch_few_rows(const AttendArgs& a, int rows, int sms, cudaStream_t stream) {
    if (rows <= 8) return launch_few<T, D, 8>(a, sms, stream);
    if constexpr (D == 64)
        if (rows > 16) return launch_few<T, D, 32>(a, sms, stream);
    return launch_few<T, D, 16>(a, sms, stream);
}

// Trees of few rows in the few-row kernel, others on tcgen05. In us, the few-row
// kernel and the other one: 8 rows of head_dim 128 324 and 321 (16 x 32768 tokens),
// 57 and 59 (64 ragged trees up to 2100), 10.9 and 12.8 (one over 1000), 132 and 136
// (windows of 4096); 16 rows 329 and 324, 68 and 59, 13.9 and 13.1, 140 and 138. 16
// rows of 64 201 and 210, 51 and 49, 10.9 and 11.3, 96 and 98; 32 rows 249 and 212,
// 80 and 50, 20.4 and 11.4, 128 and 98.
template <typename T, int D>
static int launch_tree(AttendArgs a, const h4b_paged_kv* kv, int max_query, int sms, cudaStream_t stream) {
    a.fewest = 1;
    a.most = INT_MAX;
    const long long rows = static_cast<long long>(max_query) * a.group;
    if (rows <= 8) return launch_few<T, D, 8, true>(a, sms, stream);
    if constexpr (D == 64)
        if (rows <= 16) return launch_few<T, D, 16, true>(a, sms, stream);
    return launch_tree_tiles<T, D>(a, kv, max_query, sms, stream);
}

template <typename T, int D>
static int launch_attention(AttendArgs a, const h4b_paged_kv* kv, int max_query, int sms, cudaStream_t stream) {
    // Few rows: up to 16 (32 at head_dim 64, where the registers last): 32 x
    // 32768 tokens of 8 kv heads in 615 us with 4 rows, 615 with 8, 623 with 16,
    // 1883 with 32 (spilled), the chunk kernel 926 to 958 (816 to 824 before the
    // power cap). At head_dim 64 64 ragged sequences of 4 kv heads with 32 rows:
    // 39 us, the chunk kernel 50.
    constexpr int kMost = D == 64 ? 32 : 16;
    const long long rows = static_cast<long long>(max_query) * a.group;
    a.fewest = 1;
    a.most = INT_MAX;
    if (rows > kMost) {
        // A step of few long chunks among many short ones (the mean is under
        // half of the longest): the short ones go to the kernel of few rows, in
        // a launch of its own, where they are many enough to pay for it. Three
        // 255-token chunks among 16, 20, 24, 32 and 64 sequences of 1000 to 2000
        // tokens, one launch against two: 24 / 8 heads of 64 61-66, 72-76, 74-74,
        // 82-78 and 129-98 us; 32 / 8 of 128 70-80, 80-92, 82-92, 92-96 and
        // 143-137 (40: 107-109). The same with 100 to 8000 tokens and one or
        // eight chunks, within 8 sequences; of 20 to 200 tokens two launches pay
        // from about 50 (24: 33-39, 64: 47-43).
        const int few_rows = a.group <= 8 ? 8 : (a.group <= 16 ? 16 : 32);
        if (few_rows <= kMost && a.p.sequences >= (D == 64 ? 20 : 40) &&
            2ll * a.p.tokens < static_cast<long long>(a.p.sequences) * max_query) {
            a.most = few_rows / a.group;
            if (const int rc = launch_few_rows<T, D>(a, few_rows, sms, stream)) return rc;
            a.fewest = a.most + 1;
            a.most = INT_MAX;
        }
        return launch_chunk<T, D>(a, kv, sms, stream);
    }
    return launch_few_rows<T, D>(a, static_cast<int>(rows), sms, stream);
}

template <bool TREE>
static int launch_append_types(const AppendArgs& a, const h4b_paged_kv* kv, int qkv_dtype, cudaStream_t s) {
    const bool wide = kv->head_dim == 128, from32 = qkv_dtype == H4B_FP32;
    if (kv->dtype == H4B_FP16) {
        if (from32) return wide ? launch_append<float, __half, 128, TREE>(a, s) : launch_append<float, __half, 64, TREE>(a, s);
        return wide ? launch_append<__half, __half, 128, TREE>(a, s) : launch_append<__half, __half, 64, TREE>(a, s);
    }
    using B16 = __nv_bfloat16;
    if (from32) return wide ? launch_append<float, B16, 128, TREE>(a, s) : launch_append<float, B16, 64, TREE>(a, s);
    return wide ? launch_append<B16, B16, 128, TREE>(a, s) : launch_append<B16, B16, 64, TREE>(a, s);
}

// `parents`: the new tokens are a tree's nodes (null: one after the other).
static int paged_append(const h4b_paged_kv* kv, const int32_t* parents, const void* qkv, int qkv_dtype,
                        long long qkv_stride, int heads, const float* norm_q, const float* norm_k, float eps,
                        const float* rope_cos, const float* rope_sin, int max_pos, void* q_out, long long q_stride,
                        void* stream) {
    AppendArgs a{};
    if (!paged_view(kv, &a.p) || heads < 0) return H4B_EINVAL;
    const long long row_heads = heads + 2ll * kv->kv_heads;
    if (!paged_shape_supported(kv, row_heads) || (qkv_dtype != H4B_FP32 && qkv_dtype != kv->dtype)) return H4B_EUNSUPPORTED;
    if ((norm_q == nullptr) != (norm_k == nullptr) || (rope_cos == nullptr) != (rope_sin == nullptr) ||
        (rope_cos != nullptr && max_pos < 1))
        return H4B_EINVAL;
    if (kv->tokens == 0 || kv->sequences == 0) return 0;
    if (qkv == nullptr || (heads > 0 && q_out == nullptr)) return H4B_EINVAL;
    const auto misaligned = [](const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; };
    if (qkv_stride < row_heads * kv->head_dim || (qkv_stride & 3) ||
        (heads > 0 && (q_stride < static_cast<long long>(heads) * kv->head_dim || (q_stride & 3))))
        return H4B_EINVAL;
    if (misaligned(qkv, qkv_dtype == H4B_FP32 ? 16 : 8) || misaligned(rope_cos, 16) || misaligned(rope_sin, 16) ||
        misaligned(norm_q, 16) || misaligned(norm_k, 16) || misaligned(q_out, 8))
        return H4B_EINVAL;
    a.qkv = qkv, a.qkv_stride = qkv_stride, a.norm_q = norm_q, a.norm_k = norm_k, a.cos = rope_cos, a.sin = rope_sin;
    a.max_pos = max_pos, a.heads = heads, a.eps = eps, a.q_out = q_out, a.q_stride = q_stride;
    a.k_pages = kv->k_pages, a.v_pages = kv->v_pages;
    a.parents = parents;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return parents == nullptr ? launch_append_types<false>(a, kv, qkv_dtype, s) : launch_append_types<true>(a, kv, qkv_dtype, s);
}

}  // namespace h4b

extern "C" int h4b_paged_append(const h4b_paged_kv* kv, const void* qkv, int qkv_dtype, long long qkv_stride, int heads,
                                const float* norm_q, const float* norm_k, float eps, const float* rope_cos,
                                const float* rope_sin, int max_pos, void* q_out, long long q_stride, void* stream) {
    return h4b::paged_append(kv, nullptr, qkv, qkv_dtype, qkv_stride, heads, norm_q, norm_k, eps, rope_cos, rope_sin,
                             max_pos, q_out, q_stride, stream);
}

extern "C" int h4b_paged_append_tree(const h4b_paged_kv* kv, const int32_t* parents, const void* qkv, int qkv_dtype,
                                     long long qkv_stride, int heads, const float* norm_q, const float* norm_k, float eps,
                                     const float* rope_cos, const float* rope_sin, int max_pos, void* q_out,
                                     long long q_stride, void* stream) {
    if (parents == nullptr && kv != nullptr && kv->tokens > 0) return H4B_EINVAL;
    return h4b::paged_append(kv, parents, qkv, qkv_dtype, qkv_stride, heads, norm_q, norm_k, eps, rope_cos, rope_sin,
                             max_pos, q_out, q_stride, stream);
}

extern "C" int h4b_pages_copy(void* k_pages, void* v_pages, int layers, int pages, long long page_bytes,
                              const int32_t* src, const int32_t* dst, int count, void* stream) {
    using namespace h4b;
    if (k_pages == nullptr || v_pages == nullptr || layers < 1 || layers > 65535 || pages < 1 || page_bytes < 16 ||
        (page_bytes & 15) || count < 0 || (count > 0 && (src == nullptr || dst == nullptr)) ||
        ((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15))
        return H4B_EINVAL;
    if (count == 0) return 0;
    const long long parts = (page_bytes + kCopyBytes - 1) / kCopyBytes;
    if (parts * count > 0x7fffffffll) return H4B_EUNSUPPORTED;
    pages_copy_kernel<<<dim3(static_cast<unsigned>(parts * count), layers, 2), kCopyThreads, 0,
                        static_cast<cudaStream_t>(stream)>>>(static_cast<uint8_t*>(k_pages),
                                                             static_cast<uint8_t*>(v_pages), pages, page_bytes,
                                                             static_cast<int>(parts), src, dst);
    H4B_CUDA_TRY(cudaGetLastError());
    return 0;
}

namespace h4b {

// Workspace bytes of either attention, of trees or not; negative: an error.
static long long attention_workspace_bytes(int head_dim, bool tree) {
    int sms = 0;
    if (head_dim != 64 && head_dim != 128) return H4B_EUNSUPPORTED;
    if (const int rc = paged_sm_count(&sms)) return rc > 0 ? -1000 - rc : rc;
    // two parts a CTA: an SM's rows of the few-row kernel are fewer than
    // the 256 of the chunk kernel's CTA
    static_assert(kFewCtasPerSm * kFewMaxRows <= 2 * kChunkRows, "the chunk kernel's parts are the larger");
    // (the tree kernel's are as many rows an SM: two CTAs of 128 or one of 256)
    if (kFewCtasPerSm * sms * 4 > kCounterBytes || sms * 16 > kEntryBytes || 2 * sms * 16 > kTreeEntryBytes)
        return H4B_EUNSUPPORTED;
    return kCounterBytes + (tree ? kTreeEntryBytes : kEntryBytes) + 2ll * sms * 2 * kChunkRows * (head_dim + 2) * 4;
}

// `parents`: the new tokens are a tree's nodes (null: one after the other).
static int paged_attention(const h4b_paged_kv* kv, const int32_t* parents, const void* q, long long q_stride, int heads,
                           float scale, int window, int sinks, int max_query, void* out, long long out_stride, float* lse,
                           void* workspace, long long workspace_bytes, void* stream) {
    AttendArgs a{};
    if (!paged_view(kv, &a.p) || heads < 1 || heads % kv->kv_heads || window < 0 || sinks < 0 ||
        (sinks > 0 && window == 0) || max_query < 1)
        return H4B_EINVAL;
    // Both kernels take the maxima before the scale and mask with -infinity.
    const float base2_scale = scale * 1.4426950408889634f;
    if (!(base2_scale > 0.f) || !std::isfinite(base2_scale)) return H4B_EINVAL;
    if (!paged_shape_supported(kv, heads) || heads / kv->kv_heads > kFewMaxRows ||
        static_cast<long long>(kv->pages) * kv->kv_heads > 0x7fffffffll)
        return H4B_EUNSUPPORTED;
    if (kv->tokens == 0 || kv->sequences == 0) return 0;
    if (q == nullptr || out == nullptr || workspace == nullptr) return H4B_EINVAL;
    const long long width = static_cast<long long>(heads) * kv->head_dim;
    if (q_stride < width || out_stride < width || ((q_stride | out_stride) & 7) ||
        ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) &
         15))
        return H4B_EINVAL;
    const long long need = attention_workspace_bytes(kv->head_dim, parents != nullptr);
    if (need < 0 || workspace_bytes < need) return H4B_EINVAL;
    int sms = 0;
    if (const int rc = paged_sm_count(&sms)) return rc;
    a.q = q, a.k_pages = kv->k_pages, a.v_pages = kv->v_pages, a.out = out, a.lse = lse;
    a.q_stride = q_stride, a.out_stride = out_stride, a.heads = heads, a.group = heads / kv->kv_heads;
    a.window = window < kMaxLength ? window : kMaxLength, a.sinks = sinks, a.scale = base2_scale;
    a.counters = static_cast<unsigned int*>(workspace);
    a.entries = reinterpret_cast<int4*>(static_cast<uint8_t*>(workspace) + kCounterBytes);
    a.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kCounterBytes +
                                          (parents != nullptr ? kTreeEntryBytes : kEntryBytes));
    a.parents = parents;
    const int longest = max_query < kv->tokens ? max_query : kv->tokens;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool wide = kv->head_dim == 128;
    using B16 = __nv_bfloat16;
    if (parents != nullptr) {
        if (kv->dtype == H4B_FP16)
            return wide ? launch_tree<__half, 128>(a, kv, longest, sms, s) : launch_tree<__half, 64>(a, kv, longest, sms, s);
        return wide ? launch_tree<B16, 128>(a, kv, longest, sms, s) : launch_tree<B16, 64>(a, kv, longest, sms, s);
    }
    if (kv->dtype == H4B_FP16)
        return wide ? launch_attention<__half, 128>(a, kv, longest, sms, s) : launch_attention<__half, 64>(a, kv, longest, sms, s);
    return wide ? launch_attention<B16, 128>(a, kv, longest, sms, s) : launch_attention<B16, 64>(a, kv, longest, sms, s);
}

}  // namespace h4b

extern "C" long long h4b_paged_attention_workspace_bytes(int head_dim) {
    return h4b::attention_workspace_bytes(head_dim, true);  // for both: the larger
}

extern "C" int h4b_paged_attention(const h4b_paged_kv* kv, const void* q, long long q_stride, int heads, float scale,
                                   int window, int sinks, int max_query, void* out, long long out_stride, float* lse,
                                   void* workspace, long long workspace_bytes, void* stream) {
    return h4b::paged_attention(kv, nullptr, q, q_stride, heads, scale, window, sinks, max_query, out, out_stride, lse,
                                workspace, workspace_bytes, stream);
}

extern "C" int h4b_paged_tree_attention(const h4b_paged_kv* kv, const int32_t* parents, const void* q, long long q_stride,
                                        int heads, float scale, int window, int sinks, int max_query, void* out,
                                        long long out_stride, float* lse, void* workspace, long long workspace_bytes,
                                        void* stream) {
    if (parents == nullptr && kv != nullptr && kv->tokens > 0) return H4B_EINVAL;
    return h4b::paged_attention(kv, parents, q, q_stride, heads, scale, window, sinks, max_query, out, out_stride, lse,
                                workspace, workspace_bytes, stream);
}
