// Paged attention of drafted trees of more than a few rows on the 5th-generation
// tensor cores: tcgen05.mma kind::f16, fp32 accumulators in tensor memory, pages
// fetched by TMA. The split of the work over the CTAs is that of paged.cu, the
// layout of the tiles and the operands' descriptors are those of paged_tc.cu.
//
// An item is (sequence, up to 128 query rows = nodes x q heads of a kv head, kv
// head). Its keys are read once for few products each, so HBM is the bound, and
// what has to hide under the loads is the chain S -> softmax -> P V of a block of
// 64 keys, and an item's start and end. So two CTAs share an SM, each with half of
// its tensor memory and shared memory: what one waits for the other fills. (One
// CTA with two warpgroups that took an item's blocks of 128 keys in turn: 64 trees
// of 16 nodes over ragged 2100 tokens 100 us, two CTAs 71 and, with the steps below,
// 69; 16 x 32 nodes over 32768 386, 375 and 365 to 371; over 16-token pages 570 and 402.)
//
// Warps: 0-3 are the softmax (thread = query row = TMEM lane), 4 issues the loads,
// 5 the MMAs, 6 cleans V tiles. For block n, x = n % 2:
//   MMA:     S_x = Q K_n^T                      -> s_full[x]
//   softmax: S_x to registers, p; P_x over S_x  -> p_full[x]
//   MMA:     S of block n + 1, then O += P_x V_n, whichever's operands come first
// S_x of block n + 2 is issued after P V of block n, which reads P_x: the tensor
// cores run a CTA's MMAs in issue order.
//
// A node sees the tokens before the tree and, of the tree, the nodes whose bits
// its walk to the root set (sight); blocks that hold only keys that every row
// sees need no mask. p = 2^(s scale - b + 8) with b the product m scale of a score m,
// rounded on its own: what the rounding adds to b it adds to all weights of the row
// alike, and the log-sum-exp takes it off again. m moves only where a score passes it
// by 2^7. From |b - 8| = 2^20 on, where the rounding would reach p's exponent, p = 2^((s - m)
// scale + 8), in which equal scores cancel whatever their size: one more operation a
// pair, which costs nothing in time but, under the power cap, clock (16 x 32 nodes
// over 32768 tokens, sustained: 420 -> 411 us without it), so it is left out where no row
// of the warp needs it. Which form a row's weights have goes by its own m, so l and O of
// other blocks and parts are carried over with the right factor.
//
// l is summed from the fp32 p, which is rounded to the cache's type for the product
// with V only, where both operands have one type. The rest of p as a second operand of
// that product (it fits into the columns of the scores) costs most where the tensor pipe
// and the softmax are the bound, and something everywhere: one tree of 8 nodes 12.8 ->
// 13.6 us, 64 ragged trees of 16 69 -> 76, 16 x 32 nodes over 32768 tokens 368 -> 424 (under
// the power cap 444 -> 528), of 64 nodes 620 -> 783, windowed trees at head_dim 64 58 -> 68
// to 72. The rounding is to 2^-12 of a weight (bf16 2^-9), independent from key to key,
// and its part of a sum stays below the result's own rounding: against 64 bits 2.6e-4 in
// fp16 and 2.1 to 2.3e-3 in bf16 of the result's rms, 2.1e-4 and 1.7e-3 without it.
//
// V rows of keys that no row sees are zeroed and values that are not finite are
// taken out of rows that only some see, and added at the item's end, as in
// paged_tc.cu.
//
// Every wait is bounded (mbar_wait, or a loop with its limit). A role whose wait
// runs out marks the CTA as failed and stops; the load warp waits for the copies
// it issued, the MMA warp commits a last barrier, and the tensor memory is freed
// on every path.

namespace h4b {

constexpr int kTreeKeys = 64;
constexpr int kTreeWholeFew = 6, kTreeWholeMany = 15;  // blocks of an item, at most, for whole items
constexpr int kTreeLeast = 2, kTreeExtra = 4;  // as kChunkLeast and kChunkExtra, of 64 keys

// TILES x ROWS: the query rows of an item that there is room for, in tiles of up to
// 128 that share the keys; the MMAs take 128 all the same, and what they make of
// the others' lanes goes nowhere.
template <int D, int ROWS, int TILES>
struct TreeCfg {
    static constexpr int kCtasPerSm = 2 / TILES;
    static constexpr int kLoadWarp = 4 * TILES, kMmaWarp = kLoadWarp + 1, kCleanWarp = kLoadWarp + 2;
    static constexpr int kThreads = 32 * (kLoadWarp + 3);
    static constexpr int kSlabs = D / 64;                        // 64 values of head_dim each
    static constexpr int kSlab = ROWS * 128;                     // of Q
    static constexpr int kGroup = kSlabs * 1024;                 // of K or V: 8 keys, all slabs
    static constexpr int kTile = kTreeKeys / 8 * kGroup;
    static constexpr int kStages = (TILES == 2 ? 9 : ROWS == 128 ? 4 : 5) * (128 / D);
    static constexpr int kQOff = 0, kQTile = kSlabs * kSlab, kRingOff = TILES * kQTile, kBarOff = kRingOff + kStages * kTile;
    static constexpr int kBars = 3 * kStages + 5 + 7 * TILES;
    static constexpr int kFlagOff = kBarOff + kBars * 8 + 16;
    static constexpr int kRangeOff = (kFlagOff + kStages * 4 + 7) / 8 * 8;
    static constexpr int kSightOff = (kRangeOff + static_cast<int>(sizeof(Range)) + 15) / 16 * 16;  // [kTreeNodes][kTreeWords]
    static constexpr int kDepthOff = kSightOff + kTreeNodes * kTreeWords * 4;                       // int16 [kTreeNodes]
    static constexpr int kSmem = kDepthOff + kTreeNodes * 2 + 1024;
    // S of tile t, block n at 64 (2 t + n % 2), O of tile t at kOCol + 128 t
    static constexpr uint32_t kColumns = 256 * TILES, kSCol = 0, kOCol = 128 * TILES;
    // (Q's 128 rows of the MMAs lie within the tiles' memory)
    static_assert(kQOff + TILES * kQTile - kSlab + 128 * 128 <= kBarOff, "rows that the MMAs read");
    static_assert(kCtasPerSm * (kSmem + 1024) <= 233472 && kSmem <= 232448, "shared memory per SM");
    static_assert(kStages <= 32, "a bit per stage");
};

// Whether the phase with the given parity has completed, without a wait.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(smem_addr(bar)), "r"(parity) : "memory");
    return done != 0;
}
__device__ __forceinline__ bool warp_test(uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_test(bar, parity));
}

// What each of a sequence's first `nodes` nodes sees of the tree, as bits, and its
// depth. By one warp, 32 nodes at a time, whose parents are among them or earlier:
// its descent within the 32, and the set of the earlier node that the topmost of
// them hangs from. With a window (of fewer than all nodes) what lies too far above
// is taken out at the end.
__device__ __forceinline__ void find_sights(const int (&parent)[kTreeWords], int nodes, int base, int window, int sinks,
                                            uint32_t* sights, int16_t* depths) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 0; k < kTreeWords; ++k) {
        if (32 * k >= nodes) break;
        const int i = 32 * k + lane;
        const int p = i < nodes ? checked_parent(parent[k], i) : -1;
        int above;
        const uint32_t mine = descent(p, 32 * k, &above);
        uint32_t* bits = sights + i * kTreeWords;
#pragma unroll
        for (int w = 0; w < kTreeWords; ++w)
            bits[w] = w < k ? (above >= 0 ? sights[above * kTreeWords + w] : 0u) : w == k ? mine : 0u;
        depths[i] = static_cast<int16_t>(__popc(mine) - 1 + (above >= 0 ? depths[above] + 1 : 0));
        __syncwarp();
    }
    if (window <= 0 || window >= nodes) return;
#pragma unroll 1
    for (int i = lane; i < nodes; i += 32) {
        const int depth = depths[i];
#pragma unroll 1
        for (int w = 0; w <= i >> 5; ++w) {
            uint32_t bits = sights[i * kTreeWords + w], left = bits;
            for (; left != 0u; left &= left - 1) {
                const int up = depths[32 * w + __ffs(left) - 1];
                if (depth - up >= window && base + up >= sinks) bits &= ~(left & (0u - left));
            }
            sights[i * kTreeWords + w] = bits;
        }
    }
    __syncwarp();
}

// Whether weights relative to score m, b = m scale, have the form for huge scores.
__device__ __forceinline__ bool is_huge_reference(float b) { return is_huge(__fsub_rn(8.f, b)); }
// What weights relative to score m are worth relative to `top`, each in its form:
// relative to the rounded product or, if it is huge, to the product itself.
__device__ __forceinline__ float reference_factor(float m, float top, float scale) {
    const float a = __fmul_rn(m, scale), b = __fmul_rn(top, scale);
    const bool huge = is_huge_reference(a);
    if (is_huge_reference(b)) return ex2_approx(huge ? (m - top) * scale : __fmaf_rn(-top, scale, a));
    return ex2_approx(huge ? __fmaf_rn(m, scale, -b) : __fsub_rn(a, b));
}

// Whether every row of the tile sees keys `key` .. `end`.
__device__ __forceinline__ bool tree_all_see(const Tile& t, int window, int sinks, int key, int end) {
    return end < t.p0 && (window <= 0 || key > t.p1 - window || end < sinks);
}

template <typename T, int D, int ROWS, int TILES>
__global__ void __launch_bounds__(TreeCfg<D, ROWS, TILES>::kThreads, TreeCfg<D, ROWS, TILES>::kCtasPerSm)
    paged_attention_tree_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                                const __grid_constant__ CUtensorMap vmap, const __grid_constant__ AttendArgs a) {
    using C = TreeCfg<D, ROWS, TILES>;
    using TreeWalk = Walk<kTreeKeys, true>;
    extern __shared__ uint8_t tree_smem_raw[];
    uint8_t* smem = tree_smem_raw + ((1024u - (smem_addr(tree_smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
    uint64_t* empty = full + C::kStages;
    uint64_t* raw = empty + C::kStages;  // a V tile on its way to the cleaning warp
    uint64_t* q_full = raw + C::kStages;
    uint64_t* q_empty = q_full + 1;
    uint64_t* s_full = q_empty + 1;            // [TILES][2], of blocks n % 2
    uint64_t* p_full = s_full + 2 * TILES;     // [TILES][2]
    uint64_t* pv_done = p_full + 2 * TILES;    // [TILES][2]
    uint64_t* o_full = pv_done + 2 * TILES;    // [TILES]
    uint64_t* sight_full = o_full + TILES;
    uint64_t* sight_free = sight_full + 1;
    uint64_t* mma_done = sight_free + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
    volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* wild = failed + 1;  // values that are not finite were taken out of a V tile
    volatile uint32_t* flags = reinterpret_cast<volatile uint32_t*>(smem + C::kFlagOff);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int half_tokens = a.half_tokens, tile_tokens = TILES * half_tokens;  // of a tile, of an item
    Range* shared_range = reinterpret_cast<Range*>(smem + C::kRangeOff);
    // barriers and tensor memory first: their cost hides behind the range's look-ups
    if (warp == C::kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_addr(tmem_slot)), "r"(C::kColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == 32 * C::kLoadWarp) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
            mbar_init(&raw[s], 1);
        }
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        for (int x = 0; x < 2 * TILES; ++x) {
            mbar_init(&s_full[x], 1);
            mbar_init(&p_full[x], 4);
            mbar_init(&pv_done[x], 1);
        }
        for (int t = 0; t < TILES; ++t) mbar_init(&o_full[t], 1);
        mbar_init(sight_full, 1);
        mbar_init(sight_free, 4 * TILES);
        mbar_init(mma_done, 1);
        *failed = wait_failed_before() ? 1 : 0;
        *wild = 0;
        fence_mbar_init();
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kmap)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&vmap)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&qmap)) : "memory");
    }
    pdl_trigger();  // the join waits for this grid's end in its kernel
    {
        const Range r = find_range<C::kThreads, kTreeKeys, true>(a, tile_tokens, smem);
        if (threadIdx.x == 0) {
            *shared_range = r;
            a.entries[blockIdx.x] = make_int4(-1, 0, 0, 0);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    uint32_t* sights = reinterpret_cast<uint32_t*>(smem + C::kSightOff);  // of the tile's sequence, up to its last node
    int16_t* depths = reinterpret_cast<int16_t*>(smem + C::kDepthOff);
    // One walk for all roles, in code that they share: each role's own would run cold.
    TreeWalk w;
    bool more = shared_range->begin < shared_range->end && w.start(a, *shared_range, tile_tokens);
    auto ring = [&](uint32_t i) { return smem + C::kRingOff + (i % C::kStages) * C::kTile; };
    auto phase_of = [&](uint32_t i) { return (i / C::kStages) & 1u; };

    // K of the CTA's block n is tile 2 n of the ring, V tile 2 n + 1. A block's
    // flags lie beside K's barrier, written before K's copies start.
    if (warp == C::kLoadWarp) {
        const int page_size = 1 << a.p.page_shift, box = min(page_size, kTreeKeys);  // a box: keys of one page
        const int boxes = kTreeKeys / box;
        const bool mine = lane < boxes;  // each lane one box
        auto page_of = [&](const TreeWalk& u) -> int {  // -1: read as zeros
            const int key = u.tile.block(u.unit) * kTreeKeys + lane * box;
            const Tile& t = u.tile;
            if (!mine || key > t.p1 || !(a.window <= 0 || key + box - 1 > t.p0 - a.window || key < a.sinks)) return -1;
            const int page = a.p.table[static_cast<long long>(u.b) * a.p.table_stride + (key >> a.p.page_shift)];
            if (page >= 0 && page < a.p.pages) return page;
            report(kStatusBadPage);
            return -1;
        };
        uint32_t issued = 0, raw_open = 0, raw_phase = 0;  // a bit per stage
        bool ok = !*failed;
        if (!more && lane == 0) {
            flags[0] = kStepNone;
            mbar_arrive(&full[0]);
        }
        int page = more ? page_of(w) : -1, items = 0;
        bool new_item = true;
        while (ok && more) {
            if (new_item) {  // the q rows, once the previous item's are no longer read
                if (items > 0) ok = __all_sync(0xffffffffu, !*failed && mbar_wait(q_empty, (items - 1) & 1));
                if (!ok) break;
                const int boxes_q = (w.tile.tokens > half_tokens ? TILES : 1) * C::kSlabs;
                if (lane == 0) mbar_arrive_expect_tx(q_full, boxes_q * half_tokens * a.group * 128);
                __syncwarp();
                if (lane < boxes_q)
                    tma_load_3d(smem + C::kQOff + lane * C::kSlab, &qmap, (lane % C::kSlabs) * 64, w.h * a.group,
                                w.tile.first + lane / C::kSlabs * half_tokens, q_full);
                ++items;
            }
            const int key = w.tile.block(w.unit) * kTreeKeys;
            const int y = boxes > 1 ? 0 : key & (page_size - 1);
            const int z = page < 0 ? -1 : page * a.p.kv_heads + w.h;
            const bool unclean = !tree_all_see(w.tile, a.window, a.sinks, key, key + kTreeKeys - 1);
            const uint32_t flag = (new_item ? kStepFirst : 0u) | (w.part_ends() ? kStepLast : 0u) |
                                  (w.range_ends(a) ? kStepFinal : 0u) | (w.tile.tokens > half_tokens ? kStepTwo : 0u);
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const uint32_t stage = issued % C::kStages;
                if (issued >= C::kStages)
                    ok = __all_sync(0xffffffffu, !*failed && mbar_wait(&empty[stage], phase_of(issued - C::kStages)));
                if (!ok) break;
                // a V tile with hidden keys goes through the cleaning warp
                uint64_t* bar = v == 1 && unclean ? &raw[stage] : &full[stage];
                if (lane == 0) {
                    if (v == 0) flags[stage] = flag;
                    mbar_arrive_expect_tx(bar, C::kTile);
                }
                __syncwarp();
                if (mine) tma_load_tile(ring(issued) + lane * box * 2 * D, v ? &vmap : &kmap, y >> 3, z, bar);
                if (v == 1 && unclean) raw_phase ^= 1u << stage, raw_open |= 1u << stage;
                else raw_open &= ~(1u << stage);
                ++issued;
            }
            new_item = w.part_ends();
            more = w.next(a, tile_tokens);
            if (more) page = page_of(w);
        }
        if (!ok) *failed = 1;
        // the copies issued must land before the CTA may exit
        if (items > 0) mbar_wait(q_full, (items - 1) & 1);
        for (uint32_t i = issued > C::kStages ? issued - C::kStages : 0; i < issued; ++i) {
            const uint32_t stage = i % C::kStages;
            if ((raw_open >> stage) & 1u)
                mbar_wait(&raw[stage], ((raw_phase >> stage) & 1u) ^ 1u);
            else
                mbar_wait(&full[stage], phase_of(i));
        }
        __syncwarp();
    } else if (warp == C::kCleanWarp) {
        // What the nodes of a tile see; V rows of keys that no row of the item sees:
        // zeros; values that are not finite in rows of keys that only some rows see: out
        uint32_t n = 0, raw_phase = 0, tiles = 0;
        int sight_b = -1, sight_t = 0;
        for (; more; more = w.next(a, tile_tokens), ++n) {
            if (w.b != sight_b || w.t != sight_t) {  // (the same for every kv head)
                sight_b = w.b, sight_t = w.t;
                const int nodes = w.span.base >= 0 ? w.tile.first - w.span.first + w.tile.tokens : 0;  // else it counts as empty
                int parent[kTreeWords];
#pragma unroll
                for (int k = 0; k < kTreeWords; ++k) {
                    const int i = 32 * k + lane;
                    parent[k] = i < nodes ? a.parents[w.span.first + i] : -1;
                }
                // (once the tile before is done with)
                if (tiles > 0 && !__all_sync(0xffffffffu, !*failed && mbar_wait(sight_free, (tiles - 1) & 1))) {
                    *failed = 1;
                    break;
                }
                ++tiles;
                find_sights(parent, nodes, w.span.base, a.window, a.sinks, sights, depths);
                if (lane == 0) mbar_arrive(sight_full);
            }
            const int key = w.tile.block(w.unit) * kTreeKeys;
            if (tree_all_see(w.tile, a.window, a.sinks, key, key + kTreeKeys - 1)) continue;
            const uint32_t stage = (2 * n + 1) % C::kStages;
            if (!__all_sync(0xffffffffu, !*failed && mbar_wait(&raw[stage], (raw_phase >> stage) & 1u))) {
                *failed = 1;
                break;
            }
            raw_phase ^= 1u << stage;
            uint8_t* tile = ring(2 * n + 1);
            // (eight lanes a row's 128 bytes: no two lanes in one bank)
            auto at = [&](int r, int slab) {
                return reinterpret_cast<uint4*>(tile + (r >> 3) * C::kGroup + slab * 1024 + (r & 7) * 128 + (lane & 7) * 16);
            };
            // Keys by intervals: no row sees those past the last node, nor those
            // before the first position's window that are not first tokens; some rows
            // see the tree's, and those that the window leaves from row to row.
            const Tile& t = w.tile;
            auto zero = [&](int from, int to) {
                for (int r = max(from - key, 0) + (lane >> 3); r < min(to - key, kTreeKeys); r += 4)
#pragma unroll
                    for (int slab = 0; slab < C::kSlabs; ++slab) *at(r, slab) = make_uint4(0u, 0u, 0u, 0u);
            };
            uint32_t bad = 0;
            auto search = [&](int from, int to) {
                const int end = min(to - key, kTreeKeys);
#pragma unroll 1
                for (int r = max(from - key, 0) + (lane >> 3); r < end; r += 16) {
                    uint4 v[4 * C::kSlabs];  // four rows' loads in flight (one past the end is its lane's first again)
#pragma unroll
                    for (int k = 0; k < 4 * C::kSlabs; ++k)
                        v[k] = *at(r + 4 * (k / C::kSlabs) < end ? r + 4 * (k / C::kSlabs) : r, k % C::kSlabs);
#pragma unroll
                    for (int k = 0; k < 4 * C::kSlabs; ++k)
                        bad |= not_finite<T>(v[k].x) | not_finite<T>(v[k].y) | not_finite<T>(v[k].z) | not_finite<T>(v[k].w);
                }
            };
            zero(t.p1 + 1, INT_MAX);
            search(t.p0, t.p1 + 1);
            if (a.window > 0) {
                zero(a.sinks, t.p0 - a.window + 1);
                search(max(t.p0 - a.window + 1, a.sinks), t.p1 - a.window + 1);
            }
            if (__any_sync(0xffffffffu, bad != 0)) {
#pragma unroll 1
                for (int r = lane >> 3; r < kTreeKeys; r += 4) {
                    if (tree_all_see(t, a.window, a.sinks, key + r, key + r)) continue;
#pragma unroll
                    for (int slab = 0; slab < C::kSlabs; ++slab) {
                        uint4 v = *at(r, slab);
                        v.x &= ~halves_of(not_finite<T>(v.x)), v.y &= ~halves_of(not_finite<T>(v.y));
                        v.z &= ~halves_of(not_finite<T>(v.z)), v.w &= ~halves_of(not_finite<T>(v.w));
                        *at(r, slab) = v;
                    }
                }
                *wild = 1;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[stage]);
        }
        __syncwarp();
    } else if (warp == C::kMmaWarp) {
        // The whole warp runs the loop on uniform values and one elected lane
        // issues: the MMAs' operands then stay in uniform registers.
        const uint32_t base = __shfl_sync(0xffffffffu, smem_addr(smem), 0) >> 4;
        constexpr uint64_t common = (1ull << 46) | (2ull << 61);
        constexpr uint64_t q_major = common | (1ull << 16) | (64ull << 32);
        constexpr uint64_t k_major = common | (1ull << 16) | (static_cast<uint64_t>(C::kGroup >> 4) << 32);
        constexpr uint64_t v_major = common | (64ull << 16) | (static_cast<uint64_t>(C::kGroup >> 4) << 32);
        const uint64_t q_desc = q_major | (base + (C::kQOff >> 4));
        const uint32_t t0 = __shfl_sync(0xffffffffu, tmem, 0);
        uint32_t stage = 0, phase = 0;  // of the ring: K's, then V's
        uint32_t c0 = 0, c1 = 0, q_items = 0;  // blocks of each tile so far
        bool fresh = true, issued = false;     // O has nothing of this part; S of this block is issued
        bool ok = !*failed && warp_wait(&full[0], 0);
        uint32_t flag = ok ? flags[0] : 0u;
        const bool none = (flag & kStepNone) != 0;
        if (none) ok = false;
        auto issue_s = [&](uint32_t i0, uint32_t i1, uint32_t k_stage, uint32_t f) {  // K and Q have landed
            tc_fence_after();
            if (elect_one()) {
                const uint64_t bd = k_major | (base + ((C::kRingOff + k_stage * C::kTile) >> 4));
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    if (t == 1 && !(f & kStepTwo)) break;
                    const uint32_t x = 2 * t + ((t ? i1 : i0) & 1), s_tmem = t0 + C::kSCol + kTreeKeys * x;
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t in_slab = 2 * (kk & 3), slab = kk >> 2;  // 16 values: 32 bytes
                        tc_mma_f16(s_tmem, q_desc + t * (C::kQTile >> 4) + slab * (C::kSlab >> 4) + in_slab,
                                   bd + slab * 64 + in_slab, chunk_idesc<T>(kTreeKeys, false), kk != 0);
                    }
                    tc_commit(&s_full[x]);
                }
                tc_commit(&empty[k_stage]);
                if (f & kStepLast) tc_commit(q_empty);
            }
            __syncwarp();
        };
        while (ok) {  // K of this block has landed
            const uint32_t k_stage = stage, n1 = c1 + (flag & kStepTwo ? 1 : 0);
            if (++stage == C::kStages) stage = 0, phase ^= 1u;
            const uint32_t v_stage = stage, v_phase = phase;
            if (++stage == C::kStages) stage = 0, phase ^= 1u;
            if (!issued) {
                if (flag & kStepFirst) ok = warp_wait(q_full, q_items++ & 1);
                if (!ok) break;
                issue_s(c0, c1, k_stage, flag);
            }
            // the next block's S as soon as its operands are there, and this one's P V
            uint32_t next_flag = 0, rounds = 0;
            bool landed = false, v_landed = false;  // the next block's K; this one's V
            uint32_t todo = TILES == 2 && (flag & kStepTwo) ? 3u : 1u;
            issued = false;
            PollClock clock;
            while (true) {
                if (!issued && !(flag & kStepFinal)) {
                    if (!landed && warp_test(&full[stage], phase)) {
                        landed = true;
                        next_flag = flags[stage];
                    }
                    if (landed && (!(next_flag & kStepFirst) || warp_test(q_full, q_items & 1))) {
                        if (next_flag & kStepFirst) ++q_items;
                        issue_s(c0 + 1, n1, stage, next_flag);
                        issued = true;
                    }
                }
                if (!v_landed) v_landed = warp_test(&full[v_stage], v_phase);
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    const uint32_t c = t ? c1 : c0, x = 2 * t + (c & 1);
                    if (!v_landed || !(todo & (1u << t)) || !warp_test(&p_full[x], (c >> 1) & 1)) continue;
                    todo &= ~(1u << t);
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t bd = v_major | (base + ((C::kRingOff + v_stage * C::kTile) >> 4));
                        const uint32_t s_tmem = t0 + C::kSCol + kTreeKeys * x, o_tmem = t0 + C::kOCol + 128 * t;
#pragma unroll
                        for (int kk = 0; kk < kTreeKeys / 16; ++kk)  // 16 keys: 8 columns of P, two 8-row groups of V
                            tc_mma_f16_ts(o_tmem, s_tmem + 8 * kk, bd + kk * (C::kGroup >> 3), chunk_idesc<T>(D, true),
                                          !fresh || kk != 0);
                        if (todo == 0) tc_commit(&empty[v_stage]);
                        tc_commit(&pv_done[x]);
                        if (flag & kStepLast) tc_commit(&o_full[t]);
                    }
                    __syncwarp();
                }
                if (todo == 0) break;
                if ((++rounds & 63) == 0 && __any_sync(0xffffffffu, *failed || poll_expired(clock))) {
                    ok = false;
                    break;
                }
            }
            if (!ok) break;
            fresh = (flag & kStepLast) != 0;
            if (flag & kStepFinal) break;
            if (!landed) {
                ok = warp_wait(&full[stage], phase);
                if (!ok) break;
                next_flag = flags[stage];
            }
            flag = next_flag;
            ++c0;
            c1 = n1;
        }
        if (!ok && !none) *failed = 1;
        if (elect_one()) tc_commit(mma_done);  // arrives once every MMA issued above has completed
        __syncwarp();
    } else {
        const int t = TILES == 1 ? 0 : warp >> 2, row = threadIdx.x & 127, quarter = warp & 3;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>(32 * quarter) << 16);
        const uint32_t o_col = lane_base + C::kOCol + 128 * t;
        const int node = row / a.group, head = row - node * a.group;
        bool ok = !*failed;
        bool begun = more && w.unit == 0;  // the item's first unit is in this range
        uint32_t n = 0, parts = 0, tiles = 0;
        int sight_b = -1, sight_t = 0;
        bool sighted = false;  // the tile's sights have come
        int pos = -1;
        while (ok && more) {
            const Tile tile = w.tile;
            const int base = tile.p0, first_row = tile.first + t * half_tokens, first_node = first_row - w.span.first;
            const int my_tokens = min(half_tokens, tile.tokens - t * half_tokens);
            const uint32_t* sight = sights + (first_node + node) * kTreeWords;  // this row's
            if (w.b != sight_b || w.t != sight_t) {  // (the same for every kv head)
                if (tiles > 0) {
                    // (each warp waits for every tile's sights, needed or not: none can count
                    // twice towards their release, however far it is ahead of the others)
                    if (!sighted) ok = warp_wait(sight_full, (tiles - 1) & 1);
                    if (!ok) break;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(sight_free);
                }
                sight_b = w.b, sight_t = w.t;
                ++tiles;
                sighted = false;
                pos = -1;
            }
            if (TILES == 2 && my_tokens <= 0) {  // the second tile has nothing to do for this item
                while (!w.part_ends()) w.next(a, tile_tokens);
                more = w.next(a, tile_tokens);
                begun = true;
                continue;
            }
            const bool valid = node < my_tokens;
            const bool live = 32 * quarter < my_tokens * a.group;  // of the warp: it has rows
            // Bits of the keys first .. first + 31 that the row sees.
            auto seen_bits = [&](int first) -> uint32_t {
                if (pos < 0) return 0u;
                uint32_t earlier = bits_below(base - first);
                if (a.window > 0) earlier &= ~bits_below(pos - a.window - first + 1) | bits_below(a.sinks - first);
                const int off = first - base;  // in the tree
                if (off <= -32 || off >= kTreeNodes) return earlier;
                if (off < 0) return earlier | (sight[0] << -off);
                const uint32_t low = sight[off >> 5], high = (off >> 5) + 1 < kTreeWords ? sight[(off >> 5) + 1] : 0u;
                return earlier | __funnelshift_r(low, high, off & 31);
            };
            float m = -INFINITY, l = 0.f, offset = 8.f;  // offset: 8 - b, or 8 where s - m is scaled
            bool done = false, huge = false;
            while (true) {
                const uint32_t x = 2 * t + (n & 1), s_col = lane_base + C::kSCol + kTreeKeys * x;
                ok = warp_wait(&s_full[x], (n >> 1) & 1);
                if (!ok) break;
                tc_fence_after();
                if (live) {
                    float v[kTreeKeys];
#pragma unroll
                    for (int c = 0; c < kTreeKeys; c += 16) tmem_ld16_nowait(s_col + c, v, c);
                    tmem_wait_regs(v);
                    const int key = tile.block(w.unit) * kTreeKeys;
                    if (!tree_all_see(tile, a.window, a.sinks, key, key + kTreeKeys - 1)) {
                        if (!sighted) {
                            ok = warp_wait(sight_full, (tiles - 1) & 1);
                            if (!ok) break;
                            sighted = true;
                            pos = valid && w.span.base >= 0 ? base + depths[first_node + node] : -1;
                        }
#pragma unroll
                        for (int c = 0; c < kTreeKeys; c += 32) {
                            const uint32_t bits = seen_bits(key + c);
#pragma unroll
                            for (int k = 0; k < 32; ++k) v[c + k] = (bits >> k) & 1u ? v[c + k] : -INFINITY;
                        }
                    }
                    float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                    for (int c = 4; c < kTreeKeys - 4; c += 8)
#pragma unroll
                        for (int k = 0; k < 4; ++k) top[k] = fmaxf(fmaxf(top[k], v[c + k]), v[c + k + 4]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) top[k] = fmaxf(top[k], v[kTreeKeys - 4 + k]);
                    const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                    const bool move = valid && (mx - m) * a.scale > 7.f;
                    if (__any_sync(0xffffffffu, move && m != -INFINITY)) {
                        // O at rest: P V of the block before (those before that were done before this S)
                        ok = warp_wait(&pv_done[x ^ 1], ((n - 1) >> 1) & 1);
                        if (!ok) break;
                        tc_fence_after();
                        const float f = move ? reference_factor(m, mx, a.scale) : 1.f;  // 0 for m = -inf, whose l and O are 0
                        l *= f;
                        rescale_row<D>(o_col, f);
                    }
                    if (__any_sync(0xffffffffu, move)) {
                        if (move) {
                            m = mx;
                            offset = __fsub_rn(8.f, __fmul_rn(m, a.scale));
                            if (is_huge(offset)) offset = 8.f;
                        }
                        huge = __any_sync(0xffffffffu, m != -INFINITY && is_huge_reference(__fmul_rn(m, a.scale))) != 0;
                    }
                    const uint64_t scale2 = pack2(a.scale, a.scale), offset2 = pack2(offset, offset);
                    if (huge) {
                        // (the scores less m, scaled: s - m here, the rest below; the other rows' as they are)
                        const float less = m != -INFINITY && is_huge_reference(__fmul_rn(m, a.scale)) ? -m : 0.f;
                        const uint64_t less2 = pack2(less, less);
#pragma unroll
                        for (int k = 0; k < kTreeKeys; k += 2) {
                            const float2 y = unpack2(add2(pack2(v[k], v[k + 1]), less2));
                            v[k] = y.x, v[k + 1] = y.y;
                        }
                    }
                    uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
                    for (int c = 0; c < kTreeKeys; c += 32) {
                        uint32_t p16[16];
#pragma unroll
                        for (int k = 0; k < 32; k += 2) {
                            const uint64_t p2 = exp2_pair(fma2(pack2(v[c + k], v[c + k + 1]), scale2, offset2));
                            sum[(k >> 1) & 1] = add2(sum[(k >> 1) & 1], p2);
                            const float2 p = unpack2(p2);
                            p16[k / 2] = Pair<T>::pack(p.x, p.y);
                        }
                        tmem_st16u(s_col + c / 2, p16, 0);  // (over scores that are read already)
                    }
                    const float2 sums = unpack2(add2(sum[0], sum[1]));
                    l += sums.x + sums.y;
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[x]);
                ++n;
                done = w.item_ends();
                if (w.part_ends()) break;
                w.next(a, tile_tokens);
            }
            if (!ok) break;

            // ---- the item's result, or this CTA's part of it -----------------------
            ok = warp_wait(&o_full[t], parts & 1);
            if (!ok) break;
            ++parts;
            tc_fence_after();
            const bool whole = begun && done;
            const float f = l == 0.f ? 0.f : whole ? 1.0f / l : 1.f;  // l = 0: saw no key
            constexpr int kPart = kChunkRows * (D + 2);
            // [D / 4][row] float4, then [row] (m, l): a warp's accesses are contiguous
            const long long my_part = static_cast<long long>(2 * blockIdx.x + (begun ? 1 : 0)) * TILES + t;
            float4* part = reinterpret_cast<float4*>(a.partials + my_part * kPart);
            if (live) {
                T* out_tile = static_cast<T*>(a.out) + first_row * a.out_stride + w.h * a.group * D;
                const long long my_place = valid ? node * a.out_stride + head * D : -1;
                long long to[4];  // the places of the quad's four rows
#pragma unroll
                for (int k = 0; k < 4; ++k) to[k] = __shfl_sync(0xffffffffu, my_place, (lane & 28) + k);
                // Columns c .. c + 31 of the values that the cleaning warp took out of
                // the blocks of this part, from the pages, where the row sees their key.
                auto add_wild = [&](float (&v)[32], int c) {
                    // the part's first unit, from the place of the item's unit 0 (a whole
                    // item has all its units here, and `left` may reach past the range)
                    const Range& r = *shared_range;
                    const int from = a.whole ? 0 : static_cast<int>(max(r.begin - (r.end - w.left - w.unit), 0ll));
                    for (int u = from; u <= w.unit; ++u) {
                        const int block = tile.block(u) * kTreeKeys;
                        for (int j = block; j < block + kTreeKeys; ++j) {
                            if (!tile_sees(tile, a.window, a.sinks, j) || tree_all_see(tile, a.window, a.sinks, j, j)) continue;
                            const int page = a.p.table[static_cast<long long>(w.b) * a.p.table_stride + (j >> a.p.page_shift)];
                            if (page < 0 || page >= a.p.pages) continue;
                            const long long at = ((static_cast<long long>(page) * a.p.kv_heads + w.h) << a.p.page_shift) +
                                                 (j & ((1 << a.p.page_shift) - 1));
                            const uint32_t* words = reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.v_pages) + at * D + c);
                            const bool sees = (seen_bits(j) & 1u) != 0u;
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                const uint32_t word = __ldg(words + k), which = not_finite<T>(word);
                                if (which == 0 || !sees) continue;
                                const float2 y = Pair<T>::unpack(word & halves_of(which));
                                v[2 * k] += y.x, v[2 * k + 1] += y.y;
                            }
                        }
                    }
                };
                const bool any_wild = __any_sync(0xffffffffu, *wild != 0);
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    float v[32];
                    tmem_ld16_nowait(o_col + c, v, 0);
                    tmem_ld16_nowait(o_col + c + 16, v, 16);
                    tmem_wait_regs(v);
#pragma unroll
                    for (int k = 0; k < 32; ++k) v[k] *= f;
                    if (any_wild) {
                        add_wild(v, c);
                        __syncwarp();
                    }
                    if (whole) {
                        uint32_t o16[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) o16[k] = Pair<T>::pack(v[2 * k], v[2 * k + 1]);
                        quad_transpose(o16);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (to[k] >= 0)
                                *reinterpret_cast<uint4*>(out_tile + to[k] + c + 8 * (lane & 3)) =
                                    make_uint4(o16[4 * k], o16[4 * k + 1], o16[4 * k + 2], o16[4 * k + 3]);
                    } else if (valid) {
#pragma unroll
                        for (int k = 0; k < 32; k += 4)
                            __stcg(part + ((c + k) / 4) * kChunkRows + row, make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]));
                    }
                }
            }
            tc_fence_before();  // (the next item's first P V follows this warp's next P)
            if (whole) {
                if (valid && a.lse != nullptr)
                    a.lse[static_cast<long long>(first_row + node) * a.heads + w.h * a.group + head] =
                        l == 0.f ? -INFINITY : (__fmul_rn(m, a.scale) - 8.f) * 0.6931471805599453f + logf(l);
            } else {
                if (valid) __stcg(reinterpret_cast<float2*>(part + D / 4 * kChunkRows) + row, make_float2(m, l));
                if (threadIdx.x == 0 && begun)  // the item's first part: what the join needs to know
                    a.entries[blockIdx.x] = make_int4(item_owners(*shared_range, w).y, tile.first, tile.tokens, w.h);
            }
            more = w.next(a, tile_tokens);
            begun = true;
        }
        if (!ok) *failed = 1;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == C::kMmaWarp) {
        // the MMAs must be complete before their tensor memory is released
        mbar_wait(mma_done, 0);
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kColumns) : "memory");
    }
}

// Joins the parts of the items that lie across CTAs, as paged_join_kernel does:
// block (c, tile * slices + slice) rows 16 slice .. of that tile of the item that begins last in CTA c. A warp
// holds 16 rows twice, for every other part each, and an eighth of the columns;
// the statistics and values of up to kJoinAhead parts are on their way together. The
// order of the sums is that of the CTAs, whichever came last. Maxima are scores.
constexpr int kTreeJoinThreads = 256, kJoinAhead = 2;

template <typename T, int D, int TILES>
__global__ void __launch_bounds__(kTreeJoinThreads) tree_join_kernel(const AttendArgs a) {
    constexpr int kPart = kChunkRows * (D + 2), kCols = D / 8 / 4;  // float4s a thread
    pdl_wait();
    const int4 entry = a.entries[blockIdx.x];
    const int c0 = blockIdx.x, c1 = entry.x;
    if (c1 < 0) return;
    const int lane = threadIdx.x & 31, side = lane >> 4, c = (threadIdx.x >> 5) * kCols;
    const int slices = gridDim.y / TILES, t = TILES == 1 ? 0 : blockIdx.y / slices;
    const int row = (blockIdx.y - t * slices) * kJoinRows + (lane & 15);
    const int node = row / a.group, head = row - node * a.group;
    const bool valid = node < min(a.half_tokens, entry.z - t * a.half_tokens);
    float top = -INFINITY, total = 0.f;
    float4 v[kCols];
#pragma unroll
    for (int k = 0; k < kCols; ++k) v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int cta = c0 + side; cta <= c1; cta += 2 * kJoinAhead) {
        float2 ml[kJoinAhead];
        float4 y[kJoinAhead][kCols];
#pragma unroll
        for (int u = 0; u < kJoinAhead; ++u) {
            const int which = cta + 2 * u;
            ml[u] = make_float2(-INFINITY, 0.f);
            if (which > c1 || !valid) continue;
            const float* part = a.partials + static_cast<long long>((2 * which + (which == c0)) * TILES + t) * kPart;
            ml[u] = __ldcg(reinterpret_cast<const float2*>(part + D * kChunkRows) + row);
#pragma unroll
            for (int k = 0; k < kCols; ++k) y[u][k] = __ldcg(reinterpret_cast<const float4*>(part) + (c + k) * kChunkRows + row);
        }
#pragma unroll
        for (int u = 0; u < kJoinAhead; ++u) {
            if (ml[u].y == 0.f) continue;  // saw no key
            const float most = fmaxf(top, ml[u].x);
            const float f = total == 0.f ? 0.f : reference_factor(top, most, a.scale), g = reference_factor(ml[u].x, most, a.scale);
            top = most;
            total = total * f + ml[u].y * g;
#pragma unroll
            for (int k = 0; k < kCols; ++k) {
                v[k].x = v[k].x * f + y[u][k].x * g, v[k].y = v[k].y * f + y[u][k].y * g;
                v[k].z = v[k].z * f + y[u][k].z * g, v[k].w = v[k].w * f + y[u][k].w * g;
            }
        }
    }
    // the two sides
    const float top1 = __shfl_down_sync(0xffffffffu, top, 16), total1 = __shfl_down_sync(0xffffffffu, total, 16);
    const float most = fmaxf(top, top1);
    const float f = total == 0.f ? 0.f : reference_factor(top, most, a.scale);
    const float g = total1 == 0.f ? 0.f : reference_factor(top1, most, a.scale);
    total = total * f + total1 * g;
    const float scale = total != 0.f ? 1.0f / total : 0.f;
    uint32_t words[2 * kCols];
#pragma unroll
    for (int k = 0; k < kCols; ++k) {
        const float4 w = make_float4(__shfl_down_sync(0xffffffffu, v[k].x, 16), __shfl_down_sync(0xffffffffu, v[k].y, 16),
                                     __shfl_down_sync(0xffffffffu, v[k].z, 16), __shfl_down_sync(0xffffffffu, v[k].w, 16));
        words[2 * k] = Pair<T>::pack((v[k].x * f + w.x * g) * scale, (v[k].y * f + w.y * g) * scale);
        words[2 * k + 1] = Pair<T>::pack((v[k].z * f + w.z * g) * scale, (v[k].w * f + w.w * g) * scale);
    }
    if (side != 0 || !valid) return;
    const long long out_row = entry.y + t * a.half_tokens + node;
    const int out_head = entry.w * a.group + head;
    T* out = static_cast<T*>(a.out) + out_row * a.out_stride + out_head * D + 4 * c;
#pragma unroll
    for (int k = 0; k < 2 * kCols; k += 4)
        *reinterpret_cast<uint4*>(out + 2 * k) = make_uint4(words[k], words[k + 1], words[k + 2], words[k + 3]);
    if (a.lse != nullptr && c == 0)
        a.lse[out_row * a.heads + out_head] =
            total == 0.f ? -INFINITY : (__fmul_rn(most, a.scale) - 8.f) * 0.6931471805599453f + logf(total);
}

template <typename T, int D, int ROWS, int TILES>
static int launch_tree_rows(AttendArgs a, const h4b_paged_kv* kv, int tile_tokens, int sms, cudaStream_t stream) {
    using C = TreeCfg<D, ROWS, TILES>;
    a.extra = kTreeExtra;
    a.least = kTreeLeast;
    a.half_tokens = tile_tokens;
    // Where no item can have many blocks (the tables' width bounds the lengths, which only
    // the device knows: wide tables leave items cut) they stay whole: no parts, and no
    // launch of the join, which the host needs 3 us for. A sequence counts as one item a kv
    // head here, though a large tree has several tiles. Cut and
    // whole, in us on the device: 8 items of 6 blocks 11.6 and 13.5, of 4 11.0 and 11.2;
    // 64 items of 6 14.9 and 14.3 (two tiles of rows 21.0 and 15.8), of 8 14.9 and 16.4;
    // 512 of 6 33.9 and 28.9, of 16 58.1 and 54.9 (95.6 and 95.0).
    const int ctas = C::kCtasPerSm * sms;
    const long long most = static_cast<long long>(a.p.table_stride) << a.p.page_shift;
    a.whole = most <= (static_cast<long long>(a.p.sequences) * a.p.kv_heads >= ctas ? kTreeWholeMany : kTreeWholeFew) * kTreeKeys;
    static std::atomic<bool> opted_in[kMaxDevices];
    int dev = 0;
    H4B_CUDA_TRY(cudaGetDevice(&dev));
    if (!opted_in[dev].load(std::memory_order_acquire)) {
        H4B_CUDA_TRY(cudaFuncSetAttribute(paged_attention_tree_kernel<T, D, ROWS, TILES>,
                                          cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
        opted_in[dev].store(true, std::memory_order_release);
    }
    CUtensorMap qmap, kmap, vmap;
    if (!paged_q_map(&qmap, a.q, kv, a.heads, a.group, tile_tokens, a.q_stride) ||
        !paged_kv_map(&kmap, a.k_pages, kv, kTreeKeys) || !paged_kv_map(&vmap, a.v_pages, kv, kTreeKeys))
        return H4B_EUNSUPPORTED;
    paged_attention_tree_kernel<T, D, ROWS, TILES><<<ctas, C::kThreads, C::kSmem, stream>>>(qmap, kmap, vmap, a);
    H4B_CUDA_TRY(cudaGetLastError());
    if (a.whole) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, TILES * ((tile_tokens * a.group + kJoinRows - 1) / kJoinRows));
    cfg.blockDim = dim3(kTreeJoinThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // it waits in the kernel
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    H4B_CUDA_TRY(cudaLaunchKernelEx(&cfg, tree_join_kernel<T, D, TILES>, a));
    return 0;
}

// Tiles with room for the rows of the largest tree: up to 64 leave room for a deeper
// ring of K and V; from 129 on, at head_dim 128, two tiles share the keys (trees of 64
// nodes and 4 q heads a kv head: 8 x 32768 tokens 370 -> 309 us, 64 ragged ones up to
// 2100 130 -> 108, one over 8000 29 -> 29; at head_dim 64 243 and 244, 93 and 90, and
// windowed trees 56 and 69).
template <typename T, int D>
static int launch_tree_tiles(const AttendArgs& a, const h4b_paged_kv* kv, int max_query, int sms, cudaStream_t stream) {
    const int most = kChunkRows / a.group;  // tokens of a tile
    const long long rows = static_cast<long long>(max_query) * a.group;
    if (rows <= 64) return launch_tree_rows<T, D, 64, 1>(a, kv, max_query, sms, stream);
    if constexpr (D == 128)
        if (max_query > most) return launch_tree_rows<T, D, 128, 2>(a, kv, most, sms, stream);
    return launch_tree_rows<T, D, 128, 1>(a, kv, std::min(most, max_query), sms, stream);
}

}  // namespace h4b
