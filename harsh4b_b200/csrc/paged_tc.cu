// Paged attention of long chunks on the 5th-generation tensor cores:
// tcgen05.mma kind::f16, fp32 accumulators in tensor memory, pages fetched by
// TMA. The split of the work over the CTAs and the visibility rules are those
// of paged.cu; partial results are joined by paged_join_kernel.
//
// An item is (sequence, 256 query rows, kv head): two tiles A and B of 128
// rows (128 / group tokens each, row = token * group + q head) that share
// every K/V tile of 128 keys. While the tensor cores work for one tile the
// softmax of the other runs. B is left out where A holds all tokens.
// Measured: an 8192-token prompt, 32 / 8 heads of 128, 588 to 602 us (913 to 935
// TFLOP/s) with the clock at the 1.65 GHz that the power cap leaves, 537 in a
// burst of a dozen; over 8K of history 1664 us (991 TFLOP/s), 1449 in a burst. Of
// the prompt's cycles the tensor pipe works in 52 %, the exponentials' unit in 53 %, and a
// first version without the softmax ran at 1604 TFLOP/s: what bounds it is how
// well one tile's softmax hides under the other's MMAs.
//
// Warps: 0-3 and 4-7 are the softmax of A and B (thread = query row, TMEM lane
// = thread), 8 issues the loads, 9 and 10 the MMAs of A and B, 11 cleans V
// tiles (below). Per key block n and tile x:
//   MMA:     S_x = Q_x K_n^T                              -> s_full[x]
//   softmax: S_x to registers, p; P_x over S_x    -> p_half[x] (64 keys), p_full[x]
//   MMA:     O_x += P_x V_n, then S_x of block n + 1 (the tensor cores run a
//            CTA's MMAs in issue order, so P_x is read before it is
//            overwritten)
// s_full of block n + 1 also stands for the completion of P V of block n: a
// commit tracks every earlier MMA. So a row may rescale its O after s_full,
// and o_full is needed only where an item (or the CTA's range) ends; o_free
// says that the softmax has read O and a new item may overwrite it.
//
// Operands: Q and the K/V ring in shared memory in the 128-byte swizzle
// layout, 64 values (128 bytes) of head_dim a row, one slab per 64; P in
// tensor memory. A K/V tile is 16 groups of 8 keys, each group its slabs of 8
// rows one after the other, so that a page of any size is one contiguous part
// of the tile and one 5-D box (64 values x 8 rows x slabs x groups x page): a
// box costs the copy engine about 50 cycles beside its bytes, and with boxes
// of one slab 16-token pages came at 24 bytes a cycle and SM, now at 34 (32
// KB tiles from L2, 148 SMs; 64-token pages 43 and 50). A tile's 128 keys are
// 128 / page_size boxes (or one box inside a page), issued by the lanes of the
// load warp at the same time; a page that is not there is a box outside the
// tensor, which reads as zeros. Q is one box per slab: group heads x 128 /
// group tokens.
//
// Softmax in base 2 with a lazily moved reference, as in the kernel of few
// rows: p = 2^(s - m). The scale is applied in one step with the subtraction;
// scores of 2^20 and more, where the rounding of m against that exact product
// would reach the exponent, take a slower way, scaled before it (a call, so that
// the usual way keeps its registers: the prompt 592 -> 602 us; with that code in
// the loop 612 to 688). P is rounded to
// the cache's type, which the MMA asks of an operand beside such a V; two halves
// a weight, as prompts over the other caches have them, would make the P V
// products twice as many where the tensor pipe is the longer half already. What
// the rounding does to the result is stated in paged.cu.
//
// Keys that no row of the item sees (past its last token, before its window)
// may lie in slots that hold anything: their scores are selected away, and
// their V rows are zeroed in shared memory before the product, since 0 * NaN
// would reach the sum. For the same reason infinities and NaN are taken out of
// the V rows that some rows of the item see and others do not (its own tokens,
// the window's edge); where there are any, the rows that see them get them
// added at the item's end, from the pages. A V tile with keys of either kind
// lands on a barrier of its own, warp 11 goes over it and then completes the
// tile's barrier in the loads' place.
//
// Every wait is bounded (mbar_wait). A role whose wait runs out marks the CTA
// as failed and stops; the load warp waits for the copies it issued, the MMA
// thread commits a last barrier, and the tensor memory is freed on every path.

namespace h4b {

constexpr int kChunkRows = 128, kChunkKeys = 128;
constexpr int kChunkLoadWarp = 8, kChunkMmaWarp = 9, kChunkCleanWarp = 11, kChunkThreads = 384;
// Places of a CTA's range, where there are few: a part of an item is written
// and read again, twice the bytes of a block's keys (303 tokens over 4400 of one
// kv head: 43 us with 1, 34 with 2 to 4; a 512-token prompt of 8: 21, 21, 22, 24).
constexpr int kChunkLeast = 2;
constexpr int kChunkExtra = 2;  // an item's start, end and pipeline fill, in units
// A step's flags: it has both tiles; first, last of its item in this range; last of all.
constexpr uint32_t kStepTwo = 1, kStepFirst = 2, kStepLast = 4, kStepFinal = 8;
constexpr uint32_t kStepNone = 16;  // the range held no unit
// Registers a thread: three warpgroups at the launch's 168 are shared out
// anew, 2 x 200 for the softmax (a row's 128 scores) and 104 for the others.
constexpr int kChunkSoftmaxRegs = 200, kChunkOtherRegs = 104;
static_assert(2 * kChunkSoftmaxRegs + kChunkOtherRegs <= 3 * 168, "registers of the CTA");

template <int D>
struct ChunkCfg {
    static constexpr int kSlabs = D / 64;                        // 64 values of head_dim each
    static constexpr int kSlab = 128 * 128;                      // of Q: 128 rows x 128 bytes
    static constexpr int kGroup = kSlabs * 1024;                 // of K or V: 8 keys, all slabs
    static constexpr int kTile = kSlabs * kSlab;                 // 128 keys (or query rows)
    static constexpr int kStages = D == 128 ? 5 : 10;
    static constexpr int kQOff = 0, kRingOff = 2 * kTile;
    static constexpr int kBarOff = kRingOff + kStages * kTile;
    static constexpr int kBars = 3 * kStages + 2 + 18 + 1;
    // barriers, words of the CTA, steps' flags, range, alignment slack
    static constexpr int kFlagOff = kBarOff + kBars * 8 + 16, kRangeOff = kFlagOff + kStages * 4 + 4 * (kStages & 1);
    static constexpr int kSmem = kRangeOff + sizeof(Range) + 1024;
    static constexpr uint32_t kSCol = 0, kOCol = 256;            // S_x at 128 x, O_x at 256 + 128 x
    static_assert(kSmem <= 232448, "shared memory per CTA");
};

// Instruction descriptors: D f32, A and B f16 (0) or bf16 (1), M 128.
template <typename T>
__host__ __device__ constexpr uint32_t chunk_idesc(int n, bool b_mn_major) {
    constexpr uint32_t format = Pair<T>::kBf16 ? 1u : 0u;
    return (1u << 4) | (format << 7) | (format << 10) | (b_mn_major ? 1u << 16 : 0u) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kChunkRows >> 4) << 24);
}

// Groups `group`.. of a page's head into a K/V tile.
__device__ __forceinline__ void tma_load_tile(void* dst, const CUtensorMap* map, int group, int page, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %2, %3, "
        "%4}], [%5];"
        ::"r"(smem_addr(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(group), "r"(page), "r"(smem_addr(bar))
        : "memory");
}

// True in one lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

// mbar_wait by a whole warp, with one answer for all its lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

// 4 x 4 transpose among the lanes of a quad: v[k] of lane i <-> v[i] of lane k.
// A row's 64 bytes then leave with one store of its quad; with one thread a
// row every store touched 32 rows and took 32 turns at the memory pipe.
__device__ __forceinline__ void quad_transpose(uint32_t (&v)[16]) {  // v[4 k + e]: word e of 16-byte unit k
#pragma unroll
    for (int step = 1; step <= 2; step <<= 1) {
        const bool odd = (threadIdx.x & step) != 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (k & step) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t low = v[4 * k + e], high = v[4 * (k | step) + e];
                const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? low : high, step);
                v[4 * k + e] = odd ? other : low;
                v[4 * (k | step) + e] = odd ? high : other;
            }
        }
    }
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ uint64_t exp2_pair(uint64_t y) {
    const float2 v = unpack2(y);
    return pack2(ex2_approx(v.x), ex2_approx(v.y));
}
// Whether every row of the tile sees keys `key` .. `end`.
__device__ __forceinline__ bool tile_all_see(const Tile& t, int window, int sinks, int key, int end) {
    return end <= t.p0 && (window <= 0 || key > t.p1 - window || end < sinks);
}
// Whether the block of keys from `key` on has one that some row of the tile does not see.
__device__ __forceinline__ bool has_hidden_keys(const Tile& t, int window, int sinks, int key) {
    return !tile_all_see(t, window, sinks, key, key + kChunkKeys - 1);
}

// Whether scores near this one need their product with the scale rounded on its own.
__device__ __forceinline__ bool is_huge(float score) { return fabsf(score) >= 1048576.f; }

// Bits 0 .. n - 1, of 32.
__device__ __forceinline__ uint32_t bits_below(int n) {
    return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u);
}

// A row's O times f. (P V of every earlier block has completed: see above.)
template <int D>
__device__ __forceinline__ void rescale_row(uint32_t o_col, float f) {
#pragma unroll 1
    for (int c = 0; c < D; c += 16) {  // rare: few registers beside the scores
        float v[16];
        tmem_ld16_nowait(o_col + c, v, 0);
        tmem_wait_regs(v);
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] *= f;
        tmem_st16(o_col + c, v, 0);
    }
}

// The softmax of a tile's row from a block on whose scores are huge for some row
// of the warp, to the end of the part: scaled before the subtraction, 32 at a
// time, the maximum first and then p. A call of its own, which leaves the usual
// way its registers. The first block's scores have come and its turn is taken.
struct HugeRow {
    Walk<kChunkKeys> w;
    float m, l;
    uint32_t s_count, turns;
    int pos;                  // -1: no row
    uint32_t s_col, o_col;
    bool ok;
};
template <typename T, int D>
__device__ __noinline__ void huge_scores(const AttendArgs& a, HugeRow& row, int half_tokens, uint64_t* s_full,
                                         uint64_t* p_half, uint64_t* p_full, uint64_t* my_turn, uint64_t* other_turn) {
    HugeRow r = row;
    const int lane = threadIdx.x & 31;
    const bool two = r.w.tile.tokens > half_tokens;
    const bool second = threadIdx.x >= 128;  // tile B, whose turns start one later
    while (true) {
        const int key = r.w.tile.block(r.w.unit) * kChunkKeys;
        auto scaled = [&](float (&v)[32], int c) {
            tmem_ld16_nowait(r.s_col + c, v, 0);
            tmem_ld16_nowait(r.s_col + c + 16, v, 16);
            tmem_wait_regs(v);
            uint32_t seen = bits_below(r.pos - key - c + 1);
            if (a.window > 0) seen &= ~bits_below(r.pos - a.window - key - c + 1) | bits_below(a.sinks - key - c);
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = (seen >> k) & 1u ? __fmul_rn(v[k], a.scale) : -INFINITY;
        };
        float v[32], mx = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < kChunkKeys; c += 32) {
            scaled(v, c);
#pragma unroll
            for (int k = 0; k < 32; ++k) mx = fmaxf(mx, v[k]);
        }
        const bool move = mx - r.m > kMostExponent;
        if (__any_sync(0xffffffffu, move && r.m != -INFINITY)) {
            const float f = move ? ex2_approx(r.m - softmax_reference(mx)) : 1.f;
            r.l *= f;
            rescale_row<D>(r.o_col, f);
        }
        if (move) r.m = softmax_reference(mx);
        const float base = r.m == -INFINITY ? 0.f : r.m;
#pragma unroll 1
        for (int c = 0; c < kChunkKeys; c += 32) {
            scaled(v, c);
            uint32_t p16[16];
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
                const float p0 = ex2_approx(__fsub_rn(v[k], base)), p1 = ex2_approx(__fsub_rn(v[k + 1], base));
                r.l += p0 + p1;
                p16[k / 2] = Pair<T>::pack(p0, p1);
            }
            tmem_st16u(r.s_col + c / 2, p16, 0);  // (over scores that are read already)
            if (c == kChunkKeys / 2 - 32 || c == kChunkKeys - 32) {
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(c < kChunkKeys / 2 ? p_half : p_full);
            }
        }
        if (lane == 0 && two) mbar_arrive(other_turn);
        if (r.w.part_ends()) break;
        r.w.next(a, 2 * half_tokens);
        r.ok = warp_wait(s_full, r.s_count & 1);
        if (!r.ok) break;
        ++r.s_count;
        tc_fence_after();
        if (two) {
            r.ok = warp_wait(my_turn, (r.turns - 1 + (second ? 1 : 0)) & 1);
            if (!r.ok) break;
            ++r.turns;
        }
    }
    row = r;
}

template <typename T, int D>
__global__ void __launch_bounds__(kChunkThreads, 1)
    paged_attention_chunk_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                                 const __grid_constant__ CUtensorMap vmap, const __grid_constant__ AttendArgs a) {
    using C = ChunkCfg<D>;
    extern __shared__ uint8_t chunk_smem_raw[];
    uint8_t* smem = chunk_smem_raw + ((1024u - (smem_addr(chunk_smem_raw) & 1023u)) & 1023u);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
    uint64_t* empty = full + C::kStages;
    uint64_t* raw = empty + C::kStages;  // a V tile on its way to the cleaning warp
    uint64_t* q_full = raw + C::kStages;
    uint64_t* q_empty = q_full + 1;
    uint64_t* s_full = q_empty + 1;  // [2]
    uint64_t* p_full = s_full + 2;   // [2]
    uint64_t* p_half = p_full + 2;   // [2]
    uint64_t* turn = p_half + 2;     // [2][4]: a warp may form its weights
    uint64_t* o_full = turn + 8;     // [2]
    uint64_t* o_free = o_full + 2;   // [2]
    uint64_t* mma_done = o_free + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
    volatile int* failed = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* wild = failed + 1;  // values that are not finite were taken out of a V tile
    volatile uint32_t* flags = reinterpret_cast<volatile uint32_t*>(smem + C::kFlagOff);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int half_tokens = kChunkRows / a.group, tile_tokens = 2 * half_tokens;
    Range* shared_range = reinterpret_cast<Range*>(smem + C::kRangeOff);
    {
        const Range r = find_range<kChunkThreads, kChunkKeys>(a, tile_tokens, smem);
        if (threadIdx.x == 0) {
            *shared_range = r;
            a.entries[blockIdx.x] = make_int4(-1, 0, 0, 0);
        }
        if (r.begin >= r.end) return;
    }

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 2);  // both tiles' MMA warps
            mbar_init(&raw[s], 1);
        }
        mbar_init(q_full, 1);
        mbar_init(q_empty, 2);
        for (int x = 0; x < 2; ++x) {
            mbar_init(&s_full[x], 1);
            mbar_init(&p_full[x], 4);
            mbar_init(&p_half[x], 4);
            for (int k = 0; k < 4; ++k) mbar_init(&turn[4 * x + k], 1);
            mbar_init(&o_full[x], 1);
            mbar_init(&o_free[x], 4);
        }
        mbar_init(mma_done, 2);
        *failed = wait_failed_before() ? 1 : 0;
        *wild = 0;
        fence_mbar_init();
    }
    if (warp == kChunkMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_addr(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    auto ring = [&](uint32_t i) { return smem + C::kRingOff + (i % C::kStages) * C::kTile; };
    auto phase = [&](uint32_t i) { return (i / C::kStages) & 1u; };

    // K of the CTA's step n is tile 2 n of the ring, V tile 2 n + 1. A step is a
    // unit; its flags lie beside K's barrier, written before K's copies start.
    // (Each role starts its walk after its registers are set: what is live
    // across setmaxnreg would be kept on the stack.)
    if (warp >= kChunkLoadWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kChunkOtherRegs));
        if (warp == kChunkLoadWarp) {
            Walk<kChunkKeys> w;
            const int page_size = 1 << a.p.page_shift, box = min(page_size, kChunkKeys);  // a box: keys of one page
            const int boxes = kChunkKeys / box;
            const bool mine = lane < boxes;  // each lane one box
            auto page_of = [&](const Walk<kChunkKeys>& u) -> int {  // -1: read as zeros
                const int key = u.tile.block(u.unit) * kChunkKeys + lane * box;
                const Tile& t = u.tile;
                if (!mine || key > t.p1 || !(a.window <= 0 || key + box - 1 > t.p0 - a.window || key < a.sinks)) return -1;
                const int page = a.p.table[static_cast<long long>(u.b) * a.p.table_stride + (key >> a.p.page_shift)];
                if (page >= 0 && page < a.p.pages) return page;
                report(kStatusBadPage);
                return -1;
            };
            uint32_t issued = 0, raw_open = 0, raw_phase = 0;  // a bit per stage
            bool ok = !*failed, more = w.start(a, *shared_range, tile_tokens);
            if (lane == 0) {
                asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kmap)) : "memory");
                asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&vmap)) : "memory");
                asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&qmap)) : "memory");
            }
            if (!more && lane == 0) {
                flags[0] = kStepNone;
                mbar_arrive(&full[0]);
            }
            int page = more ? page_of(w) : -1, items = 0;
            bool new_item = true;
            while (ok && more) {
                const int tiles = w.tile.tokens > half_tokens ? 2 : 1;
                if (new_item) {  // both tiles' q rows, once the previous item's are no longer read
                    if (items > 0) ok = __all_sync(0xffffffffu, !*failed && mbar_wait(q_empty, (items - 1) & 1));
                    if (!ok) break;
                    if (lane == 0)
                        mbar_arrive_expect_tx(q_full, tiles * C::kSlabs * half_tokens * a.group * 128);
                    __syncwarp();
                    if (lane < tiles * C::kSlabs) {
                        const int x = lane / C::kSlabs, my_slab = lane % C::kSlabs;
                        tma_load_3d(smem + C::kQOff + x * C::kTile + my_slab * C::kSlab, &qmap, my_slab * 64,
                                    w.h * a.group, w.tile.first + x * half_tokens, q_full);
                    }
                    ++items;
                }
                const int key = w.tile.block(w.unit) * kChunkKeys;
                const int y = boxes > 1 ? 0 : key & (page_size - 1);
                const int z = page < 0 ? -1 : page * a.p.kv_heads + w.h;
                const bool unclean = has_hidden_keys(w.tile, a.window, a.sinks, key);
                uint32_t flag = (tiles == 2 ? kStepTwo : 0u) | (new_item ? kStepFirst : 0u) | (w.part_ends() ? kStepLast : 0u);
                // the next step's page ids are on their way while this step's copies are issued
                new_item = w.part_ends();
                more = w.next(a, tile_tokens);
                if (more) page = page_of(w);
                if (!more) flag |= kStepFinal;
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const uint32_t stage = issued % C::kStages;
                    if (issued >= C::kStages)
                        ok = __all_sync(0xffffffffu, !*failed && mbar_wait(&empty[stage], phase(issued - C::kStages)));
                    if (!ok) break;
                    // a V tile with hidden keys goes through the cleaning warp
                    uint64_t* bar = v == 1 && unclean ? &raw[stage] : &full[stage];
                    if (lane == 0) {
                        if (v == 0) flags[stage] = flag;
                        mbar_arrive_expect_tx(bar, C::kTile);
                    }
                    __syncwarp();
                    if (mine)
                        tma_load_tile(ring(issued) + lane * box * 2 * D, v ? &vmap : &kmap, y >> 3, z, bar);
                    if (v == 1 && unclean) raw_phase ^= 1u << stage, raw_open |= 1u << stage;
                    else raw_open &= ~(1u << stage);
                    ++issued;
                }
            }
            if (!ok) *failed = 1;
            // the copies issued must land before the CTA may exit
            if (items > 0) mbar_wait(q_full, (items - 1) & 1);
            for (uint32_t i = issued > C::kStages ? issued - C::kStages : 0; i < issued; ++i) {
                const uint32_t stage = i % C::kStages;
                if ((raw_open >> stage) & 1u)
                    mbar_wait(&raw[stage], ((raw_phase >> stage) & 1u) ^ 1u);
                else
                    mbar_wait(&full[stage], phase(i));
            }
            __syncwarp();
        } else if (warp == kChunkCleanWarp) {
            // V rows of keys that no row of the item sees: zeros; values that are
            // not finite in rows of keys that only some rows see: out
            Walk<kChunkKeys> w;
            uint32_t n = 0, raw_phase = 0;
            bool more = w.start(a, *shared_range, tile_tokens);
            for (; more; more = w.next(a, tile_tokens), ++n) {
                const int key = w.tile.block(w.unit) * kChunkKeys;
                if (!has_hidden_keys(w.tile, a.window, a.sinks, key)) continue;
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
                // Keys by intervals: no row sees those past the last token, nor those
                // before the first row's window that are not first tokens; some rows
                // see the item's own tokens but the first, and those that the window
                // leaves from row to row.
                const Tile& t = w.tile;
                const bool windowed = a.window > 0;
                auto zero = [&](int from, int to) {
                    for (int r = max(from - key, 0) + (lane >> 3); r < min(to - key, kChunkKeys); r += 4)
#pragma unroll
                        for (int slab = 0; slab < C::kSlabs; ++slab) *at(r, slab) = make_uint4(0u, 0u, 0u, 0u);
                };
                uint32_t bad = 0;
                auto search = [&](int from, int to) {
                    const int end = min(to - key, kChunkKeys);
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
                search(t.p0 + 1, t.p1 + 1);
                if (windowed) {
                    zero(a.sinks, t.p0 - a.window + 1);
                    search(max(t.p0 - a.window + 1, a.sinks), t.p1 - a.window + 1);
                }
                if (__any_sync(0xffffffffu, bad != 0)) {
#pragma unroll 1
                    for (int r = lane >> 3; r < kChunkKeys; r += 4) {
                        if (tile_all_see(w.tile, a.window, a.sinks, key + r, key + r)) continue;
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
        } else {
            // The MMAs of tile x, one warp each, so that neither waits for the
            // other's softmax. A step without B is passed on by B's warp at once.
            // The whole warp runs the loop on uniform values and one elected
            // lane issues: the MMAs' operands then stay in uniform registers.
            const int x = __shfl_sync(0xffffffffu, warp, 0) - kChunkMmaWarp;
            // descriptors of byte 0 of shared memory; addresses are added in units of 16 bytes
            const uint32_t base = __shfl_sync(0xffffffffu, smem_addr(smem), 0) >> 4;
            // (swizzle 128 bytes; 8-row groups 1024 bytes apart in Q, kGroup in a K/V
            // tile; V, read along its rows, has its next 64 values 1024 bytes on)
            constexpr uint64_t common = (1ull << 46) | (2ull << 61);
            constexpr uint64_t q_major = common | (1ull << 16) | (64ull << 32);
            constexpr uint64_t k_major = common | (1ull << 16) | (static_cast<uint64_t>(C::kGroup >> 4) << 32);
            constexpr uint64_t v_major = common | (64ull << 16) | (static_cast<uint64_t>(C::kGroup >> 4) << 32);
            const uint64_t q_desc = q_major | (base + ((C::kQOff + x * C::kTile) >> 4));
            const uint32_t t0 = __shfl_sync(0xffffffffu, tmem, 0);
            const uint32_t s_tmem = t0 + C::kSCol + 128 * x, o_tmem = t0 + C::kOCol + 128 * x;
            uint32_t stage = 0, phase = 0;  // of the ring: K's, then V's
            uint32_t v_done = C::kStages;   // V stage whose release is due (none)
            uint32_t q_items = 0, o_items = 0, p_count = 0;
            bool ok = !*failed && warp_wait(&full[0], 0), first = false;
            uint32_t flag = ok ? flags[0] : 0u;
            if (flag & kStepNone) ok = false;
            bool none = (flag & kStepNone) != 0;
            while (ok) {  // K of this step has landed
                const bool active = x == 0 || (flag & kStepTwo);
                const uint32_t k_stage = stage;
                if (flag & kStepFirst) {
                    ok = warp_wait(q_full, q_items++ & 1);
                    if (!ok) break;
                    first = true;
                }
                tc_fence_after();
                if (elect_one()) {
                    if (active) {
                        const uint64_t bd = k_major | (base + ((C::kRingOff + k_stage * C::kTile) >> 4));
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk) {
                            const uint32_t in_slab = 2 * (kk & 3), slab = kk >> 2;  // 16 values: 32 bytes
                            tc_mma_f16(s_tmem, q_desc + slab * (C::kSlab >> 4) + in_slab, bd + slab * 64 + in_slab,
                                       chunk_idesc<T>(kChunkKeys, false), kk != 0);
                        }
                        tc_commit(&s_full[x]);
                    }
                    if (v_done < C::kStages) tc_commit(&empty[v_done]);
                    if (active) {
                        tc_commit(&empty[k_stage]);
                        if (flag & kStepLast) tc_commit(q_empty);
                    } else {
                        mbar_arrive(&empty[k_stage]);
                        if (flag & kStepLast) mbar_arrive(q_empty);
                    }
                }
                v_done = C::kStages;
                __syncwarp();
                if (++stage == C::kStages) stage = 0, phase ^= 1u;
                const uint32_t v_stage = stage, v_phase = phase;
                if (++stage == C::kStages) stage = 0, phase ^= 1u;
                ok = warp_wait(&full[v_stage], v_phase);
                // the next step's K now, so that its S follows this step's P V at once
                uint32_t next_flag = 0;
                if (ok && !(flag & kStepFinal)) {
                    ok = warp_wait(&full[stage], phase);
                    next_flag = flags[stage];
                }
                if (!ok) break;
                if (active) {
                    if (first && o_items > 0) ok = warp_wait(&o_free[x], (o_items - 1) & 1);
                    ok = ok && warp_wait(&p_half[x], p_count & 1);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t bd = v_major | (base + ((C::kRingOff + v_stage * C::kTile) >> 4));
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < kChunkKeys / 32; ++kk)  // 16 keys: 8 columns of P, two 8-row groups of V
                            tc_mma_f16_ts(o_tmem, s_tmem + 8 * kk, bd + kk * (C::kGroup >> 3), chunk_idesc<T>(D, true),
                                          !first || kk != 0);
                    }
                    __syncwarp();
                    ok = warp_wait(&p_full[x], p_count++ & 1);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int kk = kChunkKeys / 32; kk < kChunkKeys / 16; ++kk)
                            tc_mma_f16_ts(o_tmem, s_tmem + 8 * kk, bd + kk * (C::kGroup >> 3), chunk_idesc<T>(D, true), 1);
                        if (flag & kStepLast) tc_commit(&o_full[x]);
                        if (flag & kStepFinal) tc_commit(&empty[v_stage]);
                    }
                    v_done = v_stage;  // released after the next S, which nothing should hold up
                    if (flag & kStepLast) ++o_items;
                    first = false;
                } else if (lane == 0) {
                    mbar_arrive(&empty[v_stage]);
                }
                __syncwarp();
                if (flag & kStepFinal) break;
                flag = next_flag;
            }
            if (!ok && !none) *failed = 1;
            if (elect_one()) tc_commit(mma_done);  // arrives once every MMA issued above has completed
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kChunkSoftmaxRegs));
        Walk<kChunkKeys> w;
        bool more = w.start(a, *shared_range, tile_tokens);
        const int x = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lane_base = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
        const uint32_t s_col = lane_base + C::kSCol + 128 * x, o_col = lane_base + C::kOCol + 128 * x;
        const int token = row / a.group, head = row - token * a.group;
        bool ok = !*failed;
        bool begun = w.unit == 0;  // the item's first unit is in this range
        uint32_t s_count = 0, o_items = 0, turns = 0;
        while (ok && more) {
            const int my_tokens = min(half_tokens, w.tile.tokens - x * half_tokens);
            if (my_tokens <= 0) {  // B has nothing to do for this item
                while (!w.part_ends()) w.next(a, tile_tokens);
                more = w.next(a, tile_tokens);
                begun = true;
                continue;
            }
            const bool valid = token < my_tokens;
            const int pos = valid ? w.tile.p0 + x * half_tokens + token : -1;
            float m = -INFINITY, l = 0.f;
            bool done = false;
            while (true) {
                ok = warp_wait(&s_full[x], s_count & 1);
                if (!ok) break;
                ++s_count;
                tc_fence_after();
                constexpr int kHalf = kChunkKeys / 2;
                float s1[kHalf], s2[kHalf];  // the scores of the first and the last 64 keys
#pragma unroll
                for (int c = 0; c < kHalf; c += 16) tmem_ld16_nowait(s_col + c, s1, c);
                tmem_wait_regs(s1);
#pragma unroll
                for (int c = 0; c < kHalf; c += 16) tmem_ld16_nowait(s_col + kHalf + c, s2, c);
                const int key = w.tile.block(w.unit) * kChunkKeys;
                const bool all = !valid || (key + kChunkKeys - 1 <= pos &&
                                            (a.window <= 0 || key > pos - a.window || key + kChunkKeys - 1 < a.sinks));
                const bool masked = !__all_sync(0xffffffffu, all);
                auto mask = [&](float (&v)[kHalf], int first) {
                    // visible keys as bits, 32 at a time, and a select each: no branches
                    const int upto = pos - first + 1, from = a.window > 0 ? pos - a.window - first + 1 : 0;
                    const int sinks = a.window > 0 ? a.sinks - first : 0;
#pragma unroll
                    for (int c = 0; c < kHalf; c += 32) {
                        const uint32_t seen = bits_below(upto - c) & (~bits_below(from - c) | bits_below(sinks - c));
#pragma unroll
                        for (int k = 0; k < 32; ++k) v[c + k] = (seen >> k) & 1u ? v[c + k] : -INFINITY;
                    }
                };
                if (masked) mask(s1, key);
                // A and B take turns at the exponentials (warp w of each on one
                // sub-partition), so that one's run while the other's MMAs do.
                if (w.tile.tokens > half_tokens) {
                    if (x == 1 || turns > 0) ok = warp_wait(&turn[4 * x + (warp & 3)], (turns - 1 + x) & 1);
                    if (!ok) break;
                    ++turns;
                }
                uint64_t sum[2] = {0ull, 0ull};
                auto weights = [&](const float (&v)[kHalf], int column) {  // p of 64 keys, to the P columns
                    const float base = m == -INFINITY ? 0.f : -m;
                    const uint64_t scale2 = pack2(a.scale, a.scale), base2 = pack2(base, base);
#pragma unroll
                    for (int c = 0; c < kHalf; c += 32) {
                        uint32_t p16[16];
#pragma unroll
                        for (int k = 0; k < 32; k += 2) {
                            const uint64_t y = fma2(pack2(v[c + k], v[c + k + 1]), scale2, base2);
                            const uint64_t p2 = exp2_pair(y);
                            sum[(k >> 1) & 1] = add2(sum[(k >> 1) & 1], p2);
                            const float2 p = unpack2(p2);
                            p16[k / 2] = Pair<T>::pack(p.x, p.y);
                        }
                        tmem_st16u(s_col + column + c / 2, p16, 0);
                    }
                };
                auto largest = [&](const float (&v)[kHalf]) {
                    float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                    for (int c = 4; c < kHalf - 4; c += 8)
#pragma unroll
                        for (int k = 0; k < 4; ++k) top[k] = fmaxf(fmaxf(top[k], v[c + k]), v[c + k + 4]);
#pragma unroll
                    for (int k = 0; k < 4; ++k) top[k] = fmaxf(top[k], v[kHalf - 4 + k]);
                    return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                };
                // The first half's p with the m of the blocks before, while the
                // second half's scores arrive and the maximum is found beside
                // it. Where that passes m too far (always at a row's first
                // keys) m moves and they are formed anew.
                weights(s1, 0);
                const float mx1 = largest(s1);
                tmem_wait_regs(s2);
                if (masked) mask(s2, key + kHalf);
                const float mx = a.scale * fmaxf(mx1, largest(s2));
                const bool move = valid && mx - m > kMostExponent;
                if (__any_sync(0xffffffffu, move)) {
                    if (__any_sync(0xffffffffu, move && is_huge(mx))) {
                        // this block, with its scores put back, and the others go another way
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int c = 0; c < kHalf; c += 16) tmem_st16(s_col + c, s1, c);
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                        HugeRow row{w, m, l, s_count, turns, pos, s_col, o_col, true};
                        huge_scores<T, D>(a, row, half_tokens, s_full + x, p_half + x, p_full + x, turn + 4 * x + (warp & 3),
                                          turn + 4 * (x ^ 1) + (warp & 3));
                        w = row.w, m = row.m, l = row.l, s_count = row.s_count, turns = row.turns, ok = row.ok;
                        done = w.item_ends();
                        break;
                    }
                    if (__any_sync(0xffffffffu, move && m != -INFINITY)) {
                        const float f = move ? ex2_approx(m - softmax_reference(mx)) : 1.f;  // 0 for m = -inf, whose l and O are 0
                        l *= f;
                        rescale_row<D>(o_col, f);
                    }
                    if (move) m = softmax_reference(mx);
                    sum[0] = sum[1] = 0ull;
                    weights(s1, 0);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_half[x]);
                weights(s2, kHalf / 2);
                const float2 sums = unpack2(add2(sum[0], sum[1]));
                l += sums.x + sums.y;
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&p_full[x]);
                    if (w.tile.tokens > half_tokens) mbar_arrive(&turn[4 * (x ^ 1) + (warp & 3)]);
                }
                done = w.item_ends();
                if (w.part_ends()) break;
                w.next(a, tile_tokens);
            }
            if (!ok) break;
            ok = warp_wait(&o_full[x], o_items & 1);
            if (!ok) break;
            ++o_items;
            tc_fence_after();

            // ---- the tile's result, or this CTA's part of it -----------------
            const bool whole = begun && done;
            const long long out_row = w.tile.first + x * half_tokens + (valid ? token : 0);
            const int out_head = w.h * a.group + head;
            T* out_tile = static_cast<T*>(a.out) + (w.tile.first + x * half_tokens) * a.out_stride + w.h * a.group * D;
            const long long my_place = valid ? token * a.out_stride + head * D : -1;
            long long to[4];  // the places of the quad's four rows
#pragma unroll
            for (int k = 0; k < 4; ++k) to[k] = __shfl_sync(0xffffffffu, my_place, (lane & 28) + k);
            constexpr int kPart = kChunkRows * (D + 2);
            // [D / 4][row] float4, then [row] (m, l): a warp's accesses are contiguous
            float4* part = reinterpret_cast<float4*>(
                a.partials + (static_cast<long long>(2 * blockIdx.x + (begun ? 1 : 0)) * 2 + x) * kPart);
            const float inv = 1.0f / l;
            // Columns c .. c + 31 of the values that the cleaning warp took out of
            // the blocks of this part, from the pages, where the row sees their key.
            auto add_wild = [&](float (&v)[32], int c) {
                const Range& r = *shared_range;
                const long long first = r.end - w.left - w.unit;  // place of the item's unit 0
                for (int u = static_cast<int>(max(r.begin - first, 0ll)); u <= w.unit; ++u) {
                    const int block = w.tile.block(u) * kChunkKeys;
                    for (int j = block; j < block + kChunkKeys; ++j) {
                        if (!tile_sees(w.tile, a.window, a.sinks, j) || tile_all_see(w.tile, a.window, a.sinks, j, j)) continue;
                        const int page = a.p.table[static_cast<long long>(w.b) * a.p.table_stride + (j >> a.p.page_shift)];
                        if (page < 0 || page >= a.p.pages) continue;
                        const long long at = ((static_cast<long long>(page) * a.p.kv_heads + w.h) << a.p.page_shift) +
                                             (j & ((1 << a.p.page_shift) - 1));
                        const uint32_t* x = reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.v_pages) + at * D + c);
                        const bool sees = valid && j <= pos && (a.window <= 0 || j > pos - a.window || j < a.sinks);
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const uint32_t word = __ldg(x + k), which = not_finite<T>(word);
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
                if (any_wild) {
                    add_wild(v, c);
                    __syncwarp();
                }
                if (whole) {
                    uint32_t o16[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k)  // a row without keys: its O was never formed
                        o16[k] = l == 0.f ? 0u : Pair<T>::pack(v[2 * k] * inv, v[2 * k + 1] * inv);
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
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_free[x]);
            if (whole) {
                if (valid && a.lse != nullptr)
                    a.lse[out_row * a.heads + out_head] =
                        l == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(l);
            } else {
                if (valid)
                    __stcg(reinterpret_cast<float2*>(part + D / 4 * kChunkRows) + row, make_float2(m, l));
                if (threadIdx.x == 0 && begun)  // the item's first part: what the join needs to know
                    a.entries[blockIdx.x] = make_int4(item_owners(*shared_range, w).y, w.tile.first, w.tile.tokens, w.h);
            }
            more = w.next(a, tile_tokens);
            begun = true;
        }
        if (!ok) *failed = 1;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kChunkMmaWarp) {
        // the MMAs must be complete before their tensor memory is released
        mbar_wait(mma_done, 0);
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// Joins the parts of the items that lie across CTAs: block (c, tile * slices +
// slice) the item that begins last in CTA c, if it goes on in others, in the
// order of the CTAs. A launch of its own, on all SMs: one SM that reads an
// item's parts (64 KB a tile at head_dim 128) took as long as the products (64
// tokens over 16000: 60 us with the join in the CTA that ends last, 47 to 50
// so; an 8192-token prompt within 1 %).
constexpr int kJoinRows = 16, kJoinThreads = 128;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const AttendArgs a) {
    constexpr int kPart = kChunkRows * (D + 2), kCols = D / 8 / 4;  // float4s a thread
    pdl_wait();
    const int4 entry = a.entries[blockIdx.x];
    const int c0 = blockIdx.x, c1 = entry.x, x = blockIdx.y / (kChunkRows / kJoinRows);
    if (c1 < 0) return;
    const int row = (blockIdx.y % (kChunkRows / kJoinRows)) * kJoinRows + (threadIdx.x % kJoinRows);
    const int token = row / a.group, head = row - token * a.group;
    const int tokens = min(a.half_tokens, entry.z - x * a.half_tokens);
    if (token >= tokens) return;
    const int c = (threadIdx.x / kJoinRows) * kCols;
    auto part_of = [&](int cta) {
        return a.partials + (static_cast<long long>(2 * cta + (cta == c0)) * 2 + x) * kPart;
    };
    auto stat = [&](int cta) { return __ldcg(reinterpret_cast<const float2*>(part_of(cta) + D * kChunkRows) + row); };
    float most = -INFINITY, total = 0.f;
#pragma unroll 4
    for (int cta = c0; cta <= c1; ++cta) most = fmaxf(most, stat(cta).x);
    float4 v[kCols];
#pragma unroll
    for (int k = 0; k < kCols; ++k) v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int cta = c0; cta <= c1; ++cta) {
        const float2 ml = stat(cta);  // l = 0: saw no key
        const float f = ml.y == 0.f ? 0.f : ex2_approx(ml.x - most);
        total += ml.y * f;
        const float4* o = reinterpret_cast<const float4*>(part_of(cta));
#pragma unroll
        for (int k = 0; k < kCols; ++k) {
            const float4 y = __ldcg(o + (c + k) * kChunkRows + row);
            v[k].x += y.x * f, v[k].y += y.y * f, v[k].z += y.z * f, v[k].w += y.w * f;
        }
    }
    const float scale = total != 0.f ? 1.0f / total : 0.f;
    const long long out_row = entry.y + x * a.half_tokens + token;
    const int out_head = entry.w * a.group + head;
    T* out = static_cast<T*>(a.out) + out_row * a.out_stride + out_head * D + 4 * c;
#pragma unroll
    for (int k = 0; k < kCols; k += 2)
        *reinterpret_cast<uint4*>(out + 4 * k) =
            make_uint4(Pair<T>::pack(v[k].x * scale, v[k].y * scale), Pair<T>::pack(v[k].z * scale, v[k].w * scale),
                       Pair<T>::pack(v[k + 1].x * scale, v[k + 1].y * scale),
                       Pair<T>::pack(v[k + 1].z * scale, v[k + 1].w * scale));
    if (a.lse != nullptr && c == 0)
        a.lse[out_row * a.heads + out_head] =
            total == 0.f ? -INFINITY : most * 0.6931471805599453f + logf(total);
}

// A layer's pages [pages * kv_heads][page_size][D] as a 5-D tensor map (value,
// row of its group of 8, slab of 64 values, group, page and head).
static bool paged_kv_map(CUtensorMap* out, const void* base, const h4b_paged_kv* kv) {
    auto encode = tensor_map_encoder();
    if (!encode) return false;
    const cuuint64_t row = kv->head_dim * 2ull;
    const cuuint32_t slabs = kv->head_dim / 64, box_rows = kv->page_size < kChunkKeys ? kv->page_size : kChunkKeys;
    const cuuint64_t dims[5] = {64, 8, slabs, static_cast<cuuint64_t>(kv->page_size) / 8,
                                static_cast<cuuint64_t>(kv->pages) * kv->kv_heads};
    const cuuint64_t strides[4] = {row, 128, 8 * row, kv->page_size * row};
    const cuuint32_t box[5] = {64, 8, slabs, box_rows / 8, 1};
    const cuuint32_t elem[5] = {1, 1, 1, 1, 1};
    return encode(out, kv->dtype == H4B_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
                  const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The q rows [tokens][heads][D] with boxes of 64 values x group heads x
// 128 / group tokens: a tile's rows in their order.
static bool paged_q_map(CUtensorMap* out, const void* base, const h4b_paged_kv* kv, int heads, int group,
                        long long q_stride) {
    auto encode = tensor_map_encoder();
    if (!encode) return false;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(kv->head_dim), static_cast<cuuint64_t>(heads),
                                static_cast<cuuint64_t>(kv->tokens)};
    const cuuint64_t strides[2] = {kv->head_dim * 2ull, static_cast<cuuint64_t>(q_stride) * 2};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(kChunkRows / group)};
    const cuuint32_t elem[3] = {1, 1, 1};
    return encode(out, kv->dtype == H4B_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                  const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
static int launch_chunk(AttendArgs a, const h4b_paged_kv* kv, int sms, cudaStream_t stream) {
    using C = ChunkCfg<D>;
    a.extra = kChunkExtra;
    a.least = kChunkLeast;
    static std::atomic<bool> opted_in[kMaxDevices];
    int dev = 0;
    H4B_CUDA_TRY(cudaGetDevice(&dev));
    if (!opted_in[dev].load(std::memory_order_acquire)) {
        H4B_CUDA_TRY(cudaFuncSetAttribute(paged_attention_chunk_kernel<T, D>,
                                          cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
        opted_in[dev].store(true, std::memory_order_release);
    }
    CUtensorMap qmap, kmap, vmap;
    if (!paged_q_map(&qmap, a.q, kv, a.heads, a.group, a.q_stride) || !paged_kv_map(&kmap, a.k_pages, kv) ||
        !paged_kv_map(&vmap, a.v_pages, kv))
        return H4B_EUNSUPPORTED;
    a.half_tokens = kChunkRows / a.group;
    paged_attention_chunk_kernel<T, D><<<sms, kChunkThreads, C::kSmem, stream>>>(qmap, kmap, vmap, a);
    H4B_CUDA_TRY(cudaGetLastError());
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sms, 2 * kChunkRows / kJoinRows);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // it waits in the kernel
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    H4B_CUDA_TRY(cudaLaunchKernelEx(&cfg, paged_join_kernel<T, D>, a));
    return 0;
}

}  // namespace h4b
