// Attention of chunks of new tokens over a paged cache (pb_chunk_attn): part of lm_attn.cu, whose kernel for few rows, exponentials and products it uses.
//
//   out[r][h] = sum_j softmax_j(scale * q[r][h] . k_j) v_j   over the tokens that row r sees: up to its own position, with a window the last of them
//
// A launch whose sequences have few rows (new tokens x heads of a key head: up to 16, or one new token) is own_kernel's, which is bound by reading the cache (64 sequences of one token behind up to 8000: 180 us,
// 5.8 TB/s), unless they are so few and max_len is so large that its blocks could not read as fast as all SMs.  Otherwise the rows of a sequence's query heads that share a key head are cut into pairs of tiles of 128, which meet the keys and values in tiles of 128 on the tensor cores (chunk_kernel): the
// arithmetic of prefix_kernel, with a mask where a tile holds keys that not all rows see.  Bound by the products and the softmax beside them, which share shared memory and issue slots: 3950 clocks for a pair and 128 keys,
// of which the products alone take 2048 (a prompt of 8192 tokens of 8 x 4 heads of 128: 530 us, 1.04 PFLOP/s; 2048 tokens behind 65000: 2000 us, 1.1 PFLOP/s, both for a few milliseconds; launches that go on
// for a second run at 1.68 and 1.62 GHz under the power limit: 602 us, 913 TFLOP/s, and 2280 us, 972 TFLOP/s).
//
// Pairs differ in the keys that they see, and sequences in everything, all of which only the device knows.  So a block lays out the work first (plan_kernel): every pair's cost is known, all pairs for
// all key heads stand in a row, and the row is cut into equal ranges, wherever that cuts a pair's keys.  A pair that is cut leaves a part of its sums with
// each range, and join_kernel puts them together; the others are written at once.  (Under the counters, which start from cold and wait for each kernel, plan takes
// 9 us and join 11 to 17, 40 where it reads the 110 MB of parts that 2048 tokens behind 65000 leave.)
#pragma once

namespace pb {
namespace {

constexpr int kFewRows = 16, kChunkBlocks = 148, kMaxRounds = 4, kJoinSlices = 8;

// 256 rows of a sequence (fewer at its end), for every key head.
struct alignas(16) ChunkUnit {
    int32_t b, start, rows, first;       // the sequence, its first row of q, its rows, the position of its first token
    int32_t row0, tile0, tiles, end;     // its row here; the tiles of 128 keys from the first that any of these rows sees; the end of what they see
};
static_assert(sizeof(ChunkUnit) == 32, "eight words, one a lane");
struct alignas(16) ChunkCut {            // where a range begins
    int32_t unit, head, step, pad;
    ChunkUnit begins;                    // a copy of that unit, so that a block has it in one access
};

struct ChunkArgs {
    const void *q, *k, *v;
    void* out;
    const int32_t *block_table, *starts, *lens;
    int64_t q_stride, q_head, out_stride, out_head, page_stride, token_stride, head_stride, table_stride;
    int batch, tokens, q_heads, kv_heads, group, D, page, n_pages, max_new, max_len, window, box_rows;
    int few, few_ranks;                  // rows of a sequence that own_kernel may take (0: none), the blocks that it would have for one and a key head
    int q_boxes;                         // a row tile's queries are boxes of a tensor map (whole tokens to a tile, positive strides and scale)
    float scale;
    int max_units, max_ranges;
    ChunkUnit* units;
    int64_t* before;                     // [max_units + 1]: costs of the units in front
    ChunkCut* cuts;                      // [max_ranges + 1]
    int32_t* counts;                     // units, ranges, rows of a sequence that own_kernel takes
    int32_t* counted;                    // [batch + 1]: the starts as they count
    float4* part_o;                      // [2 max_ranges][2][DP / 4][128]
    float2* part_ml;                     // [2 max_ranges][2][128]: (m, l)
};

// Costs: a step of two row tiles, of one, and what a pair costs beside its steps: queries, first scores, results, some 9000 clocks.  (A prompt of 8192 tokens with 6, 9, 12 for that: 537, 522, 527 us.)
constexpr int kCostTwo = 4, kCostOne = 3, kCostPair = 9;

__device__ __forceinline__ int ceil_pos(int x, int d) { return x > 0 ? (x + d - 1) / d : 0; }

// The starts as they count: not below 0, above `tokens` or below one in front of them, so that no two sequences have a row in common and the units fit.  A block of 1024 threads; whether a start fell.
__device__ __forceinline__ bool count_starts(const ChunkArgs& a) {
    __shared__ int s_high[32];
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    bool fell = false, other = false;
    for (int b = t; b <= a.batch; b += 1024) {
        const int s = __ldcg(a.starts + b), before = __ldcg(a.starts + max(b - 1, 0)), counts = min(max(s, 0), a.tokens);
        a.counted[b] = counts;
        fell |= s < before;
        other |= s != counts;
    }
    if (fell || other) atomicExch(&g_attn_flag, kFlagLmLength);
    if (!__syncthreads_or(fell)) return false;
    const auto highest = [&](int x) {                                    // of the lanes up to this one
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x = max(x, y);
        }
        return x;
    };
    int ahead = 0;
    for (int b0 = 0; b0 <= a.batch; b0 += 1024) {
        const bool there = b0 + t <= a.batch;
        const int s = highest(there ? a.counted[b0 + t] : 0);            // (which this thread wrote)
        if (lane == 31) s_high[warp] = s;
        __syncthreads();
        const int warps = highest(s_high[lane]), in_front = __shfl_sync(0xffffffffu, warps, max(warp - 1, 0));
        if (there) a.counted[b0 + t] = max(max(s, ahead), warp ? in_front : 0);
        ahead = max(ahead, __shfl_sync(0xffffffffu, warps, 31));
        __syncthreads();
    }
    return true;
}

// In front of own_kernel alone, where a warp of it does not look through all starts (kGivenStarts).
__global__ void __launch_bounds__(1024) starts_kernel(const __grid_constant__ ChunkArgs a) {
    griddep_wait();
    griddep_launch();
    count_starts(a);
}

// The work: units, their costs, and the ranges.  One block, which the others wait for: a thread a sequence, a unit, a range, with all that is looked up in shared memory as long as there are no more than
// kPlanUnits units.
constexpr int kPlanUnits = 2048;
__global__ void __launch_bounds__(1024) plan_kernel(const __grid_constant__ ChunkArgs a) {
    __shared__ int64_t s_scan[2][32], s_before[kPlanUnits + 1];
    __shared__ int s_base[1025];
    __shared__ ChunkSeq s_seq[1024];
    __shared__ int s_tiles[kPlanUnits];            // tiles, twice, and whether there are two row tiles
    __shared__ int s_most[3];                      // sequences of few rows, the most tokens that one's rows see; the highest cost of a unit
    griddep_wait();
    griddep_launch();
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const bool in_shared = a.max_units <= kPlanUnits;
    int turn = 0;
    const auto scan_warp = [&](int64_t x) {
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        return x;
    };
    // Sums of the threads up to this one, and of all.
    const auto scan = [&](int64_t x, int64_t& all) {
        x = scan_warp(x);
        if (lane == 31) s_scan[turn][warp] = x;
        __syncthreads();
        const int64_t warps = scan_warp(s_scan[turn][lane]);
        turn ^= 1;                                 // (who writes there again has passed the next barrier, and with it everyone has read)
        all = __shfl_sync(0xffffffffu, warps, 31);
        const int64_t ahead = __shfl_sync(0xffffffffu, warps, max(warp - 1, 0));
        return x + (warp ? ahead : 0);
    };
    // Sequences of few rows: own_kernel goes through the cache faster for all of them together, but has a sequence's tokens for a few blocks only.  In nanoseconds: some 40 bytes each for a block, 6000 for all
    // of them, 5000 to begin with; here 1600 for a tile of keys and 5000 for an item, on all SMs.  (24 sequences of up to 17 new tokens behind 4000, six of which have few rows: 98 us with own_kernel, 65 without.)
    ChunkSeq own = {0, 0, 0};                      // of the thread's first sequence
    if (t < a.batch) own = chunk_seq(ChunkGiven(a.starts, a.lens, t), 0, a.tokens, a.max_new, a.max_len, true);
    if (t < 3) s_most[t] = 0;
    if (count_starts(a) && t < a.batch) own = chunk_seq(ChunkGiven(a.counted, a.lens, t), 0, a.tokens, a.max_new, a.max_len, true);
    int few = 0;
    if (a.few) {
        int many = 0, most = 0;
        for (int b = t; b < a.batch; b += 1024) {
            const ChunkSeq s = b == t ? own : chunk_seq(ChunkGiven(a.counted, a.lens, b), 0, a.tokens, a.max_new, a.max_len, false);
            if (s.rows == 0 || s.rows * a.group > a.few) continue;
            ++many;
            most = max(most, max(s.first + s.rows, 0) - (a.window ? max(s.first + 1 - a.window, 0) : 0));
        }
        many = __reduce_add_sync(0xffffffffu, many);
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0 && many) {
            atomicAdd(&s_most[0], many);
            atomicMax(&s_most[1], most);
        }
        __syncthreads();
        // (all as long as the longest)
        const float each = 4.f * a.D * s_most[1], all = (float)s_most[0] * a.kv_heads, there = fmaxf(all * each / 6000.f, each / (40.f * a.few_ranks)) + 5000.f;
        if (there < all * (s_most[1] * (1600.f / 128.f) + 5000.f) / kChunkBlocks) few = a.few;
    }
    int units = 0;
    int64_t sum = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 1024) {
        int mine = 0;
        if (b0 + t < a.batch) {
            const ChunkSeq s = b0 == 0 ? own : chunk_seq(ChunkGiven(a.counted, a.lens, b0 + t), 0, a.tokens, a.max_new, a.max_len, true);
            const int rows = s.rows * a.group;
            mine = rows > few ? (rows + 255) / 256 : 0;
            s_seq[t] = s;
        }
        int64_t all;
        const int64_t upto = scan(mine, all);
        s_base[t] = (int)min((long long)(upto - mine), 0x7fffffffLL);
        const int here = (int)min((long long)all, (long long)(a.max_units - units)), n = min(1024, a.batch - b0);      // (all of them fit, as long as starts and lens do not change meanwhile)
        __syncthreads();
        for (int i0 = 0; i0 < here; i0 += 1024) {
            const int i = i0 + t;
            int64_t cost = 0;
            int tiles = 0;
            if (i < here) {
                int lo = 0, hi = n - 1;            // the last sequence whose units begin at or in front of this one (sequences without units share their beginning with the next)
                while (lo < hi) {
                    const int mid = (lo + hi + 1) / 2;
                    if (s_base[mid] <= i) lo = mid;
                    else hi = mid - 1;
                }
                const ChunkSeq s = s_seq[lo];
                ChunkUnit u;
                u.b = b0 + lo; u.start = s.start; u.rows = s.rows * a.group; u.first = s.first; u.row0 = 256 * (i - s_base[lo]);
                const int pos0 = s.first + u.row0 / a.group, pos1 = s.first + (min(u.row0 + 256, u.rows) - 1) / a.group;
                u.end = max(pos1 + 1, 0);
                u.tile0 = a.window ? max(pos0 - a.window + 1, 0) / 128 : 0;
                u.tiles = max((u.end + 127) / 128 - u.tile0, 0);
                a.units[units + i] = u;
                const bool two = u.row0 + 128 < u.rows;
                cost = kCostPair + (int64_t)u.tiles * (two ? kCostTwo : kCostOne);
                tiles = 2 * u.tiles + two;
            }
            const int highest = __reduce_max_sync(0xffffffffu, (int)min((long long)cost, 1LL << 30));
            if (lane == 0) atomicMax(&s_most[2], highest);
            int64_t chunk;
            const int64_t before = sum + scan(cost, chunk) - cost;
            if (i < here) {
                if (in_shared) { s_before[units + i] = before; s_tiles[units + i] = tiles; }
                else a.before[units + i] = before;
            }
            sum += chunk;
        }
        units += here;
        __syncthreads();
    }
    const int64_t total = sum * a.kv_heads;
    // Ranges: one for each block, several where they are long (so that the blocks are at the same keys at the same time, and those come from the L2 cache), fewer where there is little to do.
    const long long rounds = min(max((long long)total / (kChunkBlocks * 400), 1LL), (long long)(a.max_ranges / kChunkBlocks));
    int N = (int)min(kChunkBlocks * rounds, max((long long)total / (kCostPair + 3 * kCostTwo), 1LL));
    // A pair for each block where they are few and short: cuts would cost more than they even out.  (512 tokens of 8 x 4 heads 23 us, cut 31.)
    const bool whole = (int64_t)units * a.kv_heads <= kChunkBlocks && s_most[2] <= kCostPair + 8 * kCostTwo;
    if (whole) N = units * a.kv_heads;
    for (int r = t; r <= N; r += 1024) {
        ChunkCut c = {0, a.kv_heads, 0, 0, {}};
        if (r < N && whole) {
            c.head = r / units;
            c.unit = r - c.head * units;
            c.begins = a.units[c.unit];
        } else if (r < N) {
            // (quotients of 64 bits take some hundred instructions each)
            const bool small = total < (1LL << 32) / (kChunkBlocks * kMaxRounds);
            const int64_t w = small ? (uint32_t)total * (uint32_t)r / (uint32_t)N : total * r / N;
            c.head = small ? (uint32_t)w / (uint32_t)sum : (int)(w / sum);
            const int64_t rest = w - c.head * sum;
            const int64_t* table = in_shared ? s_before : a.before;
            int lo = 0, hi = units - 1;            // the last unit that begins at or in front of it
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (table[mid] <= rest) lo = mid;
                else hi = mid - 1;
            }
            c.unit = lo;
            c.begins = a.units[lo];
            const int tiles = in_shared ? s_tiles[lo] >> 1 : c.begins.tiles;
            const int each = (in_shared ? s_tiles[lo] & 1 : c.begins.row0 + 128 < c.begins.rows) ? kCostTwo : kCostOne, near = (int)min((long long)total / N / (8 * each), 2LL);
            const int step = (int)(max((long long)(rest - table[lo] - kCostPair), 0LL) / each);
            if (step > near && step < tiles - near) {
                c.step = step;
            } else if (step > near || 2 * step > tiles) {                // a cut near a pair's end is none
                if (++c.unit == units) { c.unit = 0; ++c.head; }
                c.begins = a.units[c.unit];
            }
        }
        a.cuts[r] = c;
    }
    if (t == 0) { a.counts[0] = units; a.counts[1] = N; a.counts[2] = few; }
}

// The parts of a block's ranges, one after the other.
struct ChunkItem {
    int b, start, rows, first, row0, tile0, tiles, end, head, from, to, slot;      // slot: of the part that it leaves, -1 if it is whole
};
struct ChunkWalk {
    const ChunkArgs& a;
    int range, units, ranges, unit, head, step, to_unit, to_head, to_step, word;
    __device__ __forceinline__ ChunkWalk(const ChunkArgs& args) : a(args) {
        range = (int)blockIdx.x;
        begin();                         // (what lies there if there are fewer ranges is not used)
        units = __ldcg(a.counts);
        ranges = __ldcg(a.counts + 1);
    }
    __device__ __forceinline__ void begin() {
        const int4 c = __ldcg(reinterpret_cast<const int4*>(a.cuts + range)), d = __ldcg(reinterpret_cast<const int4*>(a.cuts + range + 1));
        word = __ldcg(reinterpret_cast<const int32_t*>(&a.cuts[range].begins) + (threadIdx.x & 7));
        unit = c.x; head = c.y; step = c.z; to_unit = d.x; to_head = d.y; to_step = d.z;
    }
    __device__ __forceinline__ bool next(ChunkItem& x) {                 // a whole warp
        while (true) {
            if (range >= ranges) return false;
            const bool in_last = head == to_head && unit == to_unit;
            if (head > to_head || (head == to_head && unit > to_unit) || (in_last && step >= to_step)) {
                range += (int)gridDim.x;
                if (range < ranges) begin();
                continue;
            }
            int32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __shfl_sync(0xffffffffu, word, i);
            x.b = w[0]; x.start = w[1]; x.rows = w[2]; x.first = w[3]; x.row0 = w[4]; x.tile0 = w[5]; x.tiles = w[6]; x.end = w[7];
            x.head = head; x.from = step; x.to = in_last ? to_step : x.tiles;
            x.slot = x.from > 0 ? 2 * range : x.to < x.tiles ? 2 * range + 1 : -1;
            step = 0;
            if (++unit == units) { unit = 0; ++head; }
            word = __ldcg(reinterpret_cast<const int32_t*>(a.units + unit) + (threadIdx.x & 7));       // the next one's, in time
            return true;
        }
    }
};

// Registers that a load from tensor memory wrote, behind its wait: what uses them stays behind it, too.
__device__ __forceinline__ void pin(uint32_t (&r)[32]) {
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
    asm volatile("" : "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}

// Warps 0-3 and 4-7: softmax of one row tile each, a row a thread; warps 8 and 11 copy keys and values; warps 9 and 10 issue the products of one row tile each.  As in prefix_kernel: S = Q K^T
// into 64 columns of tensor memory, P takes its place as the A operand of O += P V.  Rings and barriers run on from one pair to the next; the next pair's queries come while the results of the one before
// are written.
template <typename T, int DP>
__global__ void __launch_bounds__(384, 1) chunk_kernel(const __grid_constant__ ChunkArgs a, const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    constexpr int kBlocks = DP / 64, kStages = PrefixShape<DP>::stages;
    constexpr uint32_t kTile = PrefixShape<DP>::tile, kBlock = 128 * 128;
    static_assert(kStages >= 4, "a wait for an entry of the ring has seen the one before in its place");
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t s_full[kStages], s_empty[kStages], s_scores[2][2], s_probs[2][2], s_half[2], s_turn[2], s_done[2], s_free[2], s_q[2], s_edge;
    __shared__ int s_pages[2][4][16];
    __shared__ uint32_t s_odd[8];
    __shared__ uint32_t s_tmem;
    __shared__ volatile uint32_t s_abort;
    const uint32_t q_smem = (smem_u32(smem_raw) + 1023u) & ~1023u, ring = q_smem + 2 * kTile;
    const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

    if (warp == 9) {
        tcgen05_alloc(smem_u32(&s_tmem), 512);
        tcgen05_relinquish();
    }
    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int i = 0; i < kStages; ++i) {
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&s_empty[i]), 2);                         // groups that use a tile
        }
        for (int i = 0; i < 2; ++i) {
            for (int h = 0; h < 2; ++h) {
                mbar_init(smem_u32(&s_scores[i][h]), 1);
                mbar_init(smem_u32(&s_probs[i][h]), 4);
            }
            mbar_init(smem_u32(&s_half[i]), 1);
            mbar_init(smem_u32(&s_turn[i]), 1);
            mbar_init(smem_u32(&s_done[i]), 1);
            mbar_init(smem_u32(&s_free[i]), 4);
            mbar_init(smem_u32(&s_q[i]), 1);
        }
        mbar_init(smem_u32(&s_edge), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        mbar_arrive(smem_u32(&s_turn[0]));                               // the first group begins
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = uniform(s_tmem);
    griddep_wait();
    griddep_launch();

    const auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, &s_abort, &g_attn_flag, kFlagLmWait)); };
    struct Place {                       // in the ring: keys of a block's tile t at 2 t, its values at 2 t + 1, over all its items
        uint32_t st, parity;
        __device__ __forceinline__ void on() {
            st += 2;
            if (st >= kStages) { st -= kStages; parity ^= 1; }
        }
    };
    if (warp == 8 || warp == 11) {
        // One warp copies keys, one values.  A lane copies a box: `box_rows` tokens of a page, 64 values of each, whose page it looked up two copies ahead.
        const bool values = warp == 11;
        const int box = lane / kBlocks, blk = lane % kBlocks;
        const uint32_t words = smem_u32(&s_pages[values][0][box & 15]);
        struct Tiles {                   // the block's tiles in order
            ChunkWalk walk;
            ChunkItem x;
            int step, seen;              // seen: the first token that any row of the item sees
            bool more;
            __device__ __forceinline__ Tiles(const ChunkArgs& a) : walk(a) { item(); }
            __device__ __forceinline__ void item() {
                do more = walk.next(x);
                while (more && x.from >= x.to);
                step = x.from;
                seen = walk.a.window ? x.first + x.row0 / walk.a.group + 1 - walk.a.window : 0;
            }
            __device__ __forceinline__ void on() {
                if (++step >= x.to) item();
            }
        };
        Tiles ahead(a), now(a);
        int i = 0, i_ahead = 0;
        const auto look_up = [&]() {
            const int token = (ahead.x.tile0 + ahead.step) * 128 + box * a.box_rows;
            if (ahead.more && blk == 0 && box * a.box_rows < 128 && token < ahead.x.end && token + a.box_rows > ahead.seen)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(words + (i_ahead & 3) * 64), "l"(a.block_table + ahead.x.b * a.table_stride + token / a.page) : "memory");
            asm volatile("cp.async.commit_group;" ::: "memory");
            ++i_ahead;
            if (ahead.more) ahead.on();
        };
        look_up();
        look_up();
        Place at = {values ? 1u : 0u, 1};
        uint32_t edges = 0, item = 0;
        bool ok = true, fresh = true;
        while (ok && now.more) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            const int first = (now.x.tile0 + now.step) * 128, there = min(128, now.x.end - first), boxes = (there + a.box_rows - 1) / a.box_rows;
            ok = wait(&s_empty[at.st], at.parity);
            if (!ok) break;
            // Values of a tile whose keys not all rows see: what lies behind the last one is zeros, and so is what is not finite (zero times which would be NaN for
            // the rows that do not see it; s_odd tells the softmax groups to add it where it is seen).
            bool edge = false;
            const int pos0 = now.x.first + now.x.row0 / a.group, pos1 = now.x.end - 1;
            if (values) {
                edge = first + 128 > pos0 + 1 || (a.window && first < pos1 - a.window + 1);
                if (fresh && lane == 0) s_odd[item & 7] = 0;
                fresh = false;
            }
            if (!values && fresh && a.q_boxes) {
                // the item's queries, which the issuing warps will fetch
                const int tile = lane / kBlocks, row0 = now.x.row0 + tile * 128;
                if (tile < 2 && row0 < now.x.rows) tma_prefetch_4d(&qmap, (lane % kBlocks) * 64, 0, now.x.head, now.x.start + row0 / a.group);
                fresh = false;
            }
            const uint32_t to = ring + at.st * kTile, bar = smem_u32(edge ? &s_edge : &s_full[at.st]);
            if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(boxes * kBlocks * a.box_rows * 128));
            __syncwarp();
            if (box < boxes) {
                int page;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(page) : "r"(words + (i & 3) * 64) : "memory");
                const bool seen = first + (box + 1) * a.box_rows > now.seen;     // in front of the window the page may be gone, and was not looked up
                if (!seen || (uint32_t)page >= (uint32_t)a.n_pages) {
                    if (seen) atomicExch(&g_attn_flag, kFlagLmPage);
                    page = a.n_pages;                                    // outside of the map: zeros
                }
                tma_load_4d(to + blk * kBlock + box * a.box_rows * 128, values ? &vmap : &kmap, blk * 64, (first + box * a.box_rows) % a.page, now.x.head, page, bar);
            }
            __syncwarp();
            if (edge) {
                ok = wait(&s_edge, edges & 1);
                ++edges;
                if (!ok) break;
                constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u;
                bool odd = false;
                for (int c = there * 8 + lane; c < 1024; c += 32)
#pragma unroll
                    for (int i = 0; i < kBlocks; ++i) st_shared_v4(to + i * kBlock + c * 16, 0, 0, 0, 0);
                // rows that not all see: those behind the first row's position, or, under a window, all
                const int rows0 = a.window ? 0 : max(pos0 + 1 - first, 0);
#pragma unroll 1
                for (int c0 = rows0 * 8; c0 < there * 8; c0 += 128) {
                    uint4 v[4 * kBlocks];
                    uint32_t any = 0;
#pragma unroll
                    for (int i = 0; i < 4 * kBlocks; ++i) {
                        const int c = c0 + 32 * (i / kBlocks) + lane;
                        v[i] = c < there * 8 ? ld_shared_v4(to + (i % kBlocks) * kBlock + c * 16) : make_uint4(0, 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < 4 * kBlocks; ++i) any |= __vcmpeq2(v[i].x & kExp, kExp) | __vcmpeq2(v[i].y & kExp, kExp) | __vcmpeq2(v[i].z & kExp, kExp) | __vcmpeq2(v[i].w & kExp, kExp);
                    if (!any) continue;
                    odd = true;
#pragma unroll
                    for (int i = 0; i < 4 * kBlocks; ++i) {
                        const int c = c0 + 32 * (i / kBlocks) + lane;
                        if (c < there * 8)
                            st_shared_v4(to + (i % kBlocks) * kBlock + c * 16, v[i].x & ~__vcmpeq2(v[i].x & kExp, kExp), v[i].y & ~__vcmpeq2(v[i].y & kExp, kExp), v[i].z & ~__vcmpeq2(v[i].z & kExp, kExp),
                                         v[i].w & ~__vcmpeq2(v[i].w & kExp, kExp));
                    }
                }
                if (__any_sync(0xffffffffu, odd) && lane == 0) s_odd[item & 7] = 1;
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s_full[at.st]));
            }
            at.on();
            ++i;
            const bool last = now.step + 1 >= now.x.to;
            now.on();
            if (last) { ++item; fresh = true; }
            look_up();
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else if (warp == 9 || warp == 10) {
        constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);
        constexpr uint32_t idesc_s = (1u << 4) | kType | ((64u >> 3) << 17) | ((128u >> 4) << 24);
        // (All DP values of a head, zeros behind its own: with a bound on the loop below instead heads of 96 gained nothing, and heads of 128 lost 2 %.)
        constexpr uint32_t idesc_o = (1u << 4) | kType | (1u << 16) | (((uint32_t)DP >> 3) << 17) | ((128u >> 4) << 24);
        const int g = warp - 9;
        const uint32_t d_s = tmem + g * 128, d_o = tmem + 256 + g * DP;
        const uint64_t desc_q = umma_desc_sw128(q_smem + g * kTile), desc_k = umma_desc_sw128(ring), desc_v = umma_desc_sw128_mn(ring, kBlock);
        const uint32_t high_k = (uint32_t)(desc_k >> 32), high_v = (uint32_t)(desc_v >> 32), low_q = (uint32_t)desc_q;
        Place keys = {0, 0}, vals = {1, 0};
        uint32_t turn = 0, tiles = 0, items = 0;       // phases: of the turns, of this group's tiles and items
        ChunkWalk walk(a);
        ChunkItem x;
        bool ok = true;
        // This group's queries, neighbouring lanes on neighbouring bytes of a row: when the scores of the item before have become values, while its results are written.
        constexpr int kPerRow = DP / 8, kStep = 32 / kPerRow;                    // 16-byte pieces of a row; rows from one of a lane's pieces to the next
        const int piece = lane % kPerRow, r0 = lane / kPerRow, b_step = kStep / a.group, h_step = kStep - b_step * a.group;
        const int64_t q_step = b_step * a.q_stride + h_step * a.q_head, q_wrap = a.q_stride - a.group * a.q_head;
        const uint32_t q_block = q_smem + g * kTile + (piece >> 3) * kBlock;
        const auto load_q = [&](const ChunkItem& y) -> bool {
            if (a.q_boxes) {
                if (elect_one()) {
                    mbar_arrive_expect_tx(smem_u32(&s_q[g]), kTile);
#pragma unroll
                    for (int i = 0; i < kBlocks; ++i) tma_load_4d(q_smem + g * kTile + i * kBlock, &qmap, i * 64, 0, y.head, y.start + (y.row0 + g * 128) / a.group, smem_u32(&s_q[g]));
                }
                __syncwarp();
                return wait(&s_q[g], items & 1);
            }
            int r = y.row0 + g * 128 + r0;
            const int token = r / a.group;
            int h = r - token * a.group;
            const T* src = static_cast<const T*>(a.q) + (int64_t)(y.start + token) * a.q_stride + ((int64_t)y.head * a.group + h) * a.q_head + 8 * piece;
#pragma unroll 8
            for (int i = r0; i < 128; i += kStep) {
                const bool there = r < y.rows && 8 * piece < a.D;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(q_block + i * 128 + (((piece & 7) ^ (i & 7)) << 4)), "l"(there ? src : static_cast<const T*>(a.q)), "r"(there ? 16 : 0) : "memory");
                r += kStep;
                h += h_step;
                src += q_step;
                if (h >= a.group) { h -= a.group; src += q_wrap; }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (a.scale < 0.f) {                                                 // |scale| from here on
#pragma unroll 1
                for (int i = r0; i < 128; i += kStep) {
                    const uint32_t at = q_block + i * 128 + (((piece & 7) ^ (i & 7)) << 4);
                    const uint4 v = ld_shared_v4(at);
                    st_shared_v4(at, v.x ^ 0x80008000u, v.y ^ 0x80008000u, v.z ^ 0x80008000u, v.w ^ 0x80008000u);
                }
            }
            fence_proxy_async();
            __syncwarp();
            return true;
        };
        while (ok && walk.next(x)) {
            const int n = x.to - x.from;
            if (n <= 0) continue;
            const bool two = x.row0 + 128 < x.rows;
            if (g == 1 && !two) {                      // nothing to do here but to let the ring go on
                for (int u = 0; ok && u < n; ++u) {
                    ok = wait(&s_full[keys.st], keys.parity);
                    if (ok && lane == 0) mbar_arrive(smem_u32(&s_empty[keys.st]));
                    keys.on();
                    ok = ok && wait(&s_full[vals.st], vals.parity);
                    if (ok && lane == 0) mbar_arrive(smem_u32(&s_empty[vals.st]));
                    vals.on();
                }
                continue;
            }
            ok = load_q(x);
            // Two groups take turns at the tensor cores, as in prefix_kernel.
            const auto take_turn = [&]() {
                if (!two) return true;
                const bool now = wait(&s_turn[g], turn);
                turn ^= 1;
                return now;
            };
            const auto scores = [&](uint32_t h) {
                if (h == 0 && !wait(&s_full[keys.st], keys.parity)) return false;
                tcgen05_fence_after();
                const uint32_t low = (uint32_t)desc_k + keys.st * (kTile >> 4) + h * (8192 >> 4);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k) {
                        if (two && k == DP / 32) mbar_arrive(smem_u32(&s_turn[g ^ 1]));
                        tcgen05_mma_bf16(d_s + h * 64, pack_f32x2(low_q + (k >> 2) * (kBlock >> 4) + (k & 3) * 2, high_k), pack_f32x2(low + (k >> 2) * (kBlock >> 4) + (k & 3) * 2, high_k), idesc_s, k > 0);
                    }
                    tcgen05_commit(smem_u32(&s_scores[g][h]));
                    if (h == 1) tcgen05_commit(smem_u32(&s_empty[keys.st]));
                }
                __syncwarp();
                if (h == 1) keys.on();
                return true;
            };
            ok = ok && take_turn() && scores(0) && take_turn() && scores(1);
            for (int u = 0; ok && u < n; ++u, ++tiles) {
                const bool last = u == n - 1;
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    if (h == 0) {
                        ok = wait(&s_full[vals.st], vals.parity);
                        if (ok && u == 0 && items > 0) ok = wait(&s_free[g], (items - 1) & 1);          // the sums of the item before have been read
                        if (!ok) break;
                    }
                    ok = wait(&s_probs[g][h], tiles & 1) && take_turn();
                    if (!ok) break;
                    tcgen05_fence_after();
                    const uint32_t low = (uint32_t)desc_v + vals.st * (kTile >> 4) + h * (8192 >> 4), more = u > 0;
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            tcgen05_mma_f16_ts(d_o, d_s + h * 64 + k * 8, pack_f32x2(low + k * (2048 >> 4), high_v), idesc_o, more | (uint32_t)(h > 0 || k > 0));
                        if (h == 1) tcgen05_commit(smem_u32(&s_empty[vals.st]));
                        if (last) tcgen05_commit(smem_u32(h == 0 ? &s_half[g] : &s_done[g]));
                    }
                    __syncwarp();
                    if (!last) ok = scores(h);
                    else if (two && elect_one()) mbar_arrive(smem_u32(&s_turn[g ^ 1]));
                    __syncwarp();
                    if (!ok) break;
                }
                vals.on();
            }
            ++items;
        }
    } else {
        const int g = warp >> 2, in_tile = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;                       // this warp's lanes of tensor memory
        const float c = fmaxf(fabsf(a.scale) * kLog2e, 1e-38f);                  // (a scale of 0 must not meet the infinities of masked keys)
        const auto place = [&](const ChunkItem& x, int row, int64_t token_stride, int64_t head_stride) {       // of q or out
            const int token = row / a.group;
            return (int64_t)(x.start + token) * token_stride + (int64_t)(x.head * a.group + row - token * a.group) * head_stride;
        };
        const bool out_vec = (((uintptr_t)a.out | (uintptr_t)(a.out_stride * 2) | (uintptr_t)(a.out_head * 2)) & 15) == 0;
        // 32 values of each lane's row, from column `col` on.  Four lanes exchange their 16-byte pieces first, so that they write 64 bytes of one row at a time (each 16 of its own row: 7000
        // clocks for two row tiles instead of 2000).  The whole warp.
        const auto write = [&](const ChunkItem& x, T* base, int row, int col, const uint32_t (&o)[32], float f) {
            uint4 v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[e] = make_uint4(lm_pack2<T>(__uint_as_float(o[8 * e]) * f, __uint_as_float(o[8 * e + 1]) * f), lm_pack2<T>(__uint_as_float(o[8 * e + 2]) * f, __uint_as_float(o[8 * e + 3]) * f),
                                  lm_pack2<T>(__uint_as_float(o[8 * e + 4]) * f, __uint_as_float(o[8 * e + 5]) * f), lm_pack2<T>(__uint_as_float(o[8 * e + 6]) * f, __uint_as_float(o[8 * e + 7]) * f));
            if (!out_vec) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (col + 8 * e >= a.D || row >= x.rows) break;
                    const T* y = reinterpret_cast<const T*>(&v[e]);
#pragma unroll
                    for (int k = 0; k < 8; ++k) base[col + 8 * e + k] = y[k];
                }
                return;
            }
            const auto swap = [&](uint4& lo, uint4& hi, int with) {              // my `hi` for the other lane's `lo`, or the other way round
                const bool up = lane & with;
                uint4 give = up ? lo : hi;
                give.x = __shfl_xor_sync(0xffffffffu, give.x, with);
                give.y = __shfl_xor_sync(0xffffffffu, give.y, with);
                give.z = __shfl_xor_sync(0xffffffffu, give.z, with);
                give.w = __shfl_xor_sync(0xffffffffu, give.w, with);
                (up ? lo : hi) = give;
            };
            swap(v[0], v[1], 1);
            swap(v[2], v[3], 1);
            swap(v[0], v[2], 2);
            swap(v[1], v[3], 2);
            // v[k]: piece lane % 4 of the row of the quad's lane k
            const int first = row - (lane & 3), piece = col + 8 * (lane & 3);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                T* to = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, (unsigned long long)base, (lane & ~3) + k));
                if (piece < a.D && first + k < x.rows) *reinterpret_cast<uint4*>(to + piece) = v[k];
            }
        };
        // Values of V that are not finite, whose tiles held zeros in their places, into the sums of the rows that see them.
        const auto add_odd = [&](const ChunkItem& x, uint32_t from, int limit, int low) {
#pragma unroll 1
            for (int j = 0; j < a.D; j += 8) {
                uint32_t o[8];
                __syncwarp();
                tcgen05_ld8(from + j, o);
                tcgen05_wait_ld();
#pragma unroll 1
                for (int s = x.from; s < x.to; ++s) {
                    const int key = (x.tile0 + s) * 128, pos0 = x.first + x.row0 / a.group;
                    if (key + 128 <= pos0 + 1 && !(a.window && key < x.end - a.window)) continue;
#pragma unroll 1
                    for (int at = max(key, low); at < min(key + 128, limit); ++at) {
                        const int page = __ldcg(a.block_table + x.b * a.table_stride + at / a.page);
                        if ((uint32_t)page >= (uint32_t)a.n_pages) continue;
                        const uint4 w = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.v) + page * a.page_stride + (at % a.page) * a.token_stride + x.head * a.head_stride + j));
                        const T* y = reinterpret_cast<const T*>(&w);
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float z = lm_to_f<T>(y[k]);
                            if (!(fabsf(z) < INFINITY)) o[k] = __float_as_uint(__uint_as_float(o[k]) + z);
                        }
                    }
                }
                __syncwarp();
                tcgen05_st8(from + j, o);
                tcgen05_wait_st();
            }
        };
        ChunkWalk walk(a);
        ChunkItem x;
        uint32_t items = 0, all_items = 0, tiles = 0;                            // this group's, all of those with tiles, this group's tiles
        bool ok = true;
        while (ok && walk.next(x)) {
            const int row = x.row0 + g * 128 + in_tile, n = x.to - x.from;
            const bool live_warp = row - lane < x.rows;
            if (n <= 0) {                              // rows that see nothing
                if (live_warp && x.tiles == 0) {
                    const uint32_t zeros[32] = {};
                    T* const base = static_cast<T*>(a.out) + place(x, min(row, x.rows - 1), a.out_stride, a.out_head);
#pragma unroll 1
                    for (int j = 0; j < a.D; j += 32) write(x, base, row, j, zeros, 0.f);
                }
                continue;
            }
            const uint32_t item = all_items++;
            if (g == 1 && x.row0 + 128 >= x.rows) continue;
            const int limit = x.first + min(row, x.rows - 1) / a.group + 1, low = a.window ? limit - a.window : 0;     // the row sees tokens low to limit - 1
            float m = -INFINITY, l = 0.f;
            for (int i = 0; i < 2 * n; ++i) {
                const int h = i & 1;
                ok = wait(&s_scores[g][h], (tiles + (uint32_t)(i >> 1)) & 1);
                if (!ok) break;
                if (live_warp) {
                    tcgen05_fence_after();
                    const uint32_t ts = tmem + lanes + g * 128 + h * 64;
                    const int key = (x.tile0 + x.from + (i >> 1)) * 128 + h * 64, hi = limit - key, lo = low - key;
                    const bool edge = __any_sync(0xffffffffu, hi < 64 || lo > 0);
                    uint32_t p[32];
                    float sum;
                    // The exponentials are of the maximum so far, so that they need not wait for this half's; where that is too low they are done again.
                    while (true) {
                        uint32_t s[2][32];             // the second scores come while the first ones are worked on
                        float top[2] = {-INFINITY, -INFINITY};
                        const float base = m == -INFINITY ? 0.f : p_shift<T>() - m * c;
                        tcgen05_ld32(ts, s[0]);
                        sum = 0.f;
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            tcgen05_wait_ld();
                            pin(s[k]);
                            if (k == 0) tcgen05_ld32(ts + 32, s[1]);
                            if (edge) {
#pragma unroll
                                for (int j = 0; j < 32; ++j)
                                    if (32 * k + j >= hi || 32 * k + j < lo) s[k][j] = 0xff800000u;
                            }
#pragma unroll
                            for (int j = 0; j < 32; j += 2) top[(j >> 1) & 1] = max3(top[(j >> 1) & 1], __uint_as_float(s[k][j]), __uint_as_float(s[k][j + 1]));
                            sum += values_of<T>(s[k], c, base, *reinterpret_cast<uint32_t (*)[16]>(p + 16 * k));
                        }
                        const float next = fmaxf(m, fmaxf(top[0], top[1]));
                        if (!__any_sync(0xffffffffu, (next - m) * c > kSlack)) break;          // (a NaN difference, -inf to -inf, is no growth)
                        if (i > 0) {
                            // The products of the half before may still be adding to O: the scores behind them tell of their end, or, for the last half, a barrier.
                            ok = i + 1 < 2 * n ? wait(&s_scores[g][h ^ 1], (tiles + (uint32_t)((i + 1) >> 1)) & 1) : wait(&s_half[g], items & 1);
                            if (!ok) break;
                            tcgen05_fence_after();
                            const float keep = next == m ? 1.f : ex2((m - next) * c);
                            const uint32_t to = tmem + lanes + 256 + g * DP;
#pragma unroll 1
                            for (int j = 0; j < DP; j += 32) {
                                uint32_t o[32];
                                tcgen05_ld32(to + j, o);
                                tcgen05_wait_ld();
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                                tcgen05_st32(to + j, o);
                            }
                            l *= keep;
                        }
                        m = next;
                    }
                    if (!ok) break;
                    l += sum;
                    tcgen05_st32(ts, p);
                    tcgen05_wait_st();
                    tcgen05_fence_before();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&s_probs[g][h]));
            }
            if (!ok) break;
            ok = wait(&s_done[g], items & 1);
            if (!ok) break;
            tiles += (uint32_t)n;
            ++items;
            if (live_warp) {
                tcgen05_fence_after();
                const uint32_t from = tmem + lanes + 256 + g * DP;
                if (*(volatile uint32_t*)&s_odd[item & 7] != 0) add_odd(x, from, limit, low);
                const int64_t part = (int64_t)x.slot * 2 + g;
                const float inv = limit <= 0 ? 0.f : 1.f / l;                    // (0: a row that sees no token)
                T* const base = static_cast<T*>(a.out) + place(x, min(row, x.rows - 1), a.out_stride, a.out_head);
                if (x.slot >= 0) a.part_ml[part * 128 + in_tile] = make_float2(m == -INFINITY ? m : m * c, l);
                // (Rolled up: code that runs once for an item comes from memory.)
#pragma unroll 1
                for (int k = 0; k < DP / 32; ++k) {
                    uint32_t v[32];
                    __syncwarp();
                    tcgen05_ld32(from + 32 * k, v);
                    tcgen05_wait_ld();
                    pin(v);
                    if (x.slot >= 0) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            a.part_o[(part * (DP / 4) + 8 * k + e) * 128 + in_tile] = make_float4(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1]), __uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3]));
                    } else {
                        write(x, base, row, 32 * k, v, inv);
                    }
                }
                __syncwarp();
                tcgen05_fence_before();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&s_free[g]));
        }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (s_abort) {             // copies in flight end before their shared memory does
        const unsigned long long t0 = globaltimer_ns();
        for (int i = 0; i < 100000 && globaltimer_ns() - t0 < 50000; ++i) __nanosleep(500);
    }
    if (warp == 9) {
        tcgen05_fence_after();
        tcgen05_dealloc(tmem, 512);
    }
}

// The parts of pairs that were cut: sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i.  kJoinSlices blocks for each cut, which a pair's first cut works for; a row a lane, a piece of its values a warp.
template <typename T, int DP>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ ChunkArgs a, uint32_t job_id, FinishedBlockNotifier* nf) {
    griddep_wait();
    if (nf) nf->start(job_id);
    griddep_launch();
    static_assert(256 / kJoinSlices == 32, "a row a lane");
    constexpr int kEach = DP / 4 / 8;                  // 16-byte pieces of a thread
    const int slice = (int)blockIdx.x % kJoinSlices, ranges = __ldcg(a.counts + 1);
    for (int r = (int)blockIdx.x / kJoinSlices + 1; r < max(ranges, 2); r += kChunkBlocks) {
        const int4 c = __ldcg(reinterpret_cast<const int4*>(a.cuts + r)), d = __ldcg(reinterpret_cast<const int4*>(a.cuts + r - 1));   // (used if there are so many)
        const auto same = [&](const int4& x) { return x.x == c.x && x.y == c.y; };
        if (r >= ranges || c.z == 0 || (same(d) && d.z > 0)) continue;
        const ChunkUnit u = a.cuts[r].begins;
        int last = r;                                  // the pair's last range: a warp looks at 32 cuts at a time
        while (true) {
            const int at = last + 1 + (int)(threadIdx.x & 31);
            bool on = at < ranges;
            if (on) {
                const int4 e = __ldcg(reinterpret_cast<const int4*>(a.cuts + at));
                on = same(e) && e.z > 0;
            }
            const uint32_t run = __ballot_sync(0xffffffffu, on);
            last += run == 0xffffffffu ? 32 : __ffs(~run) - 1;
            if (run != 0xffffffffu) break;
        }
        const int parts = last - r + 2, in_pair = slice * 32 + (int)(threadIdx.x & 31), warp = (int)threadIdx.x >> 5, row = u.row0 + in_pair, g = in_pair >> 7, in_tile = in_pair & 127;
        const auto slot = [&](int i) { return (int64_t)(i == 0 ? 2 * (r - 1) + 1 : 2 * (r + i - 1)) * 2 + g; };
        if (row < u.rows) {
            float top = -INFINITY, sum = 0.f;
#pragma unroll 8
            for (int i = 0; i < parts; ++i) top = fmaxf(top, __ldcg(a.part_ml + slot(i) * 128 + in_tile).x);
            float4 acc[kEach] = {};
#pragma unroll 4
            for (int i = 0; i < parts; ++i) {
                const float2 ml = __ldcg(a.part_ml + slot(i) * 128 + in_tile);
                float4 o[kEach];
#pragma unroll
                for (int k = 0; k < kEach; ++k) o[k] = __ldcg(a.part_o + (slot(i) * (DP / 4) + warp * kEach + k) * 128 + in_tile);
                const float w = ml.x == -INFINITY ? 0.f : ex2(ml.x - top);
                sum = fmaf(w, ml.y, sum);
#pragma unroll
                for (int k = 0; k < kEach; ++k) {
                    acc[k].x = fmaf(w, o[k].x, acc[k].x); acc[k].y = fmaf(w, o[k].y, acc[k].y); acc[k].z = fmaf(w, o[k].z, acc[k].z); acc[k].w = fmaf(w, o[k].w, acc[k].w);
                }
            }
            const int token = row / a.group;
            const float inv = u.first + token < 0 ? 0.f : 1.f / sum;             // (as in chunk_kernel)
            T* dst = static_cast<T*>(a.out) + (int64_t)(u.start + token) * a.out_stride + (int64_t)(c.y * a.group + row - token * a.group) * a.out_head;
            const bool vec = (((uintptr_t)a.out | (uintptr_t)(a.out_stride * 2) | (uintptr_t)(a.out_head * 2)) & 7) == 0;
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                const int col = 4 * (warp * kEach + k);
                if (col >= a.D) break;
                const float x = acc[k].x * inv, y = acc[k].y * inv, z = acc[k].z * inv, w = acc[k].w * inv;
                if (vec) {
                    *reinterpret_cast<uint2*>(dst + col) = make_uint2(lm_pack2<T>(x, y), lm_pack2<T>(z, w));
                } else {
                    dst[col] = lm_from_f<T>(x); dst[col + 1] = lm_from_f<T>(y); dst[col + 2] = lm_from_f<T>(z); dst[col + 3] = lm_from_f<T>(w);
                }
            }
        }
    }
    if (nf) nf->end(job_id);
}

typedef void (*JoinFn)(ChunkArgs, uint32_t, FinishedBlockNotifier*);
typedef void (*ChunkFn)(ChunkArgs, CUtensorMap, CUtensorMap, CUtensorMap);

struct ChunkPlan {
    ChunkArgs a;
    AttnArgs few;              // own_kernel's, where it takes part
    int DP, NT;
    bool half, many, has_few;  // many: plan, chunk and join kernels
    int64_t few_blocks, join_blocks;
    uint64_t scratch;
    OwnFn own;
    uint32_t own_smem;
    ChunkFn chunk;
    JoinFn join;
};

template <typename T> void pick_chunk(ChunkPlan& pl) {
    pl.own = own_fn<T, 3>(pl.DP, pl.NT);
    pl.chunk = pl.DP == 64 ? chunk_kernel<T, 64> : chunk_kernel<T, 128>;
    pl.join = pl.DP == 64 ? join_kernel<T, 64> : join_kernel<T, 128>;
}

int plan_chunk(const pb_chunk_attn_params* p, ChunkPlan& pl) {
    const char* who = "pb_chunk_attn";
    PB_REQUIRE(p != nullptr, "%s: NULL params", who);
    PB_REQUIRE(p->dtype == PB_BF16 || p->dtype == PB_F16, "%s: dtype %d (PB_BF16 or PB_F16)", who, p->dtype);
    PB_REQUIRE(p->batch >= 0 && p->batch <= 1 << 24 && p->tokens >= 0 && p->q_heads >= 1 && p->kv_heads >= 1 && p->q_heads % p->kv_heads == 0 && p->q_heads <= 65536, "%s: batch %d, %d tokens, %d query heads, %d key heads", who,
               p->batch, p->tokens, p->q_heads, p->kv_heads);
    PB_REQUIRE(p->head_dim >= 8 && p->head_dim <= 128 && p->head_dim % 8 == 0, "%s: head_dim %d (a multiple of 8, 8 to 128)", who, p->head_dim);
    PB_REQUIRE(p->page_size >= 8 && p->page_size % 8 == 0 && p->page_size <= 1 << 24, "%s: page_size %d (a multiple of 8, at most 2^24)", who, p->page_size);
    PB_REQUIRE(p->n_pages >= 0 && p->n_pages <= 0x7fffffff, "%s: %lld pages", who, (long long)p->n_pages);
    PB_REQUIRE(p->max_new >= 0 && p->max_len >= 0 && p->max_len <= 1 << 30 && p->window >= 0, "%s: at most %d new tokens of %d, window %d", who, p->max_new, p->max_len, p->window);
    PB_REQUIRE(p->max_blocks >= 0 && p->max_len <= (int64_t)p->max_blocks * p->page_size, "%s: %d tokens do not fit %d pages of %d", who, p->max_len, p->max_blocks, p->page_size);
    PB_REQUIRE(fabsf(p->scale) <= 2e38f, "%s: scale is not finite, or above 2e38", who);        // (which in powers of two is finite, too)
    PB_REQUIRE(p->page_stride % 8 == 0 && p->token_stride % 8 == 0 && p->head_stride % 8 == 0 && p->page_stride > 0 && p->token_stride > 0 && p->head_stride > 0, "%s: strides of the cache are positive multiples of 8", who);
    PB_REQUIRE(p->q_stride % 8 == 0 && p->q_head_stride % 8 == 0, "%s: rows of q start on 16 bytes", who);
    PB_REQUIRE(rows_apart(p->tokens, p->out_stride, p->head_dim) && rows_apart(p->q_heads, p->out_head_stride, p->head_dim), "%s: rows of out overlap (strides %lld, %lld)", who, (long long)p->out_stride, (long long)p->out_head_stride);
    memset(&pl, 0, sizeof(pl));
    ChunkArgs& a = pl.a;
    a.max_new = std::min(p->max_new, p->tokens);
    a.batch = a.max_new > 0 ? p->batch : 0;
    a.group = p->q_heads / p->kv_heads;
    PB_REQUIRE((int64_t)a.max_new * a.group <= 1 << 30, "%s: %d new tokens of %d heads for a key head are too many rows", who, a.max_new, a.group);
    if (a.batch > 0) {
        PB_REQUIRE(p->q && p->out && p->starts && p->lens, "%s: NULL buffer", who);
        PB_REQUIRE(p->max_len == 0 || (p->k_cache && p->v_cache && p->block_table && p->n_pages > 0), "%s: a NULL cache or block_table, or a cache without pages", who);
        PB_REQUIRE(aligned(p->q, 16) && aligned(p->k_cache, 16) && aligned(p->v_cache, 16) && aligned(p->out, 2), "%s: q and the cache must be 16-byte aligned", who);
        PB_REQUIRE(aligned(p->block_table, 4) && aligned(p->starts, 4) && aligned(p->lens, 4), "%s: a table is not aligned to its elements", who);
    }
    a.q = p->q; a.k = p->k_cache; a.v = p->v_cache; a.out = p->out; a.block_table = p->block_table; a.starts = p->starts; a.lens = p->lens;
    a.q_stride = p->q_stride; a.q_head = p->q_head_stride; a.out_stride = p->out_stride; a.out_head = p->out_head_stride;
    a.page_stride = p->page_stride; a.token_stride = p->token_stride; a.head_stride = p->head_stride; a.table_stride = p->table_stride;
    a.tokens = p->tokens; a.q_heads = p->q_heads; a.kv_heads = p->kv_heads; a.D = p->head_dim;
    a.page = p->page_size; a.n_pages = (int)p->n_pages; a.max_len = p->max_len; a.window = p->window < p->max_len ? p->window : 0; a.scale = p->scale;
    a.q_boxes = 128 % a.group == 0 && a.scale >= 0.f && a.q_stride > 0 && a.q_head > 0 && a.q_stride < 1 << 30 && a.q_head < 1 << 30 && (int64_t)a.group * a.q_head < 1 << 30;
    a.box_rows = 8;
    while (a.box_rows < 64 && p->page_size % (2 * a.box_rows) == 0) a.box_rows *= 2;
    pl.DP = p->head_dim <= 64 ? 64 : 128;
    pl.half = p->dtype == PB_F16;
    const int64_t most_rows = (int64_t)a.max_new * a.group, tokens = a.window ? std::min<int64_t>(a.window + a.max_new, a.max_len) : a.max_len;
    // own_kernel: as for pb_prefix_attn, clusters of blocks on a sequence and key head while they fit the GPU, 128 tokens each at least.  (24 sequences of 4 tokens x 4 heads, 8 key heads, up to 4096 tokens: twice as many
    // blocks 64 us instead of 55; 32 of one token behind up to 2000 30 instead of 33.)
    const auto ranks_of = [&](int64_t units) {
        int ranks = 1;
        while (ranks < kMaxRanks && units > 0 && units * ranks * 2 <= 3 * 148 && tokens / (2 * ranks) >= 128) ranks *= 2;
        return ranks;
    };
    pl.many = a.max_new > 1 && most_rows > kFewRows;
    if (!pl.many && a.batch > 0) {
        // Few rows of long sequences that are too few for own_kernel's blocks, as if all were as long as max_len says: the times that plan_kernel compares, and 30 us for plan, beginning, parts and join.  (One new
        // token behind 30000, 8 key heads of 128: 49 us with own_kernel, 48 here; behind 60000 91 and 67, behind 130000 188 and 111.  The host knows no lengths: behind 500 tokens a lone sequence takes 9.0 us where max_len
        // is 501 and 19.4 where it is 32768 or more, 64 sequences 34.8 and, from 131072 on, 44.0.)
        const int64_t groups = ceil_div<int64_t>(most_rows, most_rows <= 8 ? 8 : 16);
        const double each = 4.0 * a.D * tokens, units = (double)a.batch * a.kv_heads;
        const double there = std::max(each * units / 6000.0, each / (40.0 * ranks_of(a.batch * a.kv_heads * groups))) + 5000.0, here = units * (tokens * 1600.0 / 128 + 5000.0) / kChunkBlocks + 30000.0;
        pl.many = here < there;
    }
    pl.many = pl.many && a.batch > 0 && a.max_len > 0;
    pl.has_few = !pl.many || a.batch > 1;
    if (pl.has_few) {
        // beside chunks: 8 rows where a token's fit (three blocks an SM), 16 otherwise (two)
        const int limit = a.group <= kFewRows / 2 ? kFewRows / 2 : kFewRows, few_rows = (int)(pl.many ? std::min<int64_t>(most_rows, limit) : std::max<int64_t>(most_rows, 1));
        pl.NT = few_rows <= 8 ? 1 : 2;
        AttnArgs& f = pl.few;
        f.q = a.q; f.k = a.k; f.v = a.v; f.out = a.out; f.block_table = a.block_table; f.own_lens = a.lens; f.starts = a.starts;
        f.q_stride = a.q_stride; f.q_head = a.q_head; f.out_stride = a.out_stride; f.out_head = a.out_head;
        f.page_stride = a.page_stride; f.token_stride = a.token_stride; f.head_stride = a.head_stride; f.table_stride = a.table_stride;
        f.batch = a.batch; f.group = a.group; f.D = a.D; f.page = a.page; f.n_pages = a.n_pages; f.max_own = a.max_len; f.scale = a.scale; f.kv_heads = a.kv_heads;
        f.given = !pl.many && a.batch <= kGivenStarts;
        f.tokens = a.tokens; f.max_new = a.max_new; f.window = a.window; f.beside = pl.many;
        f.per_piece = (uint32_t)ceil_div(1 << 16, a.D / 4);
        f.out_vec = aligned(a.out, 8) && a.out_stride % 4 == 0 && a.out_head % 4 == 0;
        f.splits = f.row_parts = 1;
        f.row_groups = (int)ceil_div<int64_t>(few_rows, 8 * pl.NT);
        const int64_t units = (int64_t)a.batch * a.kv_heads * f.row_groups;
        f.ranks = ranks_of(units);
        pl.few_blocks = std::max<int64_t>(units * f.ranks, 1);
        PB_REQUIRE(pl.few_blocks <= 0x7fffffff, "%s: too many blocks for one launch", who);
    }
    pl.own_smem = pl.DP == 64 ? OwnShape<64>::smem : OwnShape<128>::smem;
    if (pl.half) pick_chunk<__half>(pl);
    else pick_chunk<__nv_bfloat16>(pl);
    uint64_t at = 0;
    const auto take = [&](uint64_t bytes) {
        const uint64_t from = at;
        at += round_up<uint64_t>(bytes, 128);
        return (char*)p->scratch + from;
    };
    if (pl.many || !pl.few.given) {
        a.counted = (int32_t*)take((a.batch + 1ull) * sizeof(int32_t));
        pl.few.starts = a.counted;
    }
    if (pl.many) {
        a.few = !pl.has_few ? 0 : a.group <= kFewRows / 2 ? kFewRows / 2 : kFewRows;
        a.few_ranks = pl.few.ranks;
        const int64_t units = std::min((int64_t)a.tokens * a.group / 256 + a.batch, a.batch * ceil_div<int64_t>(most_rows, 256));
        PB_REQUIRE(units * a.kv_heads <= 1 << 30, "%s: %lld pairs of row tiles are too many", who, (long long)units);
        a.max_units = (int)units;
        const int64_t cache = (int64_t)a.batch * a.max_len * a.kv_heads * a.D * 4;
        const int rounds = (int)std::min<int64_t>(std::max<int64_t>(cache >> 26, 1), kMaxRounds);
        a.max_ranges = kChunkBlocks * rounds;
        a.counts = (int32_t*)take(12);
        pl.few.few_from = a.counts + 2;
        a.cuts = (ChunkCut*)take((a.max_ranges + 2) * sizeof(ChunkCut));
        a.units = (ChunkUnit*)take(a.max_units * sizeof(ChunkUnit));
        a.before = (int64_t*)take((a.max_units + 1) * sizeof(int64_t));
        a.part_ml = (float2*)take(2ull * a.max_ranges * 256 * sizeof(float2));
        a.part_o = (float4*)take(2ull * a.max_ranges * 256 * pl.DP * sizeof(float));
        pl.join_blocks = kChunkBlocks * kJoinSlices;
    }
    pl.scratch = at;
    return PB_OK;
}

}  // namespace
}  // namespace pb
