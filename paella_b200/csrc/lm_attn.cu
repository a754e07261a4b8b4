// Attention of one new token for every sequence of a batch that shares a prefix, over a paged cache.
//
//   out[b][h] = sum_j softmax_j(scale * q[b][h] . k_j) v_j   over the prefix's tokens and the sequence's own
//
// The prefix is one matrix for the whole batch: the rows of all sequences' query heads that share a key head meet it in tiles of 128 rows x
// 128 keys on the tensor cores (prefix_kernel), and its keys and values are read once for 256 rows.  A sequence's own tokens meet only its `group`
// query rows: that is bound by reading them, a block for each sequence and key head (own_kernel), which also joins the parts of the prefix with
// its own.  Softmax runs along with the sums, in fp32: each part has its rows' maximum m, sum l and unscaled O, and parts join as
// sum 2^(m_i - m) O_i / sum 2^(m_i - m) l_i.  The softmax's values are rounded to the cache's type, as the tensor cores take them (in two parts each they would be half as
// many products again); the sums l are of what they were before.  With that rounding the results' mean error against 64 bits is 0.0022 of their size in bf16 and 0.00029 in fp16, where the results'
// own rounding alone makes 0.0017 and 0.0002.
//
// What bounds it (figures here and below are of launches back to back in a graph; one call at a time, with cold caches, the two cases take 117 and 238 us): few rows, the cache's bytes (16 sequences of 8 heads a key head behind 130001 tokens, 556 MB: 99 to 102 us, 5.5 TB/s); many, the tensor cores
// and the exponentials together (2048 rows a key head behind 16384 tokens: the tensor pipe is busy 71 % of the time on the SMs that take part, 139 us cool and up to 160 where power holds the clocks down).  256
// sequences of 8 heads a key head behind 16384 tokens with up to 1024 of their own: 200 to 224 us.
#include <cuda.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "lm.cuh"
#include "umma.cuh"

namespace pb {
namespace {

__device__ uint32_t g_attn_flag;

struct AttnArgs {
    const void *q, *k, *v;
    void* out;
    const int32_t *prefix_pages, *block_table, *own_lens;
    int64_t q_stride, q_head, out_stride, out_head, page_stride, token_stride, head_stride, table_stride;
    int batch, group, D, page, n_pages, prefix_len, max_own;
    float scale;
    // the prefix's split
    int row_tiles, pairs, splits, key_tiles, box_rows;
    int row_parts;             // splits, and one more where own tokens leave a part as well
    float* part_o;             // [row_tiles][kv_heads][row_parts][128][DP], a row's 16-byte piece i at i ^ (row % 32)
    float2* part_ml;           // the same without DP: (m, l)
    // own tokens
    int kv_heads, row_groups, ranks, early, out_vec;     // early: behind a prefix_kernel, beside whose end it starts
    uint32_t per_piece;        // 2^16 / (D / 4), rounded up
    int ahead;                 // tokens of the prefix that own_kernel takes as if they were each sequence's own: all of them, or none
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^x of a pair on the multipliers, beside ex2 on the special-function unit, which alone would take as long as the products: x = i + f with |f| <= 1/2
// (the sum with 1.5 x 2^23 rounds to a whole number), 2^f as the polynomial of degree 5 with the least largest relative error (Remez's exchange;
// 2^-22.6 with the coefficients in fp32, 2^-22.1 with fp32's roundings), i added to its exponent.  Up to 2^-126: nothing.  For x < 127; a NaN stays one: the
// exponent's sum makes a finite number of it, so x comes into the last sum once more.
__device__ __forceinline__ uint64_t ex2_pair(uint64_t x) {
    const auto both = [](float v) { return pack_f32x2(__float_as_uint(v), __float_as_uint(v)); };
    float lo, hi;
    unpack_f32x2(x, lo, hi);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(lo) : "f"(-126.f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(-126.f));
    x = pack_f32x2(__float_as_uint(lo), __float_as_uint(hi));
    const uint64_t t = add_f32x2(x, both(12582912.f)), f = fma_f32x2(add_f32x2(t, both(-12582912.f)), both(-1.f), x);
    uint64_t r = fma_f32x2(both(0.0013276472454890609f), f, both(0.009675540961325169f));
    r = fma_f32x2(r, f, both(0.05550713092088699f));
    r = fma_f32x2(r, f, both(0.24022120237350464f));
    r = fma_f32x2(r, f, both(0.6931469440460205f));
    r = fma_f32x2(r, f, both(1.0000001192092896f));
    r = pack_f32x2((uint32_t)r + ((uint32_t)t << 23), (uint32_t)(r >> 32) + ((uint32_t)(t >> 32) << 23));
    return add_f32x2(r, fma_f32x2(x, both(0.f), both(-0x1.000002p-126f)));
}

__device__ __forceinline__ float max3(float x, float y, float z) {        // (NaNs lose, as in fmaxf)
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}

constexpr float kLog2e = 1.4426950408889634f;
// A row's maximum is followed only once it has grown by 2^8: until then the values are up to 2^8 times too large, which fp32 sums and the
// 16-bit values' exponents hold, and the accumulator need not be rescaled.
constexpr float kSlack = 8.f;
// fp16 has few exponents below 1: its values are scaled up by 2^5 (2^13 with the slack; the sums with them).
template <typename T> __device__ __forceinline__ constexpr float p_shift() { return sizeof(T) == 2 && std::is_same<T, __half>::value ? 5.f : 0.f; }

// 64 keys: 2^(s c + base) from their scores, rounded to pairs, and the sum of what they were.  One pair in four on the multipliers (none, one in eight, three, two:
// 156, 168, 144, 158 us against 139 behind 16384 tokens).
template <typename T>
__device__ __forceinline__ float values_of(const uint32_t* s, float c, float base, uint32_t (&p)[32]) {
    const uint64_t c2 = pack_f32x2(__float_as_uint(c), __float_as_uint(c)), base2 = pack_f32x2(__float_as_uint(base), __float_as_uint(base));
    uint64_t sum[2] = {0, 0};
    float x, y;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        uint64_t e = fma_f32x2(pack_f32x2(s[2 * j], s[2 * j + 1]), c2, base2);
        if (j % 4 == 3) {
            e = ex2_pair(e);
            unpack_f32x2(e, x, y);
        } else {
            unpack_f32x2(e, x, y);
            x = ex2(x);
            y = ex2(y);
            e = pack_f32x2(__float_as_uint(x), __float_as_uint(y));
        }
        sum[j & 1] = add_f32x2(sum[j & 1], e);
        p[j] = lm_pack2<T>(x, y);
    }
    unpack_f32x2(add_f32x2(sum[0], sum[1]), x, y);
    return x + y;
}

// ---- the prefix ----------------------------------------------------------------------------------------------
// A block takes a range of the prefix's keys for one key head and a pair of row tiles, or, where the last row tile is alone, that tile with its
// even and odd key tiles as a pair.  Warps 0-3 and 4-7: softmax of one of the pair each, a row a thread; warps 8 and 11 copy keys and values, warps 9 and 10
// issue the products of one of the pair each, 64 keys at a time: S = Q K^T into 64 columns of tensor memory, where P of 16-bit pairs takes its place as the A operand
// of O += P V, while softmax is at the other 64.  Tensor memory: S0 S1 O0 O1, all of it at 128 values a head.
// (Scores of 128 keys at once, which cost the tensor cores 512 clocks instead of 778, leave no second place for them: a tile of the pair took 4100 clocks
// from one softmax to the next instead of 3300.  A lone issuing warp for both: 4800, its waits of 100 to 200 clocks each in a row.)
template <int DP> struct PrefixShape {
    static constexpr uint32_t tile = 128 * DP * 2;                   // bytes of 128 rows
    static constexpr int stages = DP == 128 ? 5 : 10;                // tiles of keys or values in flight (three: 215 instead of 205 us)
    static constexpr uint32_t smem = 1024 + (2 + stages) * tile;     // two tiles of queries in front of them
};

template <typename T, int DP>
__global__ void __launch_bounds__(384, 1) prefix_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    constexpr int kBlocks = DP / 64, kStages = PrefixShape<DP>::stages + 1;
    constexpr uint32_t kTile = PrefixShape<DP>::tile, kBlock = 128 * 128, kHalfTile = kTile / 2;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t s_full[2 * kStages], s_empty[2 * kStages], s_scores[2][2], s_probs[2][2], s_half[2], s_turn[2], s_done[2], s_q;
    __shared__ int s_pages[2][4][32];
    __shared__ uint32_t s_tmem;
    __shared__ volatile uint32_t s_abort;
    const uint32_t q_smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

    const int pair = blockIdx.x % a.pairs, split = (blockIdx.x / a.pairs) % a.splits, kvh = blockIdx.x / (a.pairs * a.splits);
    const int kt0 = (int)((int64_t)a.key_tiles * split / a.splits), n = (int)((int64_t)a.key_tiles * (split + 1) / a.splits) - kt0;
    const bool two = 2 * pair + 1 < a.row_tiles;      // two row tiles; otherwise one, its key tiles dealt to both softmax groups
    const uint32_t ring = q_smem + (two ? 2 : 1) * kTile;                // (a lone tile leaves its partner's place to the rings)
    const int tail = min(128, a.prefix_len - (kt0 + n - 1) * 128);       // keys of the last tile

    if (warp == 9) {
        tcgen05_alloc(smem_u32(&s_tmem), 512);
        tcgen05_relinquish();
    }
    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int i = 0; i < 2 * kStages; ++i) {
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&s_empty[i]), two ? 2 : 1);       // groups that use a tile
        }
        for (int i = 0; i < 2; ++i) {
            for (int h = 0; h < 2; ++h) {
                mbar_init(smem_u32(&s_scores[i][h]), 1);
                mbar_init(smem_u32(&s_probs[i][h]), 4);
            }
            mbar_init(smem_u32(&s_half[i]), 1);
            mbar_init(smem_u32(&s_turn[i]), 1);
            mbar_init(smem_u32(&s_done[i]), 1);
        }
        mbar_init(smem_u32(&s_q), 256);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem = uniform(s_tmem);
    griddep_wait();
    griddep_launch();          // own_kernel, which reads nothing that precedes this launch in the stream but what has ended here

    // Keys and values come through rings.  With two row tiles: one ring of tiles of 128 keys or values, tile t's at 2 t and 2 t + 1, which both groups use.  With
    // a lone one: a ring for each group, of halves of tiles in the order in which its products take them.  Whoever waits for an entry has used the one before it
    // in its place (in a ring that two groups share by turns, the parity of a barrier two phases behind would let a group go on).
    const auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, &s_abort, &g_attn_flag, kFlagLmWait)); };
    // (For two row tiles and for a lone one apart, so that strides are constants.)
    const auto copies = [&](auto kind) __attribute__((always_inline)) {
        constexpr bool TWO = decltype(kind)::value;
        // With two row tiles one warp copies keys, one values, otherwise each what one group takes.  A lane copies a box: `box_rows` tokens of a page, 64 values of
        // each.  Its pages are looked up two copies ahead, by asynchronous copies into its own words: a load into a register is waited for as soon as the
        // register is moved, 1300 clocks a copy.  (One warp for all: 2500 clocks for a tile's keys and values, where all else takes 1650.)  Rolled up: what runs
        // once comes from memory, too, and cost a short prefix 4 us.
        constexpr int tokens = TWO ? 128 : 64, kAhead = 2;                        // of a copy
        const int box = lane / kBlocks, blk = lane % kBlocks, which = warp == 11, mine = TWO ? n : 2 * ((n - which + 1) / 2);
        const int pages_1 = tokens / a.page, rows_1 = tokens % a.page, pages_3 = 192 / a.page, rows_3 = 192 % a.page;
        struct Where {                                 // a copy's first token, and where it lies for this lane
            int first, at, row;
        };
        const auto advance = [&](Where& w, int i) {    // from copy i: the halves of a tile are neighbours, the group's tiles are not
            const bool far = !TWO && (i & 1);
            w.first += far ? 192 : tokens;
            w.at += far ? pages_3 : pages_1;
            w.row += far ? rows_3 : rows_1;
            if (w.row >= a.page) { w.row -= a.page; ++w.at; }
        };
        const uint32_t words = smem_u32(&s_pages[which][0][lane]);
        Where ahead = {(TWO ? kt0 : kt0 + which) * 128, 0, 0};
        ahead.at = (ahead.first + box * a.box_rows) / a.page;
        ahead.row = ahead.first + box * a.box_rows - ahead.at * a.page;
        Where keys = ahead, values = ahead;
        const auto look_up = [&](int i) {
            if (i < mine && box * a.box_rows < tokens && ahead.first + box * a.box_rows < a.prefix_len)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(words + (i & 3) * 128), "l"(a.prefix_pages + ahead.at) : "memory");
            asm volatile("cp.async.commit_group;" ::: "memory");
            advance(ahead, i);
        };
        uint32_t st = TWO ? which : 0, parity = 1;
        const auto copy = [&](const Where& w, int i, const CUtensorMap* map) {
            const int boxes = (max(min(tokens, a.prefix_len - w.first), 0) + a.box_rows - 1) / a.box_rows, entry = TWO ? (int)st : which * kStages + (int)st;
            if (!wait(&s_empty[entry], parity)) return false;                     // (the first time round at once)
            const uint32_t bar = smem_u32(&s_full[entry]);
            if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(boxes * kBlocks * a.box_rows * 128));
            __syncwarp();
            if (box < boxes) {
                int page;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(page) : "r"(words + (i & 3) * 128) : "memory");
                if ((uint32_t)page >= (uint32_t)a.n_pages) {
                    atomicExch(&g_attn_flag, kFlagLmPage);
                    page = a.n_pages;                  // outside of the map: zeros
                }
                const uint32_t to = TWO ? ring + entry * kTile + blk * kBlock : ring + entry * kHalfTile + blk * (kBlock / 2);
                tma_load_4d(to + box * a.box_rows * 128, map, blk * 64, w.row, kvh, page, bar);
            }
            __syncwarp();
            st += TWO ? 2 : 1;
            if (st >= (TWO ? kStages - 1 : kStages)) { st -= TWO ? kStages - 1 : kStages; parity ^= 1; }
            return true;
        };
#pragma unroll 1
        for (int i = 0; i < kAhead; ++i) look_up(i);
        bool ok = true;
#pragma unroll 1
        for (int i = 0; ok && i < mine + (TWO || !mine ? 0 : 2); ++i) {            // keys i and values i - 2 of a group; the one or the other
            asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
            if (!TWO && i >= 2) {
                ok = copy(values, i - 2, &vmap);
                advance(values, i - 2);
            }
            if (ok && i < mine) {
                ok = copy(keys, i, TWO && which ? &vmap : &kmap);
                advance(keys, i);
            }
            look_up(i + kAhead);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    };
    const auto products = [&](auto kind) __attribute__((always_inline)) {
        constexpr bool TWO = decltype(kind)::value;
        // The products of one softmax group: two warps, so that the waits of one lie under the products of the other.
        constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10);
        constexpr uint32_t idesc_s = (1u << 4) | kType | ((64u >> 3) << 17) | ((128u >> 4) << 24);
        constexpr uint32_t idesc_o = (1u << 4) | kType | (1u << 16) | (((uint32_t)DP >> 3) << 17) | ((128u >> 4) << 24);
        const int g = warp - 9, mine = TWO ? n : (n - g + 1) / 2;      // key tiles of this group: all, or g, g + 2 ...
        const uint32_t d_s = tmem + g * 128, d_o = tmem + 256 + g * DP, block = TWO ? kBlock : kBlock / 2, entry = TWO ? kTile : kHalfTile, first = TWO ? 0 : g * kStages;
        const uint64_t desc_q = umma_desc_sw128(q_smem + (TWO ? g * kTile : 0)), desc_k = umma_desc_sw128(ring + first * entry), desc_v = umma_desc_sw128_mn(ring + first * entry, block);
        const uint32_t high_k = (uint32_t)(desc_k >> 32), high_v = (uint32_t)(desc_v >> 32), low_q = (uint32_t)desc_q;
        struct Place {
            uint32_t st, parity;
            __device__ __forceinline__ void on(uint32_t by, uint32_t stages) {
                st += by;
                if (st >= stages) { st -= stages; parity ^= 1; }
            }
        };
        Place keys = {0, 0}, values = {1, 0};          // (with a lone row tile `keys` alone, for both)
        // With two row tiles the groups take turns at the tensor cores, a half's values and the next scores in its place at a time: one's softmax then lies under
        // the other's products.  (Left alone they fall into step: products of both mixed, then softmax of both.)  The turn goes on with half of the scores still
        // to be issued, so that the other warp has seen it when they have been.
        uint32_t turn = 0;
        const auto take_turn = [&]() {
            if (!TWO) return true;
            const bool now = wait(&s_turn[g], turn);
            turn ^= 1;
            return now;
        };
        // Scores of 64 keys, the first or second half of a tile, into their own 64 columns.
        const auto scores = [&](uint32_t h) {
            if ((h == 0 || !TWO) && !wait(&s_full[first + keys.st], keys.parity)) return false;
            tcgen05_fence_after();
            const uint32_t low = (uint32_t)desc_k + keys.st * (entry >> 4) + (TWO ? h * (8192 >> 4) : 0);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
                    if (TWO && k == DP / 32) mbar_arrive(smem_u32(&s_turn[g ^ 1]));
                    tcgen05_mma_bf16(d_s + h * 64, pack_f32x2(low_q + (k >> 2) * (kBlock >> 4) + (k & 3) * 2, high_k), pack_f32x2(low + (k >> 2) * (block >> 4) + (k & 3) * 2, high_k), idesc_s, k > 0);
                }
                tcgen05_commit(smem_u32(&s_scores[g][h]));
                if (h == 1 || !TWO) tcgen05_commit(smem_u32(&s_empty[first + keys.st]));
            }
            __syncwarp();
            if (!TWO) keys.on(1, kStages);
            else if (h == 1) keys.on(2, kStages - 1);
            return true;
        };
        bool ok = wait(&s_q, 0);
        if (ok && g == 1) ok = take_turn();
        if (ok && mine > 0) ok = scores(0);
        if (ok) ok = take_turn();
        if (ok && mine > 0) ok = scores(1);
        for (int u = 0; ok && u < mine; ++u) {
            const bool last = u == mine - 1, cut = (TWO ? u : g + 2 * u) == n - 1 && tail < 128;
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                Place& at = TWO ? values : keys;
                if (h == 0 || !TWO) {
                    ok = wait(&s_full[first + at.st], at.parity);
                    if (!ok) break;
                    if (cut) {
                        // Rows behind the prefix's last token: their P is zero, and so is what they hold, which nobody wrote or which may be NaNs.  (With two row
                        // tiles both warps write these zeros before they use them.)
                        const uint32_t v_smem = ring + (first + at.st) * entry;
                        const int all = TWO ? 128 : 64, live = TWO ? tail : min(max(tail - 64 * (int)h, 0), 64);
                        for (int c = lane; c < (all - live) * 8 * kBlocks; c += 32) {
                            const int blk = c / ((all - live) * 8), piece = c % ((all - live) * 8);
                            st_shared_v4(v_smem + blk * block + live * 128 + piece * 16, 0, 0, 0, 0);
                        }
                        fence_proxy_async();
                        __syncwarp();
                    }
                }
                ok = wait(&s_probs[g][h], (uint32_t)u & 1) && take_turn();
                if (!ok) break;
                tcgen05_fence_after();
                const uint32_t low = (uint32_t)desc_v + at.st * (entry >> 4) + (TWO ? h * (8192 >> 4) : 0), more = u > 0;
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tcgen05_mma_f16_ts(d_o, d_s + h * 64 + k * 8, pack_f32x2(low + k * (2048 >> 4), high_v), idesc_o, more | (uint32_t)(h > 0 || k > 0));
                    if (h == 1 || !TWO) tcgen05_commit(smem_u32(&s_empty[first + at.st]));
                    if (last) tcgen05_commit(smem_u32(h == 0 ? &s_half[g] : &s_done[g]));
                }
                __syncwarp();
                if (!TWO) keys.on(1, kStages);
                if (!last) ok = scores(h);
                else if (TWO && elect_one()) mbar_arrive(smem_u32(&s_turn[g ^ 1]));
                __syncwarp();
                if (!ok) break;
            }
            if (TWO) values.on(2, kStages - 1);
        }
    };
    if (warp == 8 || warp == 11) {
        if (two) copies(std::true_type());
        else copies(std::false_type());
    } else if (warp == 9 || warp == 10) {
        if (two) products(std::true_type());
        else products(std::false_type());
    } else if (warp < 8) {
        const int g = warp >> 2, in_tile = (warp & 3) * 32 + lane, rows = a.batch * a.group;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;                       // this warp's lanes of tensor memory
        const int row = (2 * pair + (two ? g : 0)) * 128 + in_tile;
        const bool live_warp = row - lane < rows;
        if (two || g == 0) {
            // neighbouring lanes on neighbouring bytes of a row
            constexpr int kPerRow = DP / 8, kStep = 128 / kPerRow;               // 16-byte pieces of a row; rows from one of a thread's pieces to the next
            const int thread = threadIdx.x & 127, c = thread % kPerRow, r0 = thread / kPerRow, b_step = kStep / a.group, h_step = kStep - b_step * a.group;
            const uint32_t mine = q_smem + g * kTile + (c >> 3) * kBlock + r0 * 128 + (((c & 7) ^ (r0 & 7)) << 4);
            int r = row - in_tile + r0, h = r % a.group;                          // (quotients in the loop took 2 us)
            const int64_t step = b_step * a.q_stride + h_step * a.q_head, wrap = a.q_stride - a.group * a.q_head;
            const T* src = static_cast<const T*>(a.q) + r / a.group * a.q_stride + ((int64_t)kvh * a.group + h) * a.q_head + 8 * c;
#pragma unroll 2
            for (int i = 0; i < kPerRow; ++i) {
                const bool there = r < rows && 8 * c < a.D;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(mine + i * (kStep * 128)), "l"(there ? src : static_cast<const T*>(a.q)), "r"(there ? 16 : 0) : "memory");
                r += kStep;
                h += h_step;
                src += step;
                if (h >= a.group) { h -= a.group; src += wrap; }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (a.scale < 0.f) {                                                 // |scale| from here on
#pragma unroll 1
                for (int i = 0; i < kPerRow; ++i) {
                    const uint4 v = ld_shared_v4(mine + i * (kStep * 128));
                    st_shared_v4(mine + i * (kStep * 128), v.x ^ 0x80008000u, v.y ^ 0x80008000u, v.z ^ 0x80008000u, v.w ^ 0x80008000u);
                }
            }
        }
        fence_proxy_async();
        mbar_arrive(smem_u32(&s_q));

        const float c = fmaxf(fabsf(a.scale) * kLog2e, 1e-38f);                  // (a scale of 0 must not meet the infinities of masked keys)
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        const int mine = two ? n : (n - g + 1) / 2;
        for (int i = 0; i < 2 * mine; ++i) {
            const int h = i & 1;
            ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_scores[g][h]), (uint32_t)(i >> 1) & 1, &s_abort, &g_attn_flag, kFlagLmWait));
            if (!ok) break;
            if (live_warp) {
                tcgen05_fence_after();
                const uint32_t ts = tmem + lanes + g * 128 + h * 64;
                uint32_t s[64], p[32];
                tcgen05_ld32(ts, s);
                tcgen05_ld32(ts + 32, s + 32);
                tcgen05_wait_ld();
                if ((two ? i >> 1 : g + 2 * (i >> 1)) == n - 1 && tail < 128) {
#pragma unroll
                    for (int j = 0; j < 64; ++j)
                        if (j >= tail - 64 * h) s[j] = 0xff800000u;
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < 64; j += 2) top[(j >> 1) & 3] = max3(top[(j >> 1) & 3], __uint_as_float(s[j]), __uint_as_float(s[j + 1]));
                const float next = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
                if (i == 0) {
                    m = next;
                } else if (__any_sync(0xffffffffu, (next - m) * c > kSlack)) {   // (a NaN difference, -inf to -inf, is no growth)
                    // The products of the half before may still be adding to O: the scores behind them tell of their end, or, for the last half, a barrier.
                    ok = __all_sync(0xffffffffu, i + 1 < 2 * mine ? mbar_wait(smem_u32(&s_scores[g][h ^ 1]), (uint32_t)((i + 1) >> 1) & 1, &s_abort, &g_attn_flag, kFlagLmWait)
                                                                  : mbar_wait(smem_u32(&s_half[g]), 0, &s_abort, &g_attn_flag, kFlagLmWait));
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
                    m = next;
                }
                l += values_of<T>(s, c, m == -INFINITY ? 0.f : p_shift<T>() - m * c, p);
                tcgen05_st32(ts, p);
                tcgen05_wait_st();
                tcgen05_fence_before();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&s_probs[g][h]));
        }
        if (ok && mine > 0) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_done[g]), 0, &s_abort, &g_attn_flag, kFlagLmWait));
        // This block's part of the rows.  A lone row tile's two accumulators become one first: the groups exchange halves of the values through the
        // shared memory that all products have left.  A row lies as DP / 4 pieces of 16 bytes, piece i at i ^ (row % 32): 32 rows are written without
        // bank conflicts and leave as one copy.
        constexpr int kPieces = DP / 4;
        const uint32_t my_row = q_smem + (uint32_t)in_tile * (DP * 4);
        const auto piece = [&](uint32_t at, int i) { return at + (uint32_t)((i ^ (in_tile & 31 & (kPieces - 1))) * 16); };
        m = m == -INFINITY ? m : m * c;
        if (!two) {
            const uint32_t swap = q_smem + 128 * DP * 4;                        // (m, l) of both groups behind the rows
            ok = all_of_256(ok);                       // both groups' products have ended
            if (ok) {
                tcgen05_fence_after();
                asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(swap + (g * 128 + in_tile) * 8), "f"(m), "f"(l) : "memory");
                // the half that the other group finishes
#pragma unroll 1
                for (int j = (g ^ 1) * (DP / 2); j < (g ^ 1) * (DP / 2) + DP / 2; j += 32) {
                    uint32_t o[32];
                    tcgen05_ld32(tmem + lanes + 256 + g * DP + j, o);
                    tcgen05_wait_ld();
#pragma unroll
                    for (int e = 0; e < 8; ++e) st_shared_v4(piece(my_row, j / 4 + e), o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                }
            }
            ok = all_of_256(ok);
            if (ok) {
                float m1, l1;
                asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(m1), "=f"(l1) : "r"(swap + ((g ^ 1) * 128 + in_tile) * 8) : "memory");
                const float both = fmaxf(m, m1), f = m == -INFINITY ? 0.f : ex2(m - both), f1 = m1 == -INFINITY ? 0.f : ex2(m1 - both);
                const bool alone = n < 2;              // the second group had no key tile: its accumulator holds nothing
#pragma unroll 1
                for (int j = g * (DP / 2); j < g * (DP / 2) + DP / 2; j += 32) {
                    uint32_t o[32];
                    tcgen05_ld32(tmem + lanes + 256 + g * DP + j, o);
                    tcgen05_wait_ld();
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint4 x = ld_shared_v4(piece(my_row, j / 4 + e));
                        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
                        uint32_t r[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float mine = __uint_as_float(o[4 * e + k]), other = __uint_as_float(w[k]);
                            r[k] = __float_as_uint(alone ? (g ? other : mine) : mine * f + other * f1);
                        }
                        st_shared_v4(piece(my_row, j / 4 + e), r[0], r[1], r[2], r[3]);
                    }
                }
                l = alone ? (g ? l1 : l) : l * f + l1 * f1;
                m = both;
            }
            fence_proxy_async();
            ok = all_of_256(ok);
        } else if (ok) {
            // the other group's products may still read queries and tiles: each group waits for both
            ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&s_done[g ^ 1]), 0, &s_abort, &g_attn_flag, kFlagLmWait));
            if (ok && live_warp) {
                tcgen05_fence_after();
#pragma unroll 1
                for (int j = 0; j < DP; j += 32) {
                    uint32_t o[32];
                    tcgen05_ld32(tmem + lanes + 256 + g * DP + j, o);
                    tcgen05_wait_ld();
#pragma unroll
                    for (int e = 0; e < 8; ++e) st_shared_v4(piece(my_row + g * (128 * DP * 4), j / 4 + e), o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                }
                fence_proxy_async();
            }
            __syncwarp();
        }
        if (ok && live_warp && (two || g == 0)) {
            const int64_t part = ((int64_t)(2 * pair + (two ? g : 0)) * a.kv_heads + kvh) * a.row_parts + split;
            if (row < rows) a.part_ml[part * 128 + in_tile] = make_float2(m, l);
            if (lane == 0) {
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(a.part_o + (part * 128 + in_tile) * DP), "r"(my_row + (two ? g * (128 * DP * 4) : 0)), "n"(32 * DP * 4) : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
            }
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

constexpr int kMaxSplits = 148, kMaxRanks = 8, kMaxParts = 192;
static_assert(kMaxSplits + 4 * kMaxRanks <= kMaxParts && kMaxParts % 32 == 0, "a row's parts");

// ---- own tokens, and the parts together ------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma_16x8x16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

// A block (or a cluster of `ranks` blocks, each a range of the tokens) takes 8 NT query rows of one sequence and key head.  A warp takes 16 tokens at a
// time, copied into a ring of its own two to four chunks ahead: 12 warps of an SM (8 for more than 8 rows) have 96 to 192 KB (64 to 128) on the way.  (In registers, a chunk ahead, it was some 60: 537 MB
// of own tokens took 141 us instead of 88 to 98.)  The order of a head's values within a product's 16 is free as long as both operands have the
// same, and so is the order of O's rows, hence each lane reads 16 bytes as they lie:
//   S^T[token][row] = K Q^T:  lane (g, c) = (lane / 4, lane % 4) holds 8 values at 8 c of every 32 of tokens g and g + 8
//   O^T[value][row] = V^T P^T: 8 values at 8 g of every 64 of tokens 2 c, 2 c + 1, 2 c + 8, 2 c + 9
// Piece i of a row lies at i ^ 4 (row % 2) for keys, at i ^ (row & 6) for values: no bank conflicts.  P^T comes out of S^T with a transposition of 8 x 8 in
// the warp.
template <int DP> struct OwnShape {
    static constexpr uint32_t half = 16 * DP * 2;                    // bytes of 16 tokens' keys or values
    static constexpr int stages = DP == 128 ? 2 : 4;
    static constexpr uint32_t smem = 4 * stages * 2 * half;
};
// Phase 0 does all of it.  Where there are more than three blocks an SM, beside a prefix_kernel, phase 1 leaves its part to phase 2, a launch of its
// own: its blocks then go on while the prefix is worked on, on the SMs that are left over and on those that become free, where blocks that wait for
// the prefix's parts would hold them (220 -> 200 us).
template <typename T, int DP, int NT, int PHASE>
__global__ void __launch_bounds__(128) own_kernel(const __grid_constant__ AttnArgs a, uint32_t job_id, FinishedBlockNotifier* nf) {
    constexpr int R = 8 * NT, KB = DP / 32, VB = DP / 64, kStages = OwnShape<DP>::stages;
    constexpr uint32_t kHalf = OwnShape<DP>::half;
    static_assert(4 * R * DP * 4 <= OwnShape<DP>::smem, "the warps' parts fit where their rings were");
    extern __shared__ __align__(128) uint8_t smem_raw[];
    float (*s_o)[R][DP] = reinterpret_cast<float (*)[R][DP]>(smem_raw);
    __shared__ __align__(8) float2 s_ml[4][R];
    __shared__ float s_w[R][kMaxParts];
    if (PHASE == 2 || !a.early) griddep_wait();
    if (PHASE == 1) griddep_launch();
    if (nf) nf->start(job_id);
    const int warp = (int)uniform(threadIdx.x >> 5), lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const int rank = blockIdx.x % a.ranks;
    int unit = blockIdx.x / a.ranks;
    const int zg = unit % a.row_groups;
    unit /= a.row_groups;
    const int kvh = unit % a.kv_heads, b = unit / a.kv_heads;
    const int row0 = zg * R, rows = b < a.batch ? min(R, a.group - row0) : 0;
    // Chunks of 16 tokens: those of the prefix that are taken here, then the sequence's own.  A lane looks a chunk's two halves of 8 tokens up (a page holds a
    // multiple of 8), for 32 chunks at a time; the first of them before the sequence's length is known, whatever it is: entries up to max_own may be read.
    const int chunks_ahead = (a.ahead + 15) / 16;
    const auto page_of = [&](int chunk, int half) {
        const int token = 16 * (chunk < chunks_ahead ? chunk : chunk - chunks_ahead) + 8 * half;
        if (b >= a.batch || token >= (chunk < chunks_ahead ? a.ahead : a.max_own)) return 0;
        return __ldcg((chunk < chunks_ahead ? a.prefix_pages : a.block_table + b * a.table_stride) + token / a.page);
    };
    int page_lo = 0, page_hi = 0;
    if (PHASE != 2 && a.ranks == 1) {
        page_lo = page_of(warp + 4 * lane, 0);
        page_hi = page_of(warp + 4 * lane, 1);
    }
    int own = 0;
    if (PHASE != 2 && b < a.batch && a.max_own > 0) {
        own = __ldcg(a.own_lens + b);
        if (own < 0 || own > a.max_own) {
            if (threadIdx.x == 0) atomicExch(&g_attn_flag, kFlagLmLength);
            own = own < 0 ? 0 : a.max_own;
        }
    }
    const int chunks = PHASE != 2 && b < a.batch ? chunks_ahead + (own + 15) / 16 : 0, first = (int)((int64_t)chunks * rank / a.ranks) + warp, last = (int)((int64_t)chunks * (rank + 1) / a.ranks);
    const auto token_of = [&](int chunk) { return 16 * (chunk < chunks_ahead ? chunk : chunk - chunks_ahead); };
    const auto limit_of = [&](int chunk) { return chunk < chunks_ahead ? a.ahead : own; };
    float o[VB][4][NT][4] = {};
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) m[t][0] = m[t][1] = -INFINITY, l[t][0] = l[t][1] = 0.f;
    if (PHASE != 2 && first < last) {
        uint4 q[NT][KB];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < KB; ++i) {
                q[t][i] = make_uint4(0, 0, 0, 0);
                if (t * 8 + g < rows && 32 * i + 8 * c < a.D)
                    q[t][i] = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + b * a.q_stride + (int64_t)(kvh * a.group + row0 + t * 8 + g) * a.q_head + 32 * i + 8 * c));
            }
        int64_t at_lo = -1, at_hi = -1;                                        // where a half lies, or -1: zeros
        const auto place = [&](int chunk, int half, int page) -> int64_t {
            const int token = token_of(chunk) + 8 * half;
            if (chunk >= last || token >= limit_of(chunk)) return -1;
            if (page < 0 || page >= a.n_pages) {
                atomicExch(&g_attn_flag, kFlagLmPage);
                return -1;
            }
            return page * a.page_stride + (token % a.page) * a.token_stride + (int64_t)kvh * a.head_stride;
        };
        const auto where = [&](int turn, int64_t& lo, int64_t& hi) {           // of chunk first + 4 turn, turns in order
            if ((turn & 31) == 0) {
                const int chunk = first + 4 * (turn + lane);
                if (turn > 0 || a.ranks > 1) {
                    page_lo = chunk < last ? page_of(chunk, 0) : 0;
                    page_hi = chunk < last ? page_of(chunk, 1) : 0;
                }
                at_lo = place(chunk, 0, page_lo);
                at_hi = place(chunk, 1, page_hi);
            }
            lo = __shfl_sync(0xffffffffu, at_lo, turn & 31);
            hi = __shfl_sync(0xffffffffu, at_hi, turn & 31);
        };
        const uint32_t ring = smem_u32(smem_raw) + warp * (kStages * 2 * kHalf);
        // 16 tokens' keys and values into a stage, neighbouring lanes on neighbouring 16 bytes of a row; what is not there comes as zeros
        constexpr int kPer = DP / 8, kRows = 32 / kPer;                          // pieces of a row, rows of a turn
        const int piece = lane % kPer, row0 = lane / kPer;
        const auto load = [&](int turn) {
            const int chunk = first + 4 * turn;
            if (chunk < last) {
                int64_t lo, hi;
                where(turn, lo, hi);
                const uint32_t to = ring + (turn % kStages) * (2 * kHalf);
                const int left = limit_of(chunk) - token_of(chunk);
                const bool col = 8 * piece < a.D;
#pragma unroll
                for (int i = 0; i < 16 / kRows; ++i) {
                    const int row = i * kRows + row0;
                    const int64_t base = row < 8 ? lo : hi;
                    const bool there = col && base >= 0 && row < left;
                    const int64_t at = there ? base + (row & 7) * a.token_stride + 8 * piece : 0;
                    const uint32_t bytes = there ? 16 : 0, dst = to + row * (DP * 2);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + ((piece ^ ((row & 1) << 2)) << 4)), "l"(static_cast<const T*>(a.k) + at), "r"(bytes) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + kHalf + ((piece ^ (row & 6)) << 4)), "l"(static_cast<const T*>(a.v) + at), "r"(bytes) : "memory");
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        const float scale = a.scale * kLog2e;
#pragma unroll
        for (int i = 0; i < kStages; ++i) load(i);
#pragma unroll 1
        for (int chunk = first, turn = 0; chunk < last; chunk += 4, ++turn) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
            __syncwarp();
            const uint32_t keys = ring + (turn % kStages) * (2 * kHalf), values = keys + kHalf;
            float s[NT][4] = {};
#pragma unroll
            for (int i = 0; i < KB; ++i) {
                const uint4 k0 = ld_shared_v4(keys + g * (DP * 2) + (((4 * i + c) ^ ((g & 1) << 2)) << 4)), k1 = ld_shared_v4(keys + (g + 8) * (DP * 2) + (((4 * i + c) ^ ((g & 1) << 2)) << 4));
                const uint32_t a0[4] = {k0.x, k1.x, k0.y, k1.y}, a1[4] = {k0.z, k1.z, k0.w, k1.w};
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    mma_16x8x16<T>(s[t], a0, q[t][i].x, q[t][i].y);
                    mma_16x8x16<T>(s[t], a1, q[t][i].z, q[t][i].w);
                }
            }
            const int left = limit_of(chunk) - token_of(chunk);
            const bool in0 = g < left, in1 = g + 8 < left;
            float up[NT][2];
            bool grown = false;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    s[t][j] = in0 ? s[t][j] * scale : -INFINITY;
                    s[t][2 + j] = in1 ? s[t][2 + j] * scale : -INFINITY;
                    float x = fmaxf(s[t][j], s[t][2 + j]);
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    up[t][j] = fmaxf(m[t][j], x);
                    grown |= up[t][j] - m[t][j] > kSlack;                // (from -inf, too)
                }
            if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float keep = up[t][j] == m[t][j] ? 1.f : ex2(m[t][j] - up[t][j]);
                        m[t][j] = up[t][j];
                        l[t][j] *= keep;
#pragma unroll
                        for (int i = 0; i < VB; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) { o[i][e][t][j] *= keep; o[i][e][t][2 + j] *= keep; }
                    }
            }
            uint32_t p0[NT], p1[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float b0 = m[t][0] == -INFINITY ? 0.f : m[t][0] - p_shift<T>(), b1 = m[t][1] == -INFINITY ? 0.f : m[t][1] - p_shift<T>();
                const float x0 = ex2(s[t][0] - b0), x1 = ex2(s[t][1] - b1), y0 = ex2(s[t][2] - b0), y1 = ex2(s[t][3] - b1);
                l[t][0] += x0 + y0;
                l[t][1] += x1 + y1;
                p0[t] = transpose_8x8(lm_pack2<T>(x0, x1));
                p1[t] = transpose_8x8(lm_pack2<T>(y0, y1));
            }
#pragma unroll
            for (int i = 0; i < VB; ++i) {
                uint4 v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = ld_shared_v4(values + (2 * c + (e & 1) + 8 * (e >> 1)) * (DP * 2) + (((8 * i + g) ^ (2 * c)) << 4));
                const uint32_t* w0 = &v[0].x; const uint32_t* w1 = &v[1].x; const uint32_t* w2 = &v[2].x; const uint32_t* w3 = &v[3].x;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t av[4] = {__byte_perm(w0[e], w1[e], 0x5410), __byte_perm(w0[e], w1[e], 0x7632), __byte_perm(w2[e], w3[e], 0x5410), __byte_perm(w2[e], w3[e], 0x7632)};
#pragma unroll
                    for (int t = 0; t < NT; ++t) mma_16x8x16<T>(o[i][e][t], av, p0[t], p1[t]);
                }
            }
            __syncwarp();
            load(turn + kStages);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    const auto first_part = [&](int row) {             // of this row's, as a row of part_ml
        const int flat = b * a.group + row0 + row;
        return (((int64_t)(flat >> 7) * a.kv_heads + kvh) * a.row_parts << 7) + (flat & 127);
    };
    constexpr int kPieces = DP / 4;                                       // 16-byte pieces of a row as it lies,
    const int pieces = a.D / 4;                                           // those that hold values
    const auto row_of = [&](int item) { return (int)((uint32_t)item * a.per_piece >> 16); };       // item / pieces, exact below 2048
    if constexpr (PHASE != 2) {
        __syncthreads();                                                  // the rings become the warps' parts
        // this warp's part: (m, l) and O of its rows, values 64 i + 8 g + 2 e and + 1
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float x = l[t][j];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                const int row = 8 * t + 2 * c + j;
                if (g == 0) s_ml[warp][row] = make_float2(m[t][j], x);
#pragma unroll
                for (int i = 0; i < VB; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) *reinterpret_cast<float2*>(&s_o[warp][row][64 * i + 8 * g + 2 * e]) = make_float2(o[i][e][t][j], o[i][e][t][2 + j]);
            }
    }
    if constexpr (PHASE == 1) {
        __syncthreads();
        // the four warps' parts as one (a block has the sequence to itself here)
        for (int item = threadIdx.x; item < rows * pieces; item += 128) {
            const int row = row_of(item), i4 = item - row * pieces;
            float top = -INFINITY, sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < 4; ++w) top = fmaxf(top, s_ml[w][row].x);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float2 ml = s_ml[w][row];
                const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - top);
                const float4 x = *reinterpret_cast<const float4*>(&s_o[w][row][4 * i4]);
                sum = fmaf(f, ml.y, sum);
                acc.x = fmaf(f, x.x, acc.x); acc.y = fmaf(f, x.y, acc.y); acc.z = fmaf(f, x.z, acc.z); acc.w = fmaf(f, x.w, acc.w);
            }
            const int64_t at = first_part(row) + (int64_t)a.splits * 128;
            if (i4 == 0) a.part_ml[at] = make_float2(top, sum);
            reinterpret_cast<float4*>(a.part_o + at * DP)[i4 ^ ((int)at & 31 & (kPieces - 1))] = acc;
        }
        if (blockIdx.x == gridDim.x - 1) griddep_wait();                  // so that this launch ends behind the prefix's
        if (nf) nf->end(job_id);
        return;
    }
    if (PHASE == 0 && a.early) griddep_wait();                            // the prefix's parts
    griddep_launch();
    if (a.ranks > 1) { cluster_arrive(); cluster_wait(); }
    else __syncthreads();

    // The parts joined.  First the weights 2^(m_i - M) / sum 2^(m_i - M) l_i of each row's parts, a row a warp, a part a lane; then a float4 of a row for
    // `lanes` neighbouring threads, which deal the parts out among themselves.
    const int ahead = a.early ? a.row_parts : 0, parts = ahead + (chunks > 0 ? 4 * a.ranks : 0);
    for (int row = warp; row < rows; row += 4) {
        const float2* ml = a.part_ml + first_part(row);
        float2 x[kMaxParts / 32];
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int k = 0; k < kMaxParts / 32; ++k) {
            const int i = lane + 32 * k, w = i - ahead;
            x[k] = make_float2(-INFINITY, 0.f);
            if (i < ahead) x[k] = __ldcg(ml + (int64_t)i * 128);
            else if (i < parts) x[k] = ld_cluster_f2(cluster_addr(smem_u32(&s_ml[w & 3][row]), (uint32_t)w >> 2));
        }
#pragma unroll
        for (int k = 0; k < kMaxParts / 32; ++k) top = fmaxf(top, x[k].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
        for (int k = 0; k < kMaxParts / 32; ++k) {
            x[k].x = x[k].x == -INFINITY ? 0.f : ex2(x[k].x - top);
            sum = fmaf(x[k].x, x[k].y, sum);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float inv = 1.f / sum;
#pragma unroll
        for (int k = 0; k < kMaxParts / 32; ++k)
            if (lane + 32 * k < parts) s_w[row][lane + 32 * k] = x[k].x * inv;
    }
    __syncthreads();
    const int items = rows * pieces;
    int lanes = 1;
    while (lanes < 32 && items * lanes * 2 <= 128 * a.ranks) lanes *= 2;
    const int sub = threadIdx.x & (lanes - 1);
    for (int base = 0; base < items; base += 128 * a.ranks / lanes) {
        const int item = base + (rank * 128 + threadIdx.x) / lanes;
        const bool real = item < items;
        const int row = real ? row_of(item) : 0, i4 = real ? item - row * pieces : 0;
        const int64_t at = first_part(row);
        const float4* src = reinterpret_cast<const float4*>(a.part_o + at * DP) + (i4 ^ ((int)at & 31 & (kPieces - 1)));
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        const auto add = [&](float w, float4 x) {
            acc.x = fmaf(w, x.x, acc.x); acc.y = fmaf(w, x.y, acc.y); acc.z = fmaf(w, x.z, acc.z); acc.w = fmaf(w, x.w, acc.w);
        };
        if (real) {
            int i = sub;
            for (; i + 7 * lanes < ahead; i += 8 * lanes) {
                float4 x[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = __ldcg(src + (int64_t)(i + k * lanes) * 128 * kPieces);
#pragma unroll
                for (int k = 0; k < 8; ++k) add(s_w[row][i + k * lanes], x[k]);
            }
            for (; i < ahead; i += lanes) add(s_w[row][i], __ldcg(src + (int64_t)i * 128 * kPieces));
            for (i = sub; i < parts - ahead; i += lanes)
                add(s_w[row][ahead + i], ld_cluster_f4(cluster_addr(smem_u32(&s_o[i & 3][row][4 * i4]), (uint32_t)i >> 2)));
        }
        for (int k = lanes >> 1; k > 0; k >>= 1) {
            acc.x += __shfl_xor_sync(0xffffffffu, acc.x, k); acc.y += __shfl_xor_sync(0xffffffffu, acc.y, k);
            acc.z += __shfl_xor_sync(0xffffffffu, acc.z, k); acc.w += __shfl_xor_sync(0xffffffffu, acc.w, k);
        }
        if (!real || sub != 0) continue;
        T* dst = static_cast<T*>(a.out) + b * a.out_stride + (int64_t)(kvh * a.group + row0 + row) * a.out_head + 4 * i4;
        if (a.out_vec) {
            *reinterpret_cast<uint2*>(dst) = make_uint2(lm_pack2<T>(acc.x, acc.y), lm_pack2<T>(acc.z, acc.w));
        } else {
            dst[0] = lm_from_f<T>(acc.x); dst[1] = lm_from_f<T>(acc.y); dst[2] = lm_from_f<T>(acc.z); dst[3] = lm_from_f<T>(acc.w);
        }
    }
    // The others have read this block's part.  (Whatever a lane has loaded of theirs has gone into a shuffle or a store in front of its arrival: nothing is left to order.)
    if (a.ranks > 1) { cluster_arrive_relaxed(); cluster_wait(); }
    if (nf) nf->end(job_id);
}

typedef void (*OwnFn)(AttnArgs, uint32_t, FinishedBlockNotifier*);

template <typename T, int PHASE> OwnFn own_fn(int DP, int NT) {
    if (DP == 64) return NT == 1 ? own_kernel<T, 64, 1, PHASE> : own_kernel<T, 64, 2, PHASE>;
    return NT == 1 ? own_kernel<T, 128, 1, PHASE> : own_kernel<T, 128, 2, PHASE>;
}

struct AttnPlan {
    AttnArgs a;
    int DP, NT;
    bool half;
    int64_t prefix_blocks, own_blocks;
    uint64_t scratch;
    OwnFn own, join;           // join: NULL, or phase 2 behind own, phase 1
    uint32_t own_smem;
};

int plan_attn(const pb_prefix_attn_params* p, AttnPlan& pl) {
    const char* who = "pb_prefix_attn";
    PB_REQUIRE(p != nullptr, "%s: NULL params", who);
    PB_REQUIRE(p->dtype == PB_BF16 || p->dtype == PB_F16, "%s: dtype %d (PB_BF16 or PB_F16)", who, p->dtype);
    PB_REQUIRE(p->batch >= 0 && p->q_heads >= 1 && p->kv_heads >= 1 && p->q_heads % p->kv_heads == 0 && p->q_heads <= 65536, "%s: batch %d, %d query heads, %d key heads", who, p->batch, p->q_heads, p->kv_heads);
    PB_REQUIRE(p->head_dim >= 8 && p->head_dim <= 128 && p->head_dim % 8 == 0, "%s: head_dim %d (a multiple of 8, 8 to 128)", who, p->head_dim);
    PB_REQUIRE(p->page_size >= 8 && p->page_size % 8 == 0, "%s: page_size %d (a multiple of 8)", who, p->page_size);
    PB_REQUIRE(p->n_pages >= 0 && p->n_pages <= 0x7fffffff, "%s: %lld pages", who, (long long)p->n_pages);
    PB_REQUIRE(p->prefix_len >= 0 && p->prefix_len <= (1 << 30) && p->max_own_len >= 0 && p->max_own_len <= (1 << 30), "%s: prefix of %d tokens, at most %d own", who, p->prefix_len, p->max_own_len);
    PB_REQUIRE(p->max_blocks >= 0 && p->max_own_len <= (int64_t)p->max_blocks * p->page_size, "%s: %d own tokens do not fit %d pages of %d", who, p->max_own_len, p->max_blocks, p->page_size);
    PB_REQUIRE(p->n_pages > 0 || (p->prefix_len == 0 && p->max_own_len == 0) || p->batch == 0, "%s: a cache without pages", who);
    PB_REQUIRE(fabsf(p->scale) <= 2e38f, "%s: scale is not finite, or above 2e38", who);        // (which in powers of two is finite, too)
    PB_REQUIRE(p->page_stride % 8 == 0 && p->token_stride % 8 == 0 && p->head_stride % 8 == 0 && p->page_stride > 0 && p->token_stride > 0 && p->head_stride > 0, "%s: strides of the cache are positive multiples of 8", who);
    PB_REQUIRE(p->q_stride % 8 == 0 && p->q_head_stride % 8 == 0, "%s: rows of q start on 16 bytes", who);
    PB_REQUIRE(rows_apart(p->batch, p->out_stride, p->head_dim) && rows_apart(p->q_heads, p->out_head_stride, p->head_dim), "%s: rows of out overlap (strides %lld, %lld)", who, (long long)p->out_stride, (long long)p->out_head_stride);
    if (p->batch > 0) {
        PB_REQUIRE(p->q && p->out && p->k_cache && p->v_cache, "%s: NULL buffer", who);
        PB_REQUIRE(aligned(p->q, 16) && aligned(p->k_cache, 16) && aligned(p->v_cache, 16) && aligned(p->out, 2), "%s: q and the cache must be 16-byte aligned", who);
        PB_REQUIRE(p->prefix_len == 0 || (p->prefix_pages && aligned(p->prefix_pages, 4)), "%s: a prefix needs its pages", who);
        PB_REQUIRE(p->max_own_len == 0 || (p->block_table && p->own_lens && aligned(p->block_table, 4) && aligned(p->own_lens, 4)), "%s: own tokens need block_table and own_lens", who);
    }
    AttnArgs& a = pl.a;
    memset(&a, 0, sizeof(a));
    a.q = p->q; a.k = p->k_cache; a.v = p->v_cache; a.out = p->out; a.prefix_pages = p->prefix_pages; a.block_table = p->block_table; a.own_lens = p->own_lens;
    a.q_stride = p->q_stride; a.q_head = p->q_head_stride; a.out_stride = p->out_stride; a.out_head = p->out_head_stride;
    a.page_stride = p->page_stride; a.token_stride = p->token_stride; a.head_stride = p->head_stride; a.table_stride = p->table_stride;
    a.batch = p->batch; a.group = p->q_heads / p->kv_heads; a.D = p->head_dim; a.page = p->page_size; a.n_pages = (int)p->n_pages; a.prefix_len = p->prefix_len;
    a.max_own = p->max_own_len; a.scale = p->scale; a.kv_heads = p->kv_heads;
    a.per_piece = (uint32_t)ceil_div(1 << 16, p->head_dim / 4);
    pl.DP = p->head_dim <= 64 ? 64 : 128;
    pl.NT = a.group <= 8 ? 1 : 2;
    pl.half = p->dtype == PB_F16;
    pl.own_smem = pl.DP == 64 ? OwnShape<64>::smem : OwnShape<128>::smem;
    // The prefix: the same number of parts for all units, as many as keep their blocks within the SMs.  (What is left over works on nothing of the prefix: 20 SMs at 64 units, as
    // many as there are short of 148 at 75 to 147, and the last wave's beyond.)
    const int64_t rows = (int64_t)a.batch * a.group;
    PB_REQUIRE(rows <= (1 << 24), "%s: %lld query rows for a key head", who, (long long)rows);
    a.row_tiles = (int)ceil_div<int64_t>(rows, 128);
    a.pairs = ceil_div(a.row_tiles, 2);
    a.key_tiles = ceil_div(a.prefix_len, 128);
    a.box_rows = 8;
    while (a.box_rows < 64 && p->page_size % (2 * a.box_rows) == 0) a.box_rows *= 2;
    // Own tokens: enough blocks of a cluster on a sequence and key head to use the GPU, 128 tokens each at least, and no more than three an SM.  Those fit it at once for
    // groups of up to 8 query heads; larger groups' blocks (79 KB) fit it two at a time, but halving their number there costs more often than it gains, since lengths differ and
    // shorter ranges even them out.  (16 heads a key head, lengths from 0 to the most, at most three / two an SM: 20 sequences of up to 2048 29.5 / 34.9 us, 25 of 4096
    // 53.9 / 61.3, 12 of 4096 35.8 / 37.4, 6 of 4096 28.7 / 24.1; behind 8192 tokens, where the number also decides whether the parts are joined apart: 20 of 2048 53.9 / 57.9, 40 of 512
    // 58.0 / 58.8, 52 of 1024 80.5 / 78.3, and of 32 heads a key head 40 of 512 57.4 / 50.0.)
    a.row_groups = ceil_div(a.group, 8 * pl.NT);
    const int64_t own_units = (int64_t)a.batch * a.kv_heads * a.row_groups;
    constexpr int kMaxOwnBlocks = 3 * 148;
    const auto ranks_of = [&](int64_t tokens) {
        int ranks = 1;
        while (ranks < kMaxRanks && own_units * ranks * 2 <= kMaxOwnBlocks && tokens / (2 * ranks) >= 128) ranks *= 2;
        return ranks;
    };
    // A short prefix is taken as if it were each sequence's own, where that costs little: a block's tokens come at some 70 bytes a nanosecond, those of all
    // blocks from the L2 cache at 9 KB.  (8 key heads of 128, with the own kernel alone / with both: one sequence behind 512, 4096, 8192 tokens 6.8 / 9.5 us,
    // 10.3 / 11.4, 16.1 / 14.7; 8 behind 256 and 1024 6.9 / 9.1, 10.8 / 9.2; 32 behind 256 and 512 10.2 / 10.0, 13.4 / 10.7.)
    const int64_t tokens = (int64_t)a.prefix_len + a.max_own;
    const double bytes = 4.0 * a.D * a.prefix_len, block_us = bytes / ranks_of(tokens) / 70e3, all_us = bytes * own_units / 9e6;
    const char* force = getenv("PB_ATTN_PREFIX");          // 1 = prefix_kernel wherever there is a prefix, 0 = never; by rule otherwise
    a.ahead = (force && force[0] ? force[0] == '0' : block_us < 6.0 && all_us < 3.5) ? a.prefix_len : 0;
    a.early = a.prefix_len > a.ahead && own_units > 0;
    a.ranks = own_units > 0 ? ranks_of(a.ahead + (int64_t)a.max_own) : 1;
    pl.own_blocks = std::max<int64_t>(own_units * a.ranks, 1);
    const int64_t units = (int64_t)a.pairs * a.kv_heads;
    a.splits = 1;
    if (units > 0 && units < kMaxSplits) a.splits = (int)(kMaxSplits / units);
    if (a.splits > a.key_tiles) a.splits = a.key_tiles > 0 ? a.key_tiles : 1;
    pl.prefix_blocks = a.early ? units * a.splits : 0;
    const bool apart = a.early && own_units > kMaxOwnBlocks && a.max_own > 0;
    a.row_parts = a.splits + (apart ? 1 : 0);
    pl.own = pl.half ? (apart ? own_fn<__half, 1> : own_fn<__half, 0>)(pl.DP, pl.NT) : (apart ? own_fn<__nv_bfloat16, 1> : own_fn<__nv_bfloat16, 0>)(pl.DP, pl.NT);
    pl.join = !apart ? nullptr : pl.half ? own_fn<__half, 2>(pl.DP, pl.NT) : own_fn<__nv_bfloat16, 2>(pl.DP, pl.NT);
    const uint64_t parts = a.early ? (uint64_t)a.row_tiles * a.kv_heads * a.row_parts * 128 : 0;
    pl.scratch = parts * ((uint64_t)pl.DP * 4 + 8);
    a.part_o = (float*)p->scratch;
    a.part_ml = (float2*)((char*)p->scratch + parts * pl.DP * 4);
    PB_REQUIRE(pl.prefix_blocks <= 0x7fffffff && pl.own_blocks <= 0x7fffffff, "%s: too many blocks for one launch", who);
    a.out_vec = aligned(p->out, 8) && a.out_stride % 4 == 0 && a.out_head % 4 == 0;
    return PB_OK;
}

const void* prefix_fn(const AttnPlan& pl) {
    if (pl.DP == 64) return pl.half ? (const void*)prefix_kernel<__half, 64> : (const void*)prefix_kernel<__nv_bfloat16, 64>;
    return pl.half ? (const void*)prefix_kernel<__half, 128> : (const void*)prefix_kernel<__nv_bfloat16, 128>;
}

template <typename T, int DP>
int launch_prefix(const AttnPlan& pl, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
    PB_CUDA(cudaFuncSetAttribute(prefix_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PrefixShape<DP>::smem));
    return lm_launch("pb_prefix_attn (prefix)", prefix_kernel<T, DP>, dim3((unsigned)pl.prefix_blocks), dim3(384), PrefixShape<DP>::smem, st, 1, pl.a, km, vm);
}

}  // namespace

uint32_t* lm_attn_error_flag_ptr() {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_attn_flag) != cudaSuccess) { cudaGetLastError(); return nullptr; }
    return (uint32_t*)p;
}

}  // namespace pb

using namespace pb;

extern "C" {

int pb_prefix_attn_info(const pb_prefix_attn_params* p, pb_launch_info* out) {
    AttnPlan pl;
    const int rc = plan_attn(p, pl);
    if (rc != PB_OK) return rc;
    PB_REQUIRE(out != nullptr, "pb_prefix_attn_info: NULL out");
    memset(out, 0, sizeof(*out));
    // The last kernel reports, so its blocks are declared; the scheduler takes what they declare from the launch on, so together they declare the most that any of the launch's
    // kernels holds.
    out->num_blocks = (uint32_t)pl.own_blocks;
    uint64_t threads = 0, smem = 0, regs = 0, columns = 0;
    const auto holds = [&](const void* fn, int64_t blocks, uint64_t block_threads, uint64_t dynamic, uint64_t block_columns) {
        cudaFuncAttributes fa = {};
        if (cudaFuncGetAttributes(&fa, fn) != cudaSuccess) cudaGetLastError();       // (without a GPU: what the host knows)
        threads = std::max<uint64_t>(threads, blocks * block_threads);
        smem = std::max<uint64_t>(smem, blocks * (fa.sharedSizeBytes + dynamic));
        regs = std::max<uint64_t>(regs, blocks * block_threads * fa.numRegs);
        columns = std::max<uint64_t>(columns, blocks * block_columns);
    };
    if (pl.prefix_blocks > 0) holds(prefix_fn(pl), pl.prefix_blocks, 384, pl.DP == 64 ? PrefixShape<64>::smem : PrefixShape<128>::smem, 512);
    holds((const void*)pl.own, pl.own_blocks, 128, pl.own_smem, 0);
    if (pl.join) holds((const void*)pl.join, pl.own_blocks, 128, 0, 0);
    out->threads_per_block = (uint32_t)ceil_div<uint64_t>(threads, pl.own_blocks);
    out->smem_per_block = (uint32_t)ceil_div<uint64_t>(smem, pl.own_blocks);
    out->regs_per_thread = (uint32_t)ceil_div<uint64_t>(regs, (uint64_t)pl.own_blocks * out->threads_per_block);
    out->tmem_cols_per_block = (uint32_t)ceil_div<uint64_t>(columns, pl.own_blocks);
    const uint64_t seen = (uint64_t)p->prefix_len + (uint64_t)p->batch * p->max_own_len;
    out->flops = 4ull * p->head_dim * p->q_heads * p->batch * ((uint64_t)p->prefix_len + p->max_own_len);
    out->bytes = p->batch ? 4ull * p->head_dim * (p->kv_heads * seen + (uint64_t)p->batch * p->q_heads) : 0;
    out->scratch_bytes = pl.scratch;
    return PB_OK;
}

int pb_prefix_attn_launch(const pb_prefix_attn_params* p, void* stream, uint32_t job_id, void* notifier) {
    AttnPlan pl;
    const int rc = plan_attn(p, pl);
    if (rc != PB_OK) return rc;
    const cudaStream_t st = (cudaStream_t)stream;
    if (pl.prefix_blocks > 0) {
        PB_REQUIRE(p->scratch != nullptr && p->scratch_bytes >= pl.scratch && aligned(p->scratch, 16), "pb_prefix_attn: %llu bytes of scratch memory are needed, 16-byte aligned (%llu given)",
                   (unsigned long long)pl.scratch, (unsigned long long)(p->scratch ? p->scratch_bytes : 0));
        // [page][head][token][value] whatever the order in memory; a dimension of one needs no stride of its own
        const uint64_t dims[4] = {(uint64_t)p->head_dim, (uint64_t)p->page_size, (uint64_t)p->kv_heads, (uint64_t)p->n_pages};
        const uint64_t strides[3] = {(uint64_t)p->token_stride * 2, p->kv_heads > 1 ? (uint64_t)p->head_stride * 2 : 16, p->n_pages > 1 ? (uint64_t)p->page_stride * 2 : 16};
        const uint32_t box[4] = {64, (uint32_t)pl.a.box_rows, 1, 1};
        const CUtensorMapDataType type = pl.half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        CUtensorMap km, vm;
        int e = encode_tiled_sw128(type, p->k_cache, 4, dims, strides, box, &km);
        if (e == PB_OK) e = encode_tiled_sw128(type, p->v_cache, 4, dims, strides, box, &vm);
        if (e == PB_OK) {
            if (pl.half) e = pl.DP == 64 ? launch_prefix<__half, 64>(pl, km, vm, st) : launch_prefix<__half, 128>(pl, km, vm, st);
            else e = pl.DP == 64 ? launch_prefix<__nv_bfloat16, 64>(pl, km, vm, st) : launch_prefix<__nv_bfloat16, 128>(pl, km, vm, st);
        }
        if (e != PB_OK) return e;
    }
    PB_CUDA(cudaFuncSetAttribute(pl.own, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pl.own_smem));
    FinishedBlockNotifier* nf = (FinishedBlockNotifier*)notifier;
    const dim3 blocks((unsigned)pl.own_blocks);
    if (!pl.join) return lm_launch("pb_prefix_attn", pl.own, blocks, dim3(128), pl.own_smem, st, pl.a.ranks, pl.a, job_id, nf);
    const int e = lm_launch("pb_prefix_attn (own tokens)", pl.own, blocks, dim3(128), pl.own_smem, st, 1, pl.a, job_id, (FinishedBlockNotifier*)nullptr);
    if (e != PB_OK) return e;
    return lm_launch("pb_prefix_attn (parts)", pl.join, blocks, dim3(128), 0, st, 1, pl.a, job_id, nf);
}

}  // extern "C"
