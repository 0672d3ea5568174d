// Attention of a packed run's sequences of many rows on the 5th-generation tensor cores (F16 precision, f16 and 8-bit caches), over pages.
//
// An item is 256 rows of one sequence against one key head, in two tiles of 128; a row is a token and a head of the group, so that short
// prompts of grouped heads fill their tiles and all heads of a group share K and V. The run's items lie in a line that is cut evenly over the SMs
// (packed.cuh); what a piece holds of an item that goes on in another is left as O, m and l for the merge. Keys go in steps of 64: S = Q K^T (128 x 64) into
// tensor memory, twice for each row tile, so that the next step's scores are made while this step's weights are formed; O += P V reads P out of
// the columns that S had. One pass: running maximum and sum by row, O in tensor memory, scaled anew only when a score passes the reference by 8.
//
// Roles: warps 0-7 the softmax, a thread to a row, a row tile to four warps; warps 8 and 9 issue a row tile's products each, so that neither waits
// for the other's weights; then the copies. f16: a warp each for K and V, since a warp issues a TMA copy (16 positions x 64 dims, half a page) every 80 cycles,
// sixteen to a tile of 128 keys. 8 bit: three warps each read codes and scales, turn them into f16(d * code) and store them swizzled; a tile's codes are asked for
// when the tile before is stored, behind the fence, which would wait for them (two warps each, at the 8-bit figure below: 493 us when three took 444). Tiles go
// through two slots for K and two for V. The copying warp of K walks the line and hands each share on; a share's queries are fetched while the
// share before has its last step. The row tiles take turns with the exponentials: side by side, both would hold the unit up and then leave it idle.
//
// Cache rows behind the item's last position may hold anything: their scores are replaced before they count, and V's are written as zeros. A
// row whose output is not finite although new tokens lie behind it may be taken again without them, when the block's shares are done (packed_rows_again).
// Rounded to fewer than 32 bits: q * scale and the weights to f16, as the product takes them (2^-11 each, what the F16 precision says), an 8-bit cache's values
// likewise, the output to f16. l sums the rounded weights, so that their error largely cancels in O / l.
//
// Bound by the round of a step, not by one unit: a row tile's scores, exponentials (16 a clock and SM, 1024 cycles for both row tiles' 64 keys), the weights' way
// into tensor memory and their product follow one another, with two row tiles and two steps in flight; with 1024 tokens behind 5000 the tensor core works 39 % of the
// time and the exponential unit 40 %. Measured: 1000 new tokens behind 9000 (64 heads on 8 key heads, behind a flush of the L2) 357 us, 871 TFLOP/s, with an 8-bit cache 445 us,
// 699 TFLOP/s (the conversions take issue slots and registers from the softmax); 14 prompts of 16 138 tokens (32 on 8) 569 us, 651 TFLOP/s.
#include <math.h>
#include <string.h>

#include "packed_tc.h"
#include "tc_device.cuh"

using namespace brasa_dev;

namespace {

constexpr uint32_t PAGE = BRASA_KV_PAGE, D = 128, WAIT_LIMIT = 1u << 22, TILE_BYTES = 128 * 128 * 2, ROWS = PACKED_TC_ROWS;
constexpr uint32_t SOFTMAX_WARPS = 8, MMA_WARP = 8, K_WARP = 10, V_WARP = 11;  // (one MMA warp for each row tile)
constexpr uint32_t THREADS = 384, WARPS_Q8 = 3, THREADS_Q8 = 512;  // an 8-bit pool's K and V have three warps each

struct PackedMaps {
    CUtensorMap k, v;
};
struct PackedTcParams {
    PackedLine l;
    const float *q;
    const uint8_t *kpool, *vpool;
    __half *o;
    float *part;
    PackedNote *notes;
    uint32_t hq;
    float scale;
    uint32_t *status;
};

// A block's share of an item, as the copying warp hands it on: the other roles keep no place in the line.
struct PackedShare {
    uint32_t t0, rows, kh, past;  // its first row of the run, its rows (0: there are no more), key head, positions before its first token
    uint32_t seq, nkeys;          // sequence, keys that its last token sees
    uint32_t j0, len, steps;      // first key tile, key tiles, steps of 64 keys as far as any are seen
    uint32_t whole;               // all of the item's keys
};
// A place of the ring is written again when every warp is done with the share that it held: the second row tile's softmax has no part in an item of up to
// 128 rows, and nothing else keeps the copies from going round while it is at an output.
constexpr uint32_t SHARES = 8;

// byte offset of the 16-byte piece of columns [c, c + 8) of row r in a swizzled 128 x 128 tile of 16-bit values
__device__ __forceinline__ uint32_t tile_piece(uint32_t r, uint32_t c) {
    return (c >> 6) * 16384 + (r >> 3) * 1024 + (r & 7) * 128 + ((((c >> 3) & 7) ^ (r & 7)) << 4);
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t v[32]) {  // (the caller waits for its loads)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
        "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
          "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
          "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]),
          "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t v[8]) {  // (the caller waits for its stores)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t v[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// adds both halves of a pair to a sum of 32 bits: the sum of the weights that the product reads, rounded as they are
__device__ __forceinline__ void add_halves(uint32_t pair, float &a, float &b) {
    asm("{\n\t.reg .b16 x, y;\n\tmov.b32 {x, y}, %2;\n\tadd.rn.f32.f16 %0, x, %0;\n\tadd.rn.f32.f16 %1, y, %1;\n\t}" : "+f"(a), "+f"(b) : "r"(pair));
}

// Rows before a value that is not finite: all warps walk the block's piece once more, now that none waits for another.
template <bool Q8>
__device__ __noinline__ void packed_tc_again(const PackedTcParams &p, PackedItem it, const PackedItem &end) {
    for (bool more = true; more && (it.first < end.first || (it.first == end.first && it.j < end.j));) {
        const uint32_t j1 = it.first == end.first ? end.j : it.tiles, token0 = it.part * p.l.item_tokens;
        packed_rows_again<Q8 ? BRASA_KV_Q8_0 : BRASA_KV_F16, true>(
            p.l, PackedAgain{p.q, p.kpool, p.vpool, p.o, p.part + (size_t)(2 * blockIdx.x + (it.j == 0)) * packed_part_floats(ROWS), p.hq, p.scale, it.seq, it.kh, it.t0 + token0,
                             line_tokens(p.l, it) * p.l.group, it.past + token0, 128 * it.j, min(line_keys(p.l, it), 128 * j1), ROWS, it.j == 0 && j1 == it.tiles});
        more = j1 == it.tiles && line_next(p.l, it);
    }
}

template <bool Q8>
__global__ void __launch_bounds__(Q8 ? THREADS_Q8 : THREADS, 1) attn_packed_tc_kernel(const __grid_constant__ PackedMaps maps, const __grid_constant__ PackedTcParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *ring = smem + 2 * TILE_BYTES;
    __shared__ uint64_t full[2][2], freed[2][2], q_full[2], s_ready[2][2], p_ready[2][2], pv_done[2], o_done[2], turn[2], share_full[SHARES], share_free[SHARES];
    __shared__ PackedShare shares[SHARES];
    __shared__ uint32_t tmem_base_s, abort_s, again_s, there_s[8];  // (there: of the last key tiles, which of their eight pages are pages)
    __shared__ PackedPieces pieces;
    __shared__ PackedNote note;
    __shared__ PackedItem begin;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = p.l.group, hkv = p.l.v.hkv;

    if (tid == 0) {
        for (uint32_t i = 0; i < 4; ++i) {  // [K or V][slot]
            mbar_init(&full[i >> 1][i & 1], Q8 ? WARPS_Q8 : 1);
            mbar_init(&freed[i >> 1][i & 1], 2);  // by either row tile's products
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 4);  // one arrival per softmax warp of the row tile
            for (int b = 0; b < 2; ++b) {
                mbar_init(&s_ready[i][b], 1);
                mbar_init(&p_ready[i][b], 4);
            }
            mbar_init(&pv_done[i], 1);
            mbar_init(&turn[i], 4);  // of the other row tile's warps
            mbar_init(&o_done[i], 1);
        }
        for (uint32_t i = 0; i < SHARES; ++i) {
            mbar_init(&share_full[i], 1);
            mbar_init(&share_free[i], 2 * (Q8 ? WARPS_Q8 : 1) - 1 + 2 + SOFTMAX_WARPS);  // by all warps but the one that walks
        }
        abort_s = again_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMA_WARP) {  // tensor memory: S of A, two steps, then P over them, in [0, 128), of B in [128, 256); O of A in [256, 384), of B in [384, 512)
        const uint32_t ncols = 512;
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(ncols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    // launched as a programmatic dependent: what the kernels before this one wrote (q, the cache, its tables) is touched after the wait
    pdl_wait();
    pdl_launch();
    const uint32_t tmem = tmem_base_s;
    volatile uint32_t *abort_flag = &abort_s;
    auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
        for (uint32_t it = 0; it < WAIT_LIMIT; ++it) {
            if (tc_mbar_try(bar, parity)) return true;
            if (*abort_flag) return false;
        }
        atomicExch(p.status, 7u);
        *abort_flag = 1;
        return false;
    };
    auto all_wait = [&](uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };

    if (smem_u32(smem) & 1023) {  // (the swizzle counts from there)
        if (tid == 0) atomicExch(p.status, 8u);
        abort_s = 1;
    }
    const bool work = line_cut<256>(p.l, pieces) && !abort_s;
    auto share_at = [&](uint32_t i) -> bool { return all_wait(&share_full[i % SHARES], (i / SHARES) & 1); };  // the block's i-th share is handed on
    auto share_done = [&](uint32_t i) {  // and this warp has read what it needs of it
        __syncwarp();
        if (lane == 0) tc_mbar_arrive(&share_free[i % SHARES]);
    };

    if (warp >= K_WARP) {  // ---- copies, as far ahead of the products as there are slots; K's warp walks the line and hands the shares on ----
        const uint32_t is_v = (warp - K_WARP) & 1;
        const bool walks = warp == K_WARP;
        PackedItem &item = pieces.at[0];  // (where the walk is: one lane's, in shared memory, since the converting warps have no registers to spare)
        const PackedItem &end = pieces.at[1];
        bool more = false, ok = true;
        if (walks && lane == 0) {
            if (work && item.j == item.tiles) line_next(p.l, item);
            begin = item;
            more = work && (item.first < end.first || (item.first == end.first && item.j < end.j));
            note = PackedNote{};
        }
        uint32_t loads = 0;  // tiles copied so far
#pragma unroll 1
        for (uint32_t n = 0; ok; ++n) {
            PackedShare &share = shares[n % SHARES];
            if (walks) {
                if (n >= SHARES && !(ok = all_wait(&share_free[n % SHARES], (n / SHARES - 1) & 1))) break;
                if (lane == 0) {
                    share.rows = 0;
                    if (more) {
                        const uint32_t j1 = item.first == end.first ? end.j : item.tiles, token0 = item.part * p.l.item_tokens, rows = line_tokens(p.l, item) * G;
                        share = PackedShare{item.t0 + token0, rows, item.kh, item.past + token0, item.seq, line_keys(p.l, item), item.j, j1 - item.j, min(2 * (j1 - item.j), (line_keys(p.l, item) - 128 * item.j + 63) / 64),
                                            item.j == 0 && j1 == item.tiles};
                        if (j1 < item.tiles && item.j == 0) note = PackedNote{1, note.closes, item.t0 + token0, rows, item.kh};
                        if (item.j > 0 && j1 == item.tiles) note.closes = 1;
                    } else p.notes[blockIdx.x] = note;
                    tc_mbar_arrive(&share_full[n % SHARES]);
                }
                __syncwarp();
            } else ok = share_at(n);
            if (!ok || share.rows == 0) break;
            const uint32_t j0 = share.j0, len = share.len, nkeys = share.nkeys, kh = share.kh;
            const int32_t *table = p.l.v.table + (size_t)share.seq * p.l.v.max_pages;
            auto page_at = [&](uint32_t i) { return (uint64_t)16 * i < nkeys ? table[i] : -1; };  // as the table has it, -1 where nothing is seen
            if (warp == V_WARP)  // the queries on their way into L2
                for (uint32_t t = lane; t * G < share.rows; t += 32)
                    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.q + ((size_t)(share.t0 + t) * p.hq + kh * G) * D), "r"(G * D * 4) : "memory");
            if constexpr (Q8) {
                // Rows are turned into f16(d * code) on the way: this warp has pages w, w + 3 and w + 6 of a tile, two rows at a time, eight codes a lane; a tile's codes are
                // fetched while the tile before is turned.
                const uint32_t w = (warp - K_WARP) >> 1, c = lane & 15, r2 = lane >> 4;
                const size_t page_bytes = (size_t)PAGE * hkv * 136;
                const uint32_t step = 2 * hkv * 136;  // two rows on
                const uint8_t *codes0 = (is_v ? p.vpool : p.kpool) + (r2 * hkv + kh) * 136 + 8 * c;
                const uint8_t *scales0 = (is_v ? p.vpool : p.kpool) + ((lane >> 1) * hkv + kh) * 136 + 128 + 4 * (lane & 1);  // two scales of a row a lane, for a page
                uint2 code[24];
                uint32_t scale[3];
                uint32_t there = 0, to[4];  // (rows four pairs apart are swizzled alike)
#pragma unroll
                for (uint32_t u = 0; u < 4; ++u) to[u] = tile_piece(16 * w + 2 * u + r2, 8 * c);
                auto fetch = [&](uint32_t j) {  // of tile j0 + j
                    const int32_t mine = j < len ? page_at(8 * (j0 + j) + (lane & 7)) : -1;
                    there = __ballot_sync(0xffffffffu, (uint32_t)mine < p.l.v.num_pages) & 255u;
#pragma unroll
                    for (uint32_t g = 0; g < 3; ++g) {
                        const uint32_t i = w + WARPS_Q8 * g, first = 128 * (j0 + j) + 16 * i;
                        const size_t at = (size_t)(uint32_t)__shfl_sync(0xffffffffu, mine, i & 7) * page_bytes;
                        const uint32_t seen = i < 8 && there >> i & 1 ? min(16u, nkeys - first) : 0;  // rows of the page (a page that is one has some that are seen)
                        scale[g] = lane >> 1 < seen ? *reinterpret_cast<const uint32_t *>(scales0 + at) : 0u;
#pragma unroll
                        for (uint32_t u = 0; u < 8; ++u) {
                            code[8 * g + u] = make_uint2(0, 0);
                            if (2 * u + r2 < seen) code[8 * g + u] = *reinterpret_cast<const uint2 *>(codes0 + at + u * step);
                        }
                    }
                };
                fetch(0);
                for (uint32_t j = 0; j < len; ++j, ++loads) {
                    const uint32_t s = loads & 1;
                    if (loads >= 2 && !(ok = all_wait(&freed[is_v][s], ((loads >> 1) - 1) & 1))) break;
                    uint8_t *slot = ring + (size_t)(2 * is_v + s) * TILE_BYTES;
                    if (walks && lane == 0) there_s[loads & 7] = there;  // (read by whoever sees this tile's scores, four tiles behind at most)
#pragma unroll
                    for (uint32_t e = 0; e < 24; ++e) {
                        if (e >= 16 && w == 2) break;  // (a tile has eight pages)
                        const uint32_t dd = __byte_perm(__shfl_sync(0xffffffffu, scale[e >> 3], 2 * (2 * (e & 7) + r2) + (c >> 3)), 0, c & 4 ? 0x3232 : 0x1010);
                        const __half2 d = *reinterpret_cast<const __half2 *>(&dd);
                        const uint32_t lo = code[e].x ^ 0x80808080u, hi = code[e].y ^ 0x80808080u;
                        *reinterpret_cast<uint4 *>(slot + to[e & 3] + 1024 * (e >> 2 & 1) + 2048 * WARPS_Q8 * (e >> 3)) =
                            make_uint4(bytes_h2(lo, 0x4140, d), bytes_h2(lo, 0x4342, d), bytes_h2(hi, 0x4140, d), bytes_h2(hi, 0x4342, d));
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) tc_mbar_arrive(&full[is_v][s]);
                    fetch(j + 1);
                }
            } else {
                int32_t now = page_at(8 * j0 + lane), ahead = page_at(8 * j0 + 32 + lane);  // the pages of four tiles, and of the next four
                for (uint32_t j = 0; j < len; ++j, ++loads) {
                    const uint32_t k = j & 3, s = loads & 1, half = lane & 1, i = (lane >> 1) & 7;  // lanes 2 i and 2 i + 1 take the halves of page i
                    if (j > 0 && k == 0) {
                        now = ahead;
                        ahead = page_at(8 * (j0 + j) + 32 + lane);
                    }
                    int32_t page = __shfl_sync(0xffffffffu, now, 8 * k + i);
                    if ((uint32_t)page >= p.l.v.num_pages) page = -1;
                    const uint32_t left = nkeys - min(nkeys, 128 * (j0 + j) + 16 * i);  // of the page's positions, those that are seen
                    if (loads >= 2 && !(ok = all_wait(&freed[is_v][s], ((loads >> 1) - 1) & 1))) break;
                    uint8_t *slot = ring + (size_t)(2 * is_v + s) * TILE_BYTES;
                    const bool whole = page >= 0 && (!is_v || left >= 16);
                    const uint32_t odd = is_v ? __ballot_sync(0xffffffffu, !whole) & 0x5555u : 0u;  // (bit 2 i) pages that are not copied whole
                    for (uint32_t bits = odd; bits; bits &= bits - 1) {                             // what is seen of such a page, and zeros
                        const uint32_t e = (__ffs(bits) - 1) >> 1, seen = __shfl_sync(0xffffffffu, page >= 0 ? left : 0u, 2 * e);
                        const int32_t from = __shfl_sync(0xffffffffu, page, 2 * e);
                        uint4 v[8];
#pragma unroll
                        for (uint32_t u = 0; u < 8; ++u) {
                            const uint32_t r = 2 * u + (lane >> 4);
                            v[u] = make_uint4(0, 0, 0, 0);
                            if (r < seen) v[u] = reinterpret_cast<const uint4 *>(p.vpool + (((size_t)from * PAGE + r) * hkv + kh) * 256)[lane & 15];
                        }
#pragma unroll
                        for (uint32_t u = 0; u < 8; ++u) *reinterpret_cast<uint4 *>(slot + tile_piece(16 * e + 2 * u + (lane >> 4), 8 * (lane & 15))) = v[u];
                    }
                    if (odd) {
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                    }
                    const uint32_t copied = __popc(__ballot_sync(0xffffffffu, whole) & 0xffffu), there = __ballot_sync(0xffffffffu, (uint32_t)now < p.l.v.num_pages) >> (8 * k) & 255u;
                    if (lane == 0) {
                        if (!is_v) there_s[loads & 7] = there;  // (K: which pages are pages; read by whoever sees this tile's scores, four tiles behind at most)
                        mbar_expect_tx(&full[is_v][s], copied * 2048);
                    }
                    __syncwarp();
                    if (whole && lane < 16) tma_load_3d(slot + half * 16384 + i * 2048, is_v ? &maps.v : &maps.k, (int)(half * 64), (int)kh, page * (int)PAGE, &full[is_v][s]);
                }
            }
            if (!walks) share_done(n);
            if (walks && ok && lane == 0) {
                const uint32_t j1 = item.first == end.first ? end.j : item.tiles;
                more = j1 == item.tiles && line_next(p.l, item) && (item.first < end.first || (item.first == end.first && end.j > 0));
            }
        }
        if (!Q8 && *abort_flag && lane == 0) {  // leaving early: let the copies in flight land before the block's shared memory is handed on
            for (uint32_t k = loads > 2 ? loads - 2 : 0; k < loads; ++k)
                for (uint32_t it = 0; it < WAIT_LIMIT && !tc_mbar_try(&full[is_v][k & 1], (k >> 1) & 1); ++it) {}
        }
    } else if (warp == MMA_WARP || warp == MMA_WARP + 1) {  // ---- products of one row tile: the warp waits, one lane issues ----
        constexpr uint32_t idesc_s = (1u << 4) | ((64u >> 3) << 17) | ((128u >> 4) << 24), idesc_o = (1u << 4) | (1u << 16) | ((128u >> 3) << 17) | ((128u >> 4) << 24);  // f16; V is MN-major
        const uint32_t x = warp - MMA_WARP, st = tmem + 128 * x, ot = tmem + 256 + 128 * x;
        const uint64_t q = tc_desc_kmajor(smem_u32(smem + x * TILE_BYTES));
        auto landed = [&](uint32_t is_v, uint32_t t) { return all_wait(&full[is_v][t & 1], (t >> 1) & 1); };
        auto slot = [&](uint32_t is_v, uint32_t t) { return smem_u32(ring + (size_t)(2 * is_v + (t & 1)) * TILE_BYTES); };
        uint32_t loads = 0, segs = 0, used = 0;  // of the shares before: key tiles, shares with this row tile, uses of either step's columns
        bool ok = true;
#pragma unroll 1
        for (uint32_t i = 0; ok; ++i) {
            if (!(ok = share_at(i))) break;
            const PackedShare &share = shares[i % SHARES];
            const uint32_t rows = share.rows, len = share.len, steps = share.steps;
            if (rows == 0) break;
            if (x == 1 && rows <= 128) {  // no rows: the slots are given back as they come
                for (uint32_t t = loads; ok && t < loads + len; ++t)
                    for (uint32_t is_v = 0; is_v < 2 && ok; ++is_v) {
                        ok = landed(is_v, t);
                        if (ok && lane == 0) tc_mbar_arrive(&freed[is_v][t & 1]);
                    }
            } else {
                auto scores = [&](uint32_t k) {  // S = Q K^T of step k, over the columns of the P that the product before it has read
                    const uint32_t t = loads + (k >> 1), b = k & 1;
                    if (tc_elect_one()) {
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint64_t kd = tc_desc_kmajor(slot(0, t) + 8192 * b);
#pragma unroll
                        for (uint32_t ks = 0; ks < 8; ++ks) {
                            const uint32_t off = ((ks >> 2) * 16384 + (ks & 3) * 32) >> 4;
                            tc_mma(st + 64 * b, q + off, kd + off, idesc_s, ks > 0 ? 1u : 0u);
                        }
                        tc_commit(&s_ready[x][b]);
                        if (b == 1 || k + 1 == steps) tc_commit(&freed[0][t & 1]);
                    }
                    __syncwarp();
                };
                ok = all_wait(&q_full[x], segs & 1) && landed(0, loads);
                if (ok) scores(0);
                if (ok && steps > 1) scores(1);
                for (uint32_t k = 0; k < steps && ok; ++k) {
                    const uint32_t t = loads + (k >> 1), b = k & 1;
                    if (b == 0) ok = landed(1, t) && (k + 2 >= steps || landed(0, t + 1));
                    ok = ok && all_wait(&p_ready[x][b], ((used >> b & 1) + (k >> 1)) & 1);
                    if (!ok) break;
                    if (tc_elect_one()) {  // O += P V
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint64_t v = tc_desc_mnmajor(slot(1, t) + 8192 * b);
#pragma unroll
                        for (uint32_t ks = 0; ks < 4; ++ks) tc_mma_ta(ot, st + 64 * b + 8 * ks, v + ks * (2048 >> 4), idesc_o, (k > 0 || ks > 0) ? 1u : 0u);
                        tc_commit(&pv_done[x]);
                        if (b == 1 || k + 1 == steps) tc_commit(&freed[1][t & 1]);
                        if (k + 1 == steps) tc_commit(&o_done[x]);
                    }
                    __syncwarp();
                    if (k + 2 < steps) scores(k + 2);
                }
                used ^= ((steps + 1) / 2 & 1) | (steps / 2 & 1) << 1;
                ++segs;
            }
            loads += len;
            share_done(i);
        }
        if (*abort_flag) {  // leaving early: the products in flight end before the block's memory is handed on (one commit more to the output's barrier)
            if (tc_elect_one()) tc_commit(&o_done[x]);
            __syncwarp();
            for (uint32_t it = 0; it < 4096 && !tc_mbar_try(&o_done[x], segs & 1); ++it) {}
        }
    } else if (warp < SOFTMAX_WARPS) {  // ---- softmax: a thread per row ----
        constexpr float LOG2E = 1.4426950408889634f, SLACK = 5.545177444f;  // 8 ln 2
        const uint32_t x = warp >> 2, wrow = (warp & 3) * 32, row = wrow + lane;
        const uint32_t ts = tmem + 128 * x + (wrow << 16), to = tmem + 256 + 128 * x + (wrow << 16);
        uint32_t used = 0, all_steps = 0, segs = 0, tiles0 = 0;  // of the shares before: uses of either step's columns, steps and shares of this row tile; all key tiles
        uint32_t turns = 0;                                              // steps so far with the other row tile beside
        // The warp's 32 rows of a share's q: fetched, and when `before` has waited for the last scores of the share before, scaled, rounded to f16 and stored
        // swizzled K-major over that one's (rows past the last are zeros).
        auto bring_q = [&](const PackedShare &it, auto before) -> bool {
            const uint32_t rows = it.rows;
            const float *q0 = p.q + ((size_t)it.t0 * p.hq + it.kh * G) * D;
            uint8_t *to_q = smem + x * TILE_BYTES;
            bool fine = true;
#pragma unroll
            for (uint32_t e0 = 0; e0 < 32; e0 += 16) {
                float4 f[16];
#pragma unroll
                for (uint32_t e = 0; e < 16; ++e) {
                    const uint32_t r = 128 * x + wrow + e0 + e, token = row_token(p.l, r);
                    f[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (r < rows) f[e] = reinterpret_cast<const float4 *>(q0 + (token * p.hq + r - token * G) * D)[lane];
                }
                if (e0 == 0) fine = before();
#pragma unroll
                for (uint32_t e = 0; e < 16; ++e) {
                    const __half2 a = __floats2half2_rn(f[e].x * p.scale, f[e].y * p.scale), b = __floats2half2_rn(f[e].z * p.scale, f[e].w * p.scale);
                    *reinterpret_cast<uint2 *>(to_q + tile_piece(wrow + e0 + e, 8 * (lane >> 1)) + 8 * (lane & 1)) =
                        make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) tc_mbar_arrive(&q_full[x]);
            return fine;
        };
        auto nothing = [] { return true; };
        bool ok = share_at(0);
        if (ok && shares[0].rows > 128 * x) ok = bring_q(shares[0], nothing);
#pragma unroll 1
        for (uint32_t i = 0; ok; ++i) {
            const PackedShare &share = shares[i % SHARES], &next = shares[(i + 1) % SHARES];
            const uint32_t rows = share.rows, steps = share.steps, j0 = share.j0;
            if (rows == 0) break;
            const uint32_t seen_all = 128 * x + row < rows ? share.past + row_token(p.l, 128 * x + row) + 1 : 0;
            const uint32_t nfree = (share.past + row_token(p.l, 128 * x) + 1) / 64;  // steps [0, nfree) of all keys lie wholly at or below every row's own position
            float m = -INFINITY, mneg = 0.0f, l[2] = {0.0f, 0.0f};
            if (rows <= 128 * x) {
                ok = share_at(i + 1);
                if (ok && next.rows > 128 * x) ok = bring_q(next, nothing);
            } else {
#pragma unroll 1
                for (uint32_t k = 0; k < steps; ++k) {
                    const uint32_t b = k & 1, at = 2 * j0 + k;
                    auto scores = [&] { return all_wait(&s_ready[x][b], ((used >> b & 1) + (k >> 1)) & 1); };  // S of this step, and with it every product issued before
                    if (k + 1 < steps) ok = scores();
                    else {  // (the next share's queries on the way)
                        ok = share_at(i + 1);
                        if (ok && next.rows > 128 * x) ok = bring_q(next, scores);
                        else ok = scores() && ok;
                    }
                    if (!ok) break;  // (what was read of S would count for nothing)
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    uint32_t v[2][32];
                    tmem_ld32(ts + 64 * b, v[0]);
                    tmem_ld32(ts + 64 * b + 32, v[1]);
                    const uint32_t there = there_s[(tiles0 + (k >> 1)) & 7] >> (4 * b) & 15;  // of the step's four pages, those that are pages
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (at >= nfree || there != 15) {
                        const int seen = (int)min(64u, seen_all - min(seen_all, at * 64));  // of the step's keys, those the row sees
#pragma unroll
                        for (int e = 0; e < 64; ++e)
                            if (e >= seen || !(there >> (e >> 4) & 1)) v[e >> 5][e & 31] = 0xff800000u;  // -inf: exp2 gives 0
                    }
                    float t[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) t[e] = fmaxf(__uint_as_float(v[0][2 * e]), __uint_as_float(v[0][2 * e + 1]));
#pragma unroll
                    for (int e = 8; e < 64; e += 2) t[(e >> 1) & 3] = max3(t[(e >> 1) & 3], __uint_as_float(v[e >> 5][e & 31]), __uint_as_float(v[e >> 5][(e & 31) + 1]));
                    const float tmax = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
                    float rescale = 1.0f;
                    bool move = false;
                    if (tmax > m + SLACK || (m == -INFINITY && tmax != -INFINITY)) {
                        move = m != -INFINITY;
                        rescale = move ? exp2_approx((m - tmax) * LOG2E) : 1.0f;
#pragma unroll
                        for (int e = 0; e < 2; ++e) l[e] *= rescale;
                        m = tmax;
                        mneg = fmaf(-m, LOG2E, WEIGHT_LOG2);
                    }
                    if (__any_sync(0xffffffffu, move)) {  // what O holds for the row was accumulated against the old reference; the last product must have ended
                        ok = all_wait(&pv_done[x], (all_steps + k - 1) & 1);
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
                        for (uint32_t c = 0; c < 128; c += 8) {
                            uint32_t o[8];
                            tmem_ld8(to + c, o);
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                            for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * rescale);
                            tmem_st8(to + c, o);
                        }
                    }
                    // The row tiles take turns with the exponentials, A first: side by side, both would hold the exponential unit up and then leave it idle.
                    if (rows > 128) {
                        if (x == 1 || turns > 0) ok = all_wait(&turn[x], (turns - (x ^ 1)) & 1);
                        ++turns;
                    }
#pragma unroll
                    for (int c = 0; c < 4; ++c) {  // 16 keys: 8 columns of P (all of the row's scores are in registers by now)
                        if (c == 3 && rows > 128 && lane == 0) tc_mbar_arrive(&turn[x ^ 1]);
                        float y[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) y[e] = exp2_approx(fmaf(__uint_as_float(v[c >> 1][(c & 1) * 16 + e]), LOG2E, mneg));
                        uint32_t w[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const __half2 pp = __floats2half2_rn(y[2 * e], y[2 * e + 1]);
                            w[e] = *reinterpret_cast<const uint32_t *>(&pp);
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e) add_halves(w[e], l[0], l[1]);
                        tmem_st8(ts + 64 * b + 8 * c, w);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) tc_mbar_arrive(&p_ready[x][b]);
                }
                used ^= ((steps + 1) / 2 & 1) | (steps / 2 & 1) << 1;
                all_steps += steps;
                // ---- output: O / l, rounded to f16, whole rows by way of shared memory; a part of the item's keys: O, m and l as they are ----
                ok = ok && all_wait(&o_done[x], segs & 1);
                ++segs;
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const float sum = l[0] + l[1];
                const uint32_t r = 128 * x + row;
                const bool live = r < rows;
                float zeros = 0.0f;  // 0 times every output: NaN when one is not finite
                if (!share.whole) {
                    float *dst = p.part + (size_t)(2 * blockIdx.x + (j0 == 0)) * packed_part_floats(ROWS);
                    if (live) {
                        dst[ROWS * D + r] = fmaf(m, LOG2E, -WEIGHT_LOG2);
                        dst[ROWS * D + ROWS + r] = sum;
                    }
#pragma unroll 1
                    for (uint32_t c = 0; c < 4; ++c) {
                        uint32_t o[32];
                        tmem_ld32(to + 32 * c, o);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int e = 0; e < 32; ++e) zeros = fmaf(__uint_as_float(o[e]), 0.0f, zeros);
#pragma unroll
                        for (int g = 0; g < 8; ++g)
                            if (live) reinterpret_cast<uint4 *>(dst + (size_t)r * D)[8 * c + g] = make_uint4(o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]);
                    }
                } else {
                    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                    uint8_t *stage = ring + 4 * TILE_BYTES + warp * 2048;  // 32 rows of 32 dims; a piece of 16 bytes goes where no two meet in a bank
#pragma unroll 1
                    for (uint32_t c = 0; c < 4; ++c) {
                        uint32_t o[32], packed[16];
                        tmem_ld32(to + 32 * c, o);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int e = 0; e < 32; ++e) zeros = fmaf(__uint_as_float(o[e]), 0.0f, zeros);
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const __half2 hh = __floats2half2_rn(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
                            packed[e >> 1] = *reinterpret_cast<const uint32_t *>(&hh);
                        }
#pragma unroll
                        for (uint32_t g = 0; g < 4; ++g)
                            *reinterpret_cast<uint4 *>(stage + 64 * lane + 16 * (g ^ (lane >> 1 & 3))) = make_uint4(packed[4 * g], packed[4 * g + 1], packed[4 * g + 2], packed[4 * g + 3]);
                        __syncwarp();
#pragma unroll
                        for (uint32_t g = 0; g < 4; ++g) {  // eight rows at a time, 64 bytes of each
                            const uint32_t e = 8 * g + (lane >> 2), re = 128 * x + wrow + e, tk = row_token(p.l, re);
                            const uint4 w = *reinterpret_cast<const uint4 *>(stage + 64 * e + 16 * ((lane & 3) ^ (e >> 1 & 3)));
                            if (re < rows) reinterpret_cast<uint4 *>(p.o + ((size_t)(share.t0 + tk) * p.hq + share.kh * G + re - tk * G) * D + 32 * c)[lane & 3] = w;
                        }
                        __syncwarp();
                    }
                }
                const uint32_t upto = min(share.nkeys, 128 * (j0 + share.len));
                if (live && zeros != 0.0f && seen_all < upto) again_s = 1;  // (looked after when all shares are done)
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            }
            tiles0 += share.len;
            share_done(i);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t ncols = 512;
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(ncols) : "memory");
    }
    if (!again_s || abort_s) return;
    packed_tc_again<Q8>(p, begin, pieces.at[1]);
}

}  // namespace

int32_t brasa_packed_tc_launch(brasa_cmd *cmd, const PackedView &v, int32_t kv, const float *q, const uint8_t *kpool, const uint8_t *vpool, void *o, float *part, PackedNote *notes,
                               uint32_t hq, float scale) {
    brasa_ctx *ctx = cmd->ctx;
    const bool q8 = kv == BRASA_KV_Q8_0;
    PackedMaps maps;
    memset(&maps, 0, sizeof maps);
    if (!q8) {
        const uint64_t dims[3] = {D, v.hkv, (uint64_t)v.num_pages * PAGE}, strides[2] = {256, (uint64_t)v.hkv * 256};
        const uint32_t box[3] = {64, 1, PAGE};
        BRASA_TRY(brasa_tmap_bf16(ctx, &maps.k, 3, kpool, dims, strides, box));  // (16-bit values are copied whatever they are)
        BRASA_TRY(brasa_tmap_bf16(ctx, &maps.v, 3, vpool, dims, strides, box));
    }
    const PackedTcParams p{packed_line(v, hq / v.hkv, ROWS, 7, 2, 2, 4, PACKED_TC_MIN_ROWS, UINT32_MAX), q, kpool, vpool, (__half *)o, part, notes, hq, scale, ctx->status};
    const size_t smem = (2 + 4) * TILE_BYTES + SOFTMAX_WARPS * 2048;
    void (*const kernel)(PackedMaps, PackedTcParams) = q8 ? attn_packed_tc_kernel<true> : attn_packed_tc_kernel<false>;
    BRASA_TRY(brasa_smem_optin(ctx, (const void *)kernel, smem));
    BRASA_CUDA(ctx, brasa_launch_dependent(ctx, kernel, dim3(ctx->sm_count), dim3(q8 ? THREADS_Q8 : THREADS), smem, maps, p));
    return brasa_post_launch(cmd, "attn_packed_tc");
}
