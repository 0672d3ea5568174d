// Verification of drafted tokens against the target model's probabilities. With p the target's and q the draft's distribution, a draft x
// drawn from q is accepted with probability min(1, p(x) / q(x)); at the first refusal a token is drawn from max(p - q, 0), normalised, and
// behind the last accepted draft one from p. Whatever q is, the tokens are then distributed as p alone would have drawn them.
//
// One row of p (and of q) per sequence is all that has to be read: 2 x 0.6 MB for a vocabulary of 151 936, so a cluster of eight blocks
// takes a sequence, each with an eighth of the ids. Masses and their sums are 64-bit: p - q of two f32 numbers is exact up to the last
// bits, and where the running sum passes the drawn point is decided far below the smallest mass. The sums' order depends on the vocabulary alone.
// 64 sequences of 151 936 ids with q 23.5 us among calls that leave the 78 MB in the L2, 32 us behind a flush (2.5 TB/s): two passes of a cluster whose second waits for the first;
// one sequence without q 9 us and 18 us, latency.
#include "brasa_internal.h"

namespace {

constexpr uint32_t CLUSTER = 8, PIECES = 16, UNIT = 128;  // blocks of a sequence, pieces of a block's ids, ids that a warp takes at a time (four a lane)

struct VerifyParams {
    const float *p, *q, *u;
    const uint32_t *drafts, *starts;
    uint32_t *tokens, *accepted;
    uint32_t seqs, rows, vocab;
    uint64_t ndrafts;  // entries of drafts (and rows of q) that there are
};

// the same shared variable of block `rank` of the cluster
__device__ __forceinline__ double cluster_double(const double *local, uint32_t rank) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(remote) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t cluster_word(const uint32_t *local, uint32_t rank) {
    uint32_t remote, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
    return v;
}
// an entry of p or q; what is no positive finite number counts as 0
__device__ __forceinline__ float probability(float x) { return __float_as_uint(x) < 0x7F800000u ? x : 0.0f; }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <uint32_t THREADS>
__global__ void __cluster_dims__(CLUSTER, 1, 1) __launch_bounds__(THREADS, 1024 / THREADS) verify_drafts_kernel(VerifyParams a) {
    constexpr uint32_t WARPS = THREADS / 32;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // (launched as a programmatic dependent: see brasa_launch_dependent)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ double block_sum[2], piece_sum[PIECES], piece_start[PIECES + 1];
    __shared__ uint32_t stop_s, token_s, last_s;
    const uint32_t s = blockIdx.x / CLUSTER, me = blockIdx.x % CLUSTER, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t first = min(a.starts[s], a.rows), end = max(first, min(a.starts[s + 1], a.rows));
    // ---- drafts lie without the sequences' last rows: as many fewer as sequences before this one have rows ----
    uint32_t before = 0;
    for (uint32_t i = tid; i - tid < s; i += THREADS) before += __syncthreads_count(i < s && min(a.starts[i + 1], a.rows) > min(a.starts[i], a.rows));
    if (end == first) {  // (the same for the whole cluster)
        if (me == 0 && tid == 0) a.accepted[s] = 0;
        return;
    }
    const uint32_t n = end - first - 1;  // drafts
    const size_t draft0 = (size_t)first - min(before, first);
    if (tid == 0) {
        stop_s = n;
        last_s = 0;
        token_s = UINT32_MAX;
    }
    __syncthreads();
    for (uint32_t i = tid; i < n; i += THREADS) {
        bool take = false;
        const uint32_t x = draft0 + i < a.ndrafts ? a.drafts[draft0 + i] : UINT32_MAX;
        if (x < a.vocab) {
            const double px = probability(a.p[(size_t)(first + i) * a.vocab + x]), qx = a.q ? probability(a.q[(draft0 + i) * a.vocab + x]) : 1.0f;
            take = (double)a.u[first + i] * qx < px;
        }
        if (!take) atomicMin(&stop_s, i);
    }
    __syncthreads();
    const uint32_t stop = stop_s;
    const bool drafted = stop < n && draft0 + stop < a.ndrafts;
    const float *p = a.p + (size_t)(first + stop) * a.vocab, *q = drafted && a.q ? a.q + (draft0 + stop) * a.vocab : nullptr;
    uint32_t gone = drafted && !a.q ? a.drafts[draft0 + stop] : UINT32_MAX;  // (a given draft: its own probability was 1)
    // ---- masses of this block's ids, piece by piece; the second time round nothing is subtracted, when nothing was left. Whatever the number of warps,
    // a piece is the same ids, and a lane adds up the same of them in the same order ----
    const uint32_t units = (a.vocab + UNIT - 1) / UNIT;
    auto piece_at = [&](uint32_t n) { return min((uint32_t)((uint64_t)units * (me * PIECES + n) / (CLUSTER * PIECES)) * UNIT, a.vocab); };
    const bool vec = (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (!q || (reinterpret_cast<uintptr_t>(q) & 15) == 0);
    auto load4 = [&](const float *row, uint32_t i) {
        if (vec && i + 4 <= a.vocab) return *reinterpret_cast<const float4 *>(row + i);
        return make_float4(i < a.vocab ? row[i] : 0.0f, i + 1 < a.vocab ? row[i + 1] : 0.0f, i + 2 < a.vocab ? row[i + 2] : 0.0f, i + 3 < a.vocab ? row[i + 3] : 0.0f);
    };
    auto masses = [&](uint32_t i, const float4 &x4, const float4 &y4, double m[4], uint32_t &held) {  // held: the last of the ids that has any
        float x[4] = {x4.x, x4.y, x4.z, x4.w}, y[4] = {y4.x, y4.y, y4.z, y4.w};
        auto most = [](const float z[4]) { return max(max(__float_as_uint(z[0]), __float_as_uint(z[1])), max(__float_as_uint(z[2]), __float_as_uint(z[3]))); };
        if (max(most(x), most(y)) >= 0x7F800000u || gone - i < 4)  // (rare: looked at together)
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                x[k] = gone - i != k ? probability(x[k]) : 0.0f;
                y[k] = probability(y[k]);
            }
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            x[k] = fmaxf(x[k], y[k]);
            m[k] = (double)x[k] - (double)y[k];
            if (x[k] > y[k]) held = i + k;
        }
    };
    const float4 none = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    double total = 0.0, start = 0.0;
    uint32_t last = 0;  // the last of this thread's ids that has mass
    int round = 0;
    for (;; ++round) {
        for (uint32_t n = warp; n < PIECES; n += WARPS) {
            const uint32_t end_id = piece_at(n + 1);
            double sum = 0.0;
#pragma unroll 4
            for (uint32_t i = piece_at(n) + 4 * lane; i < end_id; i += UNIT) {
                double m[4];
                masses(i, load4(p, i), q ? load4(q, i) : none, m, last);
                sum += (m[0] + m[1]) + (m[2] + m[3]);
            }
            for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
            if (lane == 0) piece_sum[n] = sum;
        }
        __syncthreads();
        if (warp == 0) {
            double v = lane < PIECES ? piece_sum[lane] : 0.0;
            for (uint32_t x = 1; x < PIECES; x <<= 1) {
                const double o = __shfl_up_sync(0xffffffffu, v, x);
                if (lane >= x) v += o;
            }
            if (lane < PIECES) piece_start[lane + 1] = v;
            if (lane == 0) piece_start[0] = 0.0;
            if (lane == PIECES - 1) block_sum[round] = v;
        }
        cluster_sync();
        double sums[CLUSTER];
#pragma unroll
        for (uint32_t r = 0; r < CLUSTER; ++r) sums[r] = cluster_double(&block_sum[round], r);
        total = start = 0.0;
#pragma unroll
        for (uint32_t r = 0; r < CLUSTER; ++r) {
            if (r < me) start += sums[r];
            total += sums[r];
        }
        if (total > 0.0 || round == 1) break;
        q = nullptr;
        gone = UINT32_MAX;
    }
    // ---- the first id at which the running sum exceeds the point. A piece of [0, total) ends where the next one begins, in the very same sums, so one
    // holds the point; two can only where rounding moved an end by a bit, and then the lower id counts ----
    const double point = (double)a.u[end - 1] * total, block_start = start, block_end = start + block_sum[round];
    for (uint32_t n = warp; n < PIECES; n += WARPS) {
        const uint32_t end_id = piece_at(n + 1);
        start = block_start + piece_start[n];
        const double piece_end = n + 1 < PIECES ? block_start + piece_start[n + 1] : block_end;
        if (!(start <= point && point < piece_end)) continue;
        uint32_t id = UINT32_MAX, held = 0;
        float4 x = load4(p, piece_at(n) + 4 * lane), y = q ? load4(q, piece_at(n) + 4 * lane) : none;
        for (uint32_t i0 = piece_at(n); i0 < end_id && id == UINT32_MAX; i0 += UNIT) {
            const uint32_t i = i0 + 4 * lane;
            double m[4];
            masses(i, x, y, m, held);
            x = load4(p, i + UNIT);
            y = q ? load4(q, i + UNIT) : none;
            const double sum = (m[0] + m[1]) + (m[2] + m[3]);
            double upto = sum;
            for (uint32_t z = 1; z < 32; z <<= 1) {
                const double v = __shfl_up_sync(0xffffffffu, upto, z);
                if (lane >= z) upto += v;
            }
            uint32_t mine = UINT32_MAX;
            double run = start + (upto - sum);
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                run += m[k];
                if (mine == UINT32_MAX && m[k] > 0.0 && run > point) mine = i + k;
            }
            id = __reduce_min_sync(0xffffffffu, mine);
            start += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (id == UINT32_MAX) id = __reduce_max_sync(0xffffffffu, held);  // (rounding: the piece's last mass)
        if (lane == 0) atomicMin(&token_s, id);
    }
    last = __reduce_max_sync(0xffffffffu, last);
    if (lane == 0) atomicMax(&last_s, last);
    cluster_sync();
    if (me == 0 && warp == 0) {
        uint32_t token = UINT32_MAX, final = 0;
        for (uint32_t r = 0; r < CLUSTER; ++r) {
            token = min(token, cluster_word(&token_s, r));
            final = max(final, cluster_word(&last_s, r));
        }
        if (token == UINT32_MAX) token = final;  // (a point behind every sum: the last id that has mass; none has: 0)
        if (lane == 0) {
            a.accepted[s] = stop;
            a.tokens[first + stop] = token;
        }
        for (uint32_t i = lane; i <= n; i += 32)
            if (i != stop) a.tokens[first + i] = i < stop ? a.drafts[draft0 + i] : 0u;
    }
    cluster_sync();  // (no block leaves while another reads its words)
}

}  // namespace

extern "C" int32_t brasa_k_verify_drafts(brasa_cmd *cmd, brasa_arg p, brasa_arg q, brasa_arg drafts, brasa_arg u, brasa_arg starts, uint32_t seqs, uint32_t rows,
                                         uint32_t vocab, brasa_arg tokens, brasa_arg accepted) {
    if (!cmd) return BRASA_EINVAL;
    brasa_ctx *ctx = cmd->ctx;
    BRASA_REQUIRE(ctx, seqs >= 1 && rows >= 1 && vocab >= 1, "verify_drafts: no sequences, rows or vocabulary");
    BRASA_REQUIRE(ctx, seqs <= (1u << 31) / CLUSTER - 1 && vocab <= 1u << 31, "verify_drafts: more than 2^28 sequences or 2^31 ids");
    // at least so many drafts: a sequence without rows makes it more, which the kernel holds against what there is
    const uint64_t nd = rows > seqs ? rows - seqs : 0;
    BRASA_REQUIRE(ctx, arg_fits(p, (uint64_t)rows * vocab * 4) && arg_fits(u, (uint64_t)rows * 4) && arg_fits(starts, ((uint64_t)seqs + 1) * 4),
                  "verify_drafts: p, u or starts too small");
    BRASA_REQUIRE(ctx, arg_fits(drafts, nd * 4) && (!q.buf || arg_fits(q, nd * vocab * 4)), "verify_drafts: drafts or q too small");
    BRASA_REQUIRE(ctx, arg_fits(tokens, (uint64_t)rows * 4) && arg_fits(accepted, (uint64_t)seqs * 4), "verify_drafts: tokens or accepted too small");
    for (const brasa_arg *a : {&p, &q, &drafts, &u, &starts, &tokens, &accepted}) BRASA_REQUIRE(ctx, a->offset % 4 == 0, "verify_drafts: misaligned buffer");
    // sequences run side by side, and a sequence's tokens begin behind its drafts' places: nothing can be written in place
    const std::pair<const brasa_arg *, uint64_t> ins[] = {{&p, (uint64_t)rows * vocab * 4}, {&q, nd * vocab * 4}, {&drafts, nd * 4}, {&u, (uint64_t)rows * 4}, {&starts, ((uint64_t)seqs + 1) * 4}};
    for (const auto &i : ins)
        BRASA_REQUIRE(ctx, !arg_overlap(*i.first, i.second, tokens, (uint64_t)rows * 4) && !arg_overlap(*i.first, i.second, accepted, (uint64_t)seqs * 4),
                      "verify_drafts: tokens and accepted must not overlap what is read");
    BRASA_REQUIRE(ctx, !arg_overlap(tokens, (uint64_t)rows * 4, accepted, (uint64_t)seqs * 4), "verify_drafts: tokens and accepted must not overlap");
    VerifyParams a{(const float *)arg_ptr(p), (const float *)arg_ptr(q), (const float *)arg_ptr(u), (const uint32_t *)arg_ptr(drafts), (const uint32_t *)arg_ptr(starts),
                   (uint32_t *)arg_ptr(tokens), (uint32_t *)arg_ptr(accepted), seqs, rows, vocab, drafts.buf ? (drafts.buf->bytes - drafts.offset) / 4 : 0};
    if (q.buf) a.ndrafts = std::min(a.ndrafts, (q.buf->bytes - q.offset) / 4 / vocab);
    // 16 warps a block while all blocks are resident at once (clusters of eight fill 128 of the SMs, two blocks to each), eight warps where there are more sequences. 151 936 ids
    // with q, 16 | 8 warps: 1 sequence 18.4 | 23.6 us, 32 sequences 22.6 | 28.7, 34 sequences 32.8 | 28.7, 64 sequences 38.9 | 31.7 (each behind a flush of the L2).
    const bool wide = seqs <= 32;
    BRASA_CUDA(ctx, brasa_launch_dependent(ctx, wide ? verify_drafts_kernel<512> : verify_drafts_kernel<256>, dim3(seqs * CLUSTER), dim3(wide ? 512 : 256), 0, a));
    return brasa_post_launch(cmd, "verify_drafts");
}
