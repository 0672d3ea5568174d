// Norm, RoPE and store, and attention, of a packed run: any number of new tokens per sequence over the paged pool.
#include <math.h>

#include "packed.cuh"

using namespace brasa_dev;

namespace {

constexpr uint32_t PAGE = BRASA_KV_PAGE;
constexpr int D = 128, TS = D + 4;

// One warp per row of q, k or v of one token: y = x / sqrt(mean x^2 + eps) * w, rotated by the token's own position.
template <int KV>
__global__ void __launch_bounds__(128) qk_norm_rope_store_packed_kernel(const float *q, const float *k, const float *v, const float *q_norm, const float *k_norm,
                                                                        const float *cos_t, const float *sin_t, uint8_t *kpool, uint8_t *vpool, PackedView p,
                                                                        float *q_out, uint32_t hq, float eps, uint64_t rows) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // (launched as a programmatic dependent: see brasa_launch_dependent)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    __shared__ __align__(16) uint8_t scratch[4][528];
    const uint64_t gr = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, hkv = p.hkv, per_tok = hq + 2 * hkv;
    if (gr >= rows) return;
    const uint32_t t = (uint32_t)(gr / per_tok), r = (uint32_t)(gr % per_tok);
    uint32_t seq, pos;
    if (!packed_row(p, t, lane, seq, pos) || pos / PAGE >= p.max_pages) return;
    const int32_t page = packed_page(p, seq, pos);
    const size_t slot = (size_t)max(page, 0) * PAGE + pos % PAGE;
    float y[4];
    if (r >= hq + hkv) {
        if (page < 0) return;
        const uint32_t kh = r - hq - hkv;
        for (int j = 0; j < 4; ++j) y[j] = v[((size_t)t * hkv + kh) * D + lane + 32 * j];
        put_row<KV>(vpool + (slot * hkv + kh) * KvRow<KV>::BYTES, scratch[warp], y, lane);
        return;
    }
    if (r < hq) {
        norm_rope_row(q + ((size_t)t * hq + r) * D, q_norm, cos_t, sin_t, pos, eps, lane, y);
        for (int j = 0; j < 4; ++j) q_out[((size_t)t * hq + r) * D + lane + 32 * j] = y[j];
    } else if (page >= 0) {
        norm_rope_row(k + ((size_t)t * hkv + r - hq) * D, k_norm, cos_t, sin_t, pos, eps, lane, y);
        put_row<KV>(kpool + (slot * hkv + r - hq) * KvRow<KV>::BYTES, scratch[warp], y, lane);
    }
}

// One block per token and key head: the group's rows against 64 keys at a time, K and V as f32 in shared memory, a running maximum, sum
// and output per row.
template <int KV, bool HALF_OUT>
__global__ void __launch_bounds__(128) attn_packed_rows_kernel(const float *q, const uint8_t *kpool, const uint8_t *vpool, PackedView p, void *o, uint32_t hq,
                                                               float scale) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr uint32_t KEYS = 64;
    __shared__ __align__(16) float ts[KEYS * TS], qs[8 * D], ps[8 * KEYS];
    __shared__ float ms[8], ls[8], alpha[8];
    const uint32_t t = blockIdx.x, kh = blockIdx.y, hkv = p.hkv, G = hq / hkv, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t seq, pos;
    if (!packed_row(p, t, lane, seq, pos) || pos / PAGE >= p.max_pages) return;
    const uint32_t nkeys = pos + 1;
    for (uint32_t i = tid; i < G * D; i += 128) qs[i] = q[((size_t)t * hq + kh * G) * D + i];
    if (tid < 8) {
        ms[tid] = -INFINITY;
        ls[tid] = 0.0f;
    }
    float acc[8];
    for (int g = 0; g < 8; ++g) acc[g] = 0.0f;
    auto load = [&](const uint8_t *pool, uint32_t key0) {
        for (uint32_t i = tid; i < KEYS * (D / 8); i += 128) {
            const uint32_t key = key0 + i / (D / 8), v8 = i % (D / 8);
            const int32_t page = key < nkeys ? packed_page(p, seq, key) : -1;
            float v[8] = {};
            if (page >= 0) tile_load8<KV>(pool + (((size_t)page * PAGE + key % PAGE) * hkv + kh) * KvRow<KV>::BYTES, (int)(v8 * 8), v);
            for (int j = 0; j < 8; ++j) ts[(i / (D / 8)) * TS + v8 * 8 + j] = v[j];
        }
    };
    for (uint32_t key0 = 0; key0 < nkeys; key0 += KEYS) {
        load(kpool, key0);
        __syncthreads();
        const uint32_t key = key0 + (tid & 63);
        const bool there = key < nkeys && packed_page(p, seq, key) >= 0;
        for (uint32_t g = tid >> 6; g < G; g += 2) {
            float a = 0.0f;
            for (int d = 0; d < D; ++d) a = fmaf(qs[g * D + d], ts[(tid & 63) * TS + d], a);
            ps[g * KEYS + (tid & 63)] = there ? a * scale : -INFINITY;
        }
        __syncthreads();
        load(vpool, key0);
        for (uint32_t g = warp; g < G; g += 4) {
            const float s0 = ps[g * KEYS + lane], s1 = ps[g * KEYS + 32 + lane];
            float m = fmaxf(s0, s1);
            for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
            const float before = ms[g], now = fmaxf(before, m);
            const float p0 = s0 == -INFINITY ? 0.0f : expf(s0 - now), p1 = s1 == -INFINITY ? 0.0f : expf(s1 - now);
            float l = p0 + p1;
            for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
            ps[g * KEYS + lane] = p0;
            ps[g * KEYS + 32 + lane] = p1;
            __syncwarp();
            if (lane == 0) {
                const float a = before == -INFINITY ? 0.0f : expf(before - now);
                alpha[g] = a;
                ls[g] = ls[g] * a + l;
                ms[g] = now;
            }
        }
        __syncthreads();
        for (uint32_t g = 0; g < G; ++g) {
            float a = acc[g] * alpha[g];
            for (uint32_t j = 0; j < KEYS; ++j) a = fmaf(ps[g * KEYS + j], ts[j * TS + tid], a);
            acc[g] = a;
        }
        __syncthreads();
    }
    for (uint32_t g = 0; g < G; ++g) {
        const float r = ls[g] == 0.0f ? 0.0f : acc[g] / ls[g];
        const size_t at = ((size_t)t * hq + kh * G + g) * D + tid;
        if (HALF_OUT) static_cast<__half *>(o)[at] = __float2half_rn(r);
        else static_cast<float *>(o)[at] = r;
    }
}

// What both operators ask of a run beside its pool; the run's view for the kernels.
int32_t packed_view(brasa_ctx *ctx, const char *who, const brasa_paged_kv &pg, const brasa_packed_run &run, uint32_t hq, uint32_t hkv, PackedView *out) {
    BRASA_TRY(brasa_check_paged(ctx, pg, hq, hkv));
    BRASA_REQUIRE(ctx, hq > 0, "%s: no heads", who);
    BRASA_REQUIRE(ctx, run.tokens >= 1 && run.longest >= 1, "%s: empty run", who);
    BRASA_REQUIRE(ctx, run.starts.offset % 4 == 0 && arg_fits(run.starts, ((uint64_t)pg.seqs + 1) * 4), "%s: starts too small or misaligned", who);
    *out = PackedView{(const int32_t *)arg_ptr(pg.table), (const uint32_t *)arg_ptr(pg.lens), (const uint32_t *)arg_ptr(run.starts), pg.seqs, pg.max_pages,
                      pg.num_pages, run.tokens, run.longest, hkv};
    return BRASA_OK;
}

}  // namespace

extern "C" {

int32_t brasa_k_qk_norm_rope_store_packed(brasa_cmd *cmd, brasa_arg q, brasa_arg k, brasa_arg v, brasa_arg q_norm, brasa_arg k_norm, brasa_arg rope_cos,
                                          brasa_arg rope_sin, float eps, brasa_paged_kv pg, brasa_packed_run run, brasa_arg q_out, uint32_t hq, uint32_t hkv) {
    if (!cmd) return BRASA_EINVAL;
    brasa_ctx *ctx = cmd->ctx;
    PackedView p;
    BRASA_TRY(packed_view(ctx, "qk_norm_rope_store_packed", pg, run, hq, hkv, &p));
    const uint64_t nq = (uint64_t)run.tokens * hq * 512, nkv = (uint64_t)run.tokens * hkv * 512;
    BRASA_REQUIRE(ctx, arg_fits(q, nq) && arg_fits(q_out, nq) && arg_fits(k, nkv) && arg_fits(v, nkv), "qk_norm_rope_store_packed: q, k, v or q_out too small");
    BRASA_REQUIRE(ctx, arg_fits(q_norm, 512) && arg_fits(k_norm, 512), "qk_norm_rope_store_packed: norm weights too small");
    const uint64_t table_bytes = (uint64_t)pg.max_pages * PAGE * 64 * 4;
    BRASA_REQUIRE(ctx, arg_fits(rope_cos, table_bytes) && arg_fits(rope_sin, table_bytes), "qk_norm_rope_store_packed: RoPE tables shorter than max_pages pages");
    for (const brasa_arg *a : {&q, &k, &v, &q_norm, &k_norm, &rope_cos, &rope_sin, &q_out})
        BRASA_REQUIRE(ctx, a->offset % 16 == 0, "qk_norm_rope_store_packed: misaligned buffer");
    const uint64_t rows = (uint64_t)run.tokens * (hq + 2 * hkv);
    BRASA_REQUIRE(ctx, rows <= 1ull << 32, "qk_norm_rope_store_packed: more than 2^32 rows");
    const dim3 grid((uint32_t)((rows + 3) / 4));
#define STORE_PACKED(KVT)                                                                                                                                       \
    BRASA_CUDA(ctx, brasa_launch_dependent(ctx, qk_norm_rope_store_packed_kernel<KVT>, grid, dim3(128), 0, (const float *)arg_ptr(q), (const float *)arg_ptr(k), \
                                           (const float *)arg_ptr(v), (const float *)arg_ptr(q_norm), (const float *)arg_ptr(k_norm),                           \
                                           (const float *)arg_ptr(rope_cos), (const float *)arg_ptr(rope_sin), arg_ptr(pg.kpool), arg_ptr(pg.vpool), p,          \
                                           (float *)arg_ptr(q_out), hq, eps, rows))
    if (pg.kv == BRASA_KV_F32) STORE_PACKED(BRASA_KV_F32);
    else if (pg.kv == BRASA_KV_F16) STORE_PACKED(BRASA_KV_F16);
    else STORE_PACKED(BRASA_KV_Q8_0);
#undef STORE_PACKED
    return brasa_post_launch(cmd, "qk_norm_rope_store_packed");
}

int32_t brasa_k_attention_packed(brasa_cmd *cmd, brasa_arg q, brasa_paged_kv pg, brasa_packed_run run, brasa_arg o, uint32_t hq, uint32_t hkv, int32_t precision) {
    if (!cmd) return BRASA_EINVAL;
    brasa_ctx *ctx = cmd->ctx;
    PackedView p;
    BRASA_TRY(packed_view(ctx, "attention_packed", pg, run, hq, hkv, &p));
    BRASA_REQUIRE(ctx, precision == BRASA_PREFILL_F16 || precision == BRASA_PREFILL_F32, "attention_packed: unknown precision %d", precision);
    const bool half = precision == BRASA_PREFILL_F16;
    const uint64_t n = (uint64_t)run.tokens * hq * D;
    BRASA_REQUIRE(ctx, arg_fits(q, n * 4) && arg_fits(o, n * (half ? 2 : 4)), "attention_packed: q or o too small");
    BRASA_REQUIRE(ctx, q.offset % 16 == 0 && o.offset % 16 == 0, "attention_packed: misaligned buffer");
    BRASA_REQUIRE(ctx, run.tokens < 1u << 31 && hkv <= 65535, "attention_packed: more than 2^31 tokens or 65 535 key heads");
    const float scale = 1.0f / sqrtf((float)D);
#define ATTN_PACKED(KVT)                                                                                                                                  \
    BRASA_CUDA(ctx, brasa_launch_dependent(ctx, half ? attn_packed_rows_kernel<KVT, true> : attn_packed_rows_kernel<KVT, false>, dim3(run.tokens, hkv), dim3(128), 0, \
                                           (const float *)arg_ptr(q), (const uint8_t *)arg_ptr(pg.kpool), (const uint8_t *)arg_ptr(pg.vpool), p, (void *)arg_ptr(o), hq, scale))
    if (pg.kv == BRASA_KV_F32) ATTN_PACKED(BRASA_KV_F32);
    else if (pg.kv == BRASA_KV_F16) ATTN_PACKED(BRASA_KV_F16);
    else ATTN_PACKED(BRASA_KV_Q8_0);
#undef ATTN_PACKED
    return brasa_post_launch(cmd, "attn_packed_rows");
}

}  // extern "C"
