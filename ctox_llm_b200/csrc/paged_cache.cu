// Bookkeeping and contents of a paged K/V cache that many requests share: pages and slots of new tokens, pages given back,
// and a layer's queries, keys and values between their projection and attention.
#include <cmath>

#include "paged.cuh"

namespace ctox {
namespace paged {
namespace {

constexpr uint32_t kPageThreads = 1024, kPageCtas = 8;

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Two running sums over the requests (new tokens, pages needed) say where everything goes. Every CTA of the one cluster forms
// both sums over all requests, 2 KB of lengths, instead of handing them on; once all have read their input (the barrier of
// the cluster: outputs may lie over inputs) each writes its share of the tokens. A token's page is the table's entry, or,
// if it is new, the stack's entry directly, so no CTA reads what another writes. Bound by latency: three dependent
// reads, two block scans and a barrier for a few hundred KB at most.
__global__ void __launch_bounds__(kPageThreads) k_page_slots(const __grid_constant__ ctox_page_slots_op op, int32_t *error_word) {
    __shared__ int32_t first_token[CTOX_MAX_BATCH + 1], first_page[CTOX_MAX_BATCH + 1];
    __shared__ int32_t len[CTOX_MAX_BATCH], row[CTOX_MAX_BATCH];
    __shared__ unsigned long long scan[32];
    const uint32_t tid = threadIdx.x, n = op.n_requests;
    pdl_launch();
    pdl_wait();
    uint32_t flags = 0;
    const int32_t count = *op.free_count_in;
    if (count < 0 || (uint32_t)count > op.n_pages) flags |= CTOX_PAGES_BAD_INPUT;
    // two neighbouring requests per thread
    uint32_t fresh[2] = {0, 0}, pages[2] = {0, 0};
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t r = 2 * tid + i;
        if (r >= n) continue;
        const int32_t a = op.kv_lens_in[r], b = op.new_tokens[r], at = op.rows ? op.rows[r] : (int32_t)r;
        len[r] = a;
        row[r] = at;
        if (a < 0 || b < 0 || at < 0 || (uint32_t)at >= op.table_rows) {
            flags |= CTOX_PAGES_BAD_INPUT;
            continue;
        }
        const uint64_t held = ((uint64_t)a + op.page_tokens - 1) / op.page_tokens;
        const uint64_t wanted = ((uint64_t)a + b + op.page_tokens - 1) / op.page_tokens;
        if (wanted > op.max_pages) flags |= CTOX_PAGES_ROW_FULL;
        fresh[i] = (uint32_t)b;
        pages[i] = (uint32_t)(wanted - held);
    }
    // lengths below 2^31 and at most 2048 of them: no sum passes 2^42
    const unsigned long long tokens_to = block_scan<unsigned long long>((unsigned long long)fresh[0] + fresh[1], scan);
    const unsigned long long pages_to = block_scan<unsigned long long>((unsigned long long)pages[0] + pages[1], scan);
    if (tid == blockDim.x - 1) {
        if (tokens_to > op.n_tokens) flags |= CTOX_PAGES_TOO_MANY;
        if (pages_to > (unsigned long long)max(count, 0)) flags |= CTOX_PAGES_NONE_FREE;
    }
    __shared__ uint32_t all_flags;
    if (tid == 0) all_flags = 0;
    __syncthreads();
    if (flags) atomicOr(&all_flags, flags);
    __syncthreads();
    flags = all_flags;
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {  // with no flag set every sum below fits
        const uint32_t r = 2 * tid + i;
        if (r >= n) continue;
        first_token[r] = flags ? 0 : (int32_t)(tokens_to - fresh[1] - (i ? 0 : fresh[0]));
        first_page[r] = flags ? 0 : (int32_t)(pages_to - pages[1] - (i ? 0 : pages[0]));
        if (r == n - 1) {
            first_token[n] = flags ? 0 : (int32_t)tokens_to - (i ? 0 : (int32_t)fresh[1]);
            first_page[n] = flags ? 0 : (int32_t)pages_to - (i ? 0 : (int32_t)pages[1]);
        }
    }
    __syncthreads();
    if (gridDim.x > 1) cluster_sync();
    const uint32_t me = blockIdx.x * blockDim.x + tid, all = gridDim.x * blockDim.x;
    const uint32_t total = (uint32_t)first_token[n], taken = (uint32_t)first_page[n];
    for (uint32_t i = me; i <= n; i += all) {
        op.query_offsets[i] = first_token[i];
        if (i < n) op.kv_lens_out[i] = len[i] + (flags ? 0 : first_token[i + 1] - first_token[i]);
    }
    if (me == 0) {
        *op.free_count_out = count - (int32_t)taken;
        op.status[0] = (int32_t)taken;
        op.status[1] = (int32_t)flags;
    }
    for (uint32_t i = me; i < taken; i += all) {
        const uint32_t r = last_at_most(first_page, n, (int32_t)i);
        const uint32_t held = ((uint32_t)len[r] + op.page_tokens - 1) / op.page_tokens;
        op.block_table[(uint64_t)row[r] * op.table_stride + held + (i - first_page[r])] = op.free_pages[count - 1 - (int32_t)i];
    }
    for (uint32_t t = me; t < op.n_tokens; t += all) {
        int32_t slot = -1, position = 0, request = -1;
        if (t < total) {
            const uint32_t r = last_at_most(first_token, n, (int32_t)t);
            const uint32_t place = (uint32_t)len[r] + (t - first_token[r]), at = place / op.page_tokens;
            const uint32_t held = ((uint32_t)len[r] + op.page_tokens - 1) / op.page_tokens;
            const int32_t page = at < held ? op.block_table[(uint64_t)row[r] * op.table_stride + at]
                                           : op.free_pages[count - 1 - (first_page[r] + (int32_t)(at - held))];
            if (page >= 0 && (uint32_t)page < op.n_pages)
                slot = page * (int32_t)op.page_tokens + (int32_t)(place % op.page_tokens);
            else
                bad_index(error_word);
            position = (int32_t)place;
            request = (int32_t)r;
        }
        op.slots[t] = slot;
        op.positions[t] = position;
        if (op.requests) op.requests[t] = request;
    }
}

// One CTA: requests end one at a time, and their pages are at most a few thousand words.
__global__ void __launch_bounds__(kPageThreads) k_page_release(const __grid_constant__ ctox_page_release_op op) {
    __shared__ int32_t first_page[CTOX_MAX_BATCH + 1], row[CTOX_MAX_BATCH];
    __shared__ unsigned long long scan[32];
    __shared__ uint32_t all_flags;
    const uint32_t tid = threadIdx.x, n = op.n_requests;
    pdl_launch();
    pdl_wait();
    uint32_t flags = 0, pages[2] = {0, 0};
    const int32_t count = *op.free_count_in;
    if (count < 0 || (uint32_t)count > op.n_pages) flags |= CTOX_PAGES_BAD_INPUT;
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t r = 2 * tid + i;
        if (r >= n) continue;
        const int32_t a = op.kv_lens[r], at = op.rows ? op.rows[r] : (int32_t)r;
        row[r] = at;
        if (a < 0 || at < 0 || (uint32_t)at >= op.table_rows) {
            flags |= CTOX_PAGES_BAD_INPUT;
            continue;
        }
        const uint64_t held = ((uint64_t)a + op.page_tokens - 1) / op.page_tokens;
        if (held > op.max_pages) flags |= CTOX_PAGES_ROW_FULL;
        pages[i] = (uint32_t)held;
    }
    const unsigned long long pages_to = block_scan<unsigned long long>((unsigned long long)pages[0] + pages[1], scan);
    if (tid == blockDim.x - 1 && pages_to + (unsigned long long)max(count, 0) > op.n_pages) flags |= CTOX_PAGES_TOO_MANY;
    if (tid == 0) all_flags = 0;
    __syncthreads();
    if (flags) atomicOr(&all_flags, flags);
    __syncthreads();
    flags = all_flags;
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t r = 2 * tid + i;
        if (r >= n) continue;
        first_page[r] = flags ? 0 : (int32_t)(pages_to - pages[1] - (i ? 0 : pages[0]));
        if (r == n - 1) first_page[n] = flags ? 0 : (int32_t)pages_to - (i ? 0 : (int32_t)pages[1]);
    }
    __syncthreads();
    const uint32_t given = (uint32_t)first_page[n];
    for (uint32_t i = tid; i < given; i += blockDim.x) {
        const uint32_t r = last_at_most(first_page, n, (int32_t)i);
        int32_t *entry = op.block_table + (uint64_t)row[r] * op.table_stride + (i - first_page[r]);
        op.free_pages[count + (int32_t)i] = *entry;
        *entry = -1;
    }
    if (tid == 0) {
        *op.free_count_out = count + (int32_t)given;
        op.status[0] = (int32_t)given;
        op.status[1] = (int32_t)flags;
    }
}

// ---- queries, keys and values of one layer ----

struct RopeArgs {
    ctox_rope_append_op op;
    double turns[128];  // of pair i per position: rope_base^(-2i / rot_dim) / 2 pi
};

__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float (&v)[8]) {
    const uint4 w = *reinterpret_cast<const uint4 *>(p);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void load8(const __half *p, float (&v)[8]) {
    const uint4 w = *reinterpret_cast<const uint4 *>(p);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }

// Eight dimensions from d0 on behind the norm, if there is one.
__device__ __forceinline__ void normed8(const float (&v)[8], const float *w, uint32_t d0, float inv, float offset, float (&r)[8]) {
    float f[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
    if (w) {
        load8(w + d0, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = inv * (offset + f[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = v[j] * f[j];
}

// One CTA per token (and share of its heads): the turn of every pair of dimensions once into shared memory, then
// D / 8 lanes per head with eight dimensions each, the norm's sum through shuffles.
template <typename S, typename T, int D>
__global__ void __launch_bounds__(256) k_rope_append(const __grid_constant__ RopeArgs a, int32_t *error_word) {
    constexpr uint32_t L = D / 8;  // lanes of a head
    __shared__ float2 turn[128];   // cosine and sine of each pair
    const ctox_rope_append_op &op = a.op;
    const uint32_t token = blockIdx.x, pairs = op.rot_dim / 2;
    pdl_launch();
    pdl_wait();
    for (uint32_t p = threadIdx.x; p < pairs; p += blockDim.x) {
        // whole turns leave in 64 bits: a far position times the fastest pair is thousands of turns
        const double t = (double)op.positions[op.axis[p] * op.position_stride + token] * a.turns[p];
        float sn, cs;
        sincospif((float)(2.0 * (t - rint(t))), &sn, &cs);
        turn[p] = make_float2(cs, sn);
    }
    const int32_t slot = op.k ? op.slots[token] : -1;
    const bool stored = slot >= 0 && (uint32_t)slot < op.kv.n_pages * op.kv.page_tokens;
    if (slot >= 0 && !stored && threadIdx.x == 0) bad_index(error_word);
    const uint64_t place = stored ? (uint64_t)(slot / op.kv.page_tokens) * op.kv.page_stride +
                                        (uint64_t)(slot % op.kv.page_tokens) * op.kv.token_stride
                                  : 0;
    __syncthreads();
    const uint32_t q_heads = op.q ? op.heads : 0, heads = q_heads + (stored ? 2 * op.kv_heads : 0);
    const uint32_t lane = threadIdx.x % L, d0 = lane * 8, rot = op.rot_dim, half = rot / 2;
    const uint32_t step = gridDim.y * (blockDim.x / L);
    // all lanes of a warp take the same number of trips: the norm's shuffles want them together
    for (uint32_t first = blockIdx.y * (blockDim.x / L); first < heads; first += step) {
        const uint32_t i = first + threadIdx.x / L;
        const bool live = i < heads, is_q = i < q_heads, is_k = !is_q && i < q_heads + op.kv_heads;
        const uint32_t h = is_q ? i : is_k ? i - q_heads : i - q_heads - op.kv_heads;
        const S *x = nullptr;
        T *out = nullptr;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (live) {
            x = is_q   ? (const S *)op.q + token * op.q_token_stride + h * op.q_head_stride
                : is_k ? (const S *)op.k + token * op.k_token_stride + h * op.k_head_stride
                       : (const S *)op.v + token * op.v_token_stride + h * op.v_head_stride;
            out = is_q   ? (T *)op.q_out + token * op.q_out_token_stride + h * op.q_out_head_stride
                  : is_k ? (T *)op.kv.k + place + h * op.kv.head_stride
                         : (T *)op.kv.v + place + h * op.kv.head_stride;
            load8(x + d0, v);
        }
        const float *w = is_q ? op.q_norm : is_k ? op.k_norm : nullptr;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += v[j] * v[j];
#pragma unroll
        for (uint32_t o = L / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (!live) continue;
        const float inv = 1.0f / sqrtf(sum / (float)D + op.norm_eps);
        float r[8];
        normed8(v, w, d0, inv, op.norm_offset, r);
        if ((is_q || is_k) && d0 < rot) {
            if (op.pairing == CTOX_ROPE_ADJACENT) {
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    if (d0 + j >= rot) continue;
                    const float2 t = turn[(d0 + j) / 2];
                    const float u = r[j], y = r[j + 1];
                    r[j] = u * t.x - y * t.y;
                    r[j + 1] = y * t.x + u * t.y;
                }
            } else if (half % 8 == 0) {  // eight partners lie together
                const bool low = d0 < half;
                const uint32_t e0 = low ? d0 + half : d0 - half, p0 = low ? d0 : e0;
                float y[8];
                load8(x + e0, y);
                normed8(y, w, e0, inv, op.norm_offset, y);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float2 t = turn[p0 + j];
                    r[j] = low ? r[j] * t.x - y[j] * t.y : r[j] * t.x + y[j] * t.y;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t d = d0 + j;
                    if (d >= rot) continue;
                    const bool low = d < half;
                    const uint32_t other = low ? d + half : d - half;
                    const float y = as_float(x[other]) * (w ? inv * (op.norm_offset + w[other]) : 1.0f);
                    const float2 t = turn[low ? d : other];
                    r[j] = low ? r[j] * t.x - y * t.y : r[j] * t.x + y * t.y;
                }
            }
        }
        *reinterpret_cast<uint4 *>(out + d0) =
            make_uint4(pack_pair<T>(r[0], r[1]), pack_pair<T>(r[2], r[3]), pack_pair<T>(r[4], r[5]), pack_pair<T>(r[6], r[7]));
    }
}

template <typename S, typename T>
cudaError_t launch_rope(ctox_ctx *ctx, const RopeArgs &a) {
    const uint32_t per_trip = 256 / (a.op.dim / 8);
    const uint32_t heads = (a.op.q ? a.op.heads : 0) + (a.op.k ? 2 * a.op.kv_heads : 0);
    const uint32_t trips = (heads + per_trip - 1) / per_trip;
    const dim3 grid(a.op.tokens, a.op.tokens < 2 * (uint32_t)ctx->sm_count ? trips : 1);
    auto kernel = a.op.dim == 64 ? k_rope_append<S, T, 64> : a.op.dim == 128 ? k_rope_append<S, T, 128> : k_rope_append<S, T, 256>;
    return launch_pdl(kernel, grid, dim3(256), 0, ctx->stream, a, ctx->dev_error);
}
template <typename S>
cudaError_t launch_rope(ctox_ctx *ctx, const RopeArgs &a) {
    return a.op.kv.dtype == CTOX_BF16 ? launch_rope<S, __nv_bfloat16>(ctx, a) : launch_rope<S, __half>(ctx, a);
}

ctox_status check_pages(ctox_ctx *ctx, const char *what, uint32_t n, uint32_t page_tokens, uint32_t n_pages, uint32_t table_rows,
                        uint32_t max_pages, uint64_t table_stride) {
    if (!n || n > CTOX_MAX_BATCH) return fail(ctx, CTOX_SHAPE, "%s: %u requests (1 to %u)", what, n, CTOX_MAX_BATCH);
    if (!page_tokens || page_tokens % 16 || !n_pages || (uint64_t)n_pages * page_tokens > 0x7fffffffull)
        return fail(ctx, CTOX_SHAPE, "%s: %u pages of %u tokens (a multiple of 16, below 2^31 tokens in all)", what, n_pages, page_tokens);
    if (!table_rows || !max_pages || table_stride < max_pages || (uint64_t)max_pages * page_tokens > 0x7fffffffull)
        return fail(ctx, CTOX_SHAPE, "%s: block table of %u rows, %u pages each, stride %llu", what, table_rows, max_pages,
                    (unsigned long long)table_stride);
    return CTOX_OK;
}

}  // namespace
}  // namespace paged
}  // namespace ctox

using namespace ctox;
using namespace ctox::paged;

extern "C" {

ctox_status ctox_page_slots(ctox_ctx *ctx, const ctox_page_slots_op *op) {
    if (!op) return fail(ctx, CTOX_SHAPE, "page slots: no operation");
    EX(check_pages(ctx, "page slots", op->n_requests, op->page_tokens, op->n_pages, op->table_rows, op->max_pages, op->table_stride));
    if (op->n_tokens > 0x7fffffffu) return fail(ctx, CTOX_SHAPE, "page slots: %u tokens", op->n_tokens);
    if (!op->new_tokens || !op->kv_lens_in || !op->kv_lens_out || !op->block_table || !op->free_pages || !op->free_count_in ||
        !op->free_count_out || !op->query_offsets || !op->status || (op->n_tokens && (!op->slots || !op->positions)))
        return fail(ctx, CTOX_SHAPE, "page slots: null device pointer");
    if (!ctx) return fail(ctx, CTOX_INVALID_STATE, "page slots: no context");
    const DeviceGuard guard(ctx->device);
    CTOX_CUDA(ctx, guard.error());
    const uint32_t most = op->n_tokens > op->n_requests ? op->n_tokens : op->n_requests;
    const uint32_t want = (most + kPageThreads - 1) / kPageThreads, ctas = want < kPageCtas ? want : kPageCtas;
    // a thread takes two requests; few requests and tokens need no more than a few warps
    const uint32_t threads = ctas > 1 || op->n_requests > 512 ? kPageThreads : most <= 256 ? 256 : kPageThreads;
    CTOX_CUDA(ctx, launch_pdl_cluster(k_page_slots, dim3(ctas), dim3(threads), 0, ctx->stream, ctas, *op, ctx->dev_error));
    return CTOX_OK;
}

ctox_status ctox_page_release(ctox_ctx *ctx, const ctox_page_release_op *op) {
    if (!op) return fail(ctx, CTOX_SHAPE, "page release: no operation");
    EX(check_pages(ctx, "page release", op->n_requests, op->page_tokens, op->n_pages, op->table_rows, op->max_pages, op->table_stride));
    if (!op->kv_lens || !op->block_table || !op->free_pages || !op->free_count_in || !op->free_count_out || !op->status)
        return fail(ctx, CTOX_SHAPE, "page release: null device pointer");
    if (!ctx) return fail(ctx, CTOX_INVALID_STATE, "page release: no context");
    const DeviceGuard guard(ctx->device);
    CTOX_CUDA(ctx, guard.error());
    CTOX_CUDA(ctx, launch_pdl(k_page_release, dim3(1), dim3(kPageThreads), 0, ctx->stream, *op));
    return CTOX_OK;
}

ctox_status ctox_rope_append(ctox_ctx *ctx, const ctox_rope_append_op *op) {
    const char *what = "rope append";
    if (!op) return fail(ctx, CTOX_SHAPE, "%s: no operation", what);
    EX(check_dim(ctx, op->dim, what));
    if (!op->q && !op->k) return fail(ctx, CTOX_SHAPE, "%s: neither queries nor keys", what);
    if (!op->k != !op->v) return fail(ctx, CTOX_SHAPE, "%s: keys and values come together", what);
    if (op->source_dtype != CTOX_F32 && op->source_dtype != CTOX_BF16 && op->source_dtype != CTOX_F16)
        return fail(ctx, CTOX_UNSUPPORTED_DTYPE, "%s: sources of dtype %u", what, op->source_dtype);
    if (op->kv.dtype != CTOX_BF16 && op->kv.dtype != CTOX_F16) return fail(ctx, CTOX_UNSUPPORTED_DTYPE, "%s: dtype %u", what, op->kv.dtype);
    if (op->tokens > 0x7fffffffu) return fail(ctx, CTOX_SHAPE, "%s: %u tokens", what, op->tokens);
    if ((op->q && (!op->heads || op->heads > 65535)) || (op->k && (!op->kv_heads || op->kv_heads > 65535)))
        return fail(ctx, CTOX_SHAPE, "%s: %u query heads, %u KV heads", what, op->heads, op->kv_heads);
    if (op->rot_dim % 2 || op->rot_dim > op->dim) return fail(ctx, CTOX_SHAPE, "%s: %u rotated of %u dimensions", what, op->rot_dim, op->dim);
    if (op->rot_dim) {
        if (!op->positions || op->axes < 1 || op->axes > 255) return fail(ctx, CTOX_SHAPE, "%s: positions on %u axes", what, op->axes);
        for (uint32_t i = 0; i < op->rot_dim / 2; ++i)
            if (op->axis[i] >= op->axes) return fail(ctx, CTOX_SHAPE, "%s: pair %u on axis %u of %u", what, i, op->axis[i], op->axes);
        if (op->pairing != CTOX_ROPE_HALF && op->pairing != CTOX_ROPE_ADJACENT)
            return fail(ctx, CTOX_UNSUPPORTED_OPERATION, "%s: pairing %u", what, op->pairing);
        if (!std::isfinite(op->rope_base) || op->rope_base <= 0) return fail(ctx, CTOX_SHAPE, "%s: base %g", what, op->rope_base);
    }
    if ((op->q_norm && !aligned16(op->q_norm)) || (op->k_norm && !aligned16(op->k_norm)))
        return fail(ctx, CTOX_SHAPE, "%s: norm weights want 16-byte aligned vectors", what);
    if ((op->q_norm || op->k_norm) && !(std::isfinite(op->norm_offset) && op->norm_eps >= 0 && std::isfinite(op->norm_eps)))
        return fail(ctx, CTOX_SHAPE, "%s: norm offset %g, epsilon %g", what, op->norm_offset, op->norm_eps);
    if (op->q && (!op->q_out || !aligned16(op->q) || !aligned16(op->q_out) || op->q_token_stride % 8 || op->q_head_stride % 8 ||
                  op->q_out_token_stride % 8 || op->q_out_head_stride % 8))
        return fail(ctx, CTOX_SHAPE, "%s: queries want 16-byte aligned matrices and strides of multiples of 8", what);
    if (op->k) {
        if (!op->slots) return fail(ctx, CTOX_SHAPE, "%s: keys and values without slots", what);
        if (!aligned16(op->k) || !aligned16(op->v) || op->k_token_stride % 8 || op->k_head_stride % 8 || op->v_token_stride % 8 ||
            op->v_head_stride % 8)
            return fail(ctx, CTOX_SHAPE, "%s: keys and values want 16-byte aligned matrices and strides of multiples of 8", what);
        EX(check_kv(ctx, op->kv, op->kv_heads, what));
    }
    if (!ctx) return fail(ctx, CTOX_INVALID_STATE, "%s: no context", what);
    if (!op->tokens) return CTOX_OK;
    RopeArgs a;
    a.op = *op;
    // rope_base^(-2i / rot_dim) as powers of one factor, in 80 bits: at most 128 roundings of 2^-64
    const long double ratio = op->rot_dim ? powl((long double)op->rope_base, -2.0L / op->rot_dim) : 1.0L;
    long double f = 1.0L / 6.283185307179586476925286766559L;
    for (uint32_t i = 0; i < op->rot_dim / 2; ++i, f *= ratio) a.turns[i] = (double)f;
    const DeviceGuard guard(ctx->device);
    CTOX_CUDA(ctx, guard.error());
    CTOX_CUDA(ctx, op->source_dtype == CTOX_F32    ? launch_rope<float>(ctx, a)
                   : op->source_dtype == CTOX_BF16 ? launch_rope<__nv_bfloat16>(ctx, a)
                                                   : launch_rope<__half>(ctx, a));
    return CTOX_OK;
}

}  // extern "C"
