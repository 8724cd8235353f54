// Attention over a paged K/V cache for requests with many rows: pieces of prompts, whole prompts, long verify passes.
//
// The rows of a request and KV head, (token, query head) pairs in order, are cut into tiles of 128, so that one read of a key
// serves all query heads that share it and a tile is full whatever their number. Scores S = Q K^T and the output O += P V run
// on tcgen05 with accumulators in tensor memory; a thread owns a row for the softmax (running maximum and sum in
// registers) and writes the weights P over its scores, where the next product takes them from. The output is rescaled only when a
// row's maximum has grown by more than 2^8 since its last reference; the division at the end makes up for it.
//
// Up to 128 dimensions a CTA works on two tiles of rows against the same keys: while the tensor cores form one tile's scores and
// output, four warps each do the other's softmax, and a key tile in shared memory serves 256 rows. With 256 dimensions the output
// of one tile fills half of tensor memory, and with one tile of rows there is only one: then even and odd key tiles take turns with
// the two score buffers, so that the scores of the next key tile are formed while the softmax of this one runs.
#include "paged_attention.cuh"
#include "f32x2.cuh"

namespace ctox {
namespace paged {
namespace {

constexpr uint32_t kTileRows = 128, kTileKeys = 128, kTileThreads = 384;
constexpr uint32_t kLoadWarp = 8, kIssueWarp = 9, kMostSlots = 8;
// Registers: twelve warps are launched with 168 each. The softmax warps hold a row of 128 scores and take 208; the four others (copies,
// products, two without work) keep 88: 8 * 208 + 4 * 88 = 12 * 168.
constexpr uint32_t kSoftmaxRegisters = 208, kOtherRegisters = 88;

template <int D>
struct Tile {
    static constexpr uint32_t NQ = D == 256 ? 1 : 2;      // tiles of rows
    static constexpr uint32_t CH = D == 64 ? 1 : 2;       // chunks of 64 dimensions in a slot of the ring
    static constexpr uint32_t HALVES = D == 256 ? 2 : 1;  // slots of a key tile, and of its values
    static constexpr uint32_t SLOT = kTileKeys * CH * 128;
    static constexpr uint32_t Q_BYTES = kTileRows * D * 2;
    static constexpr uint32_t N_O = D < 128 ? D : 128;  // columns of a product with values
    static uint32_t slots(size_t room, uint32_t n) {
        const size_t left = room - 1024 - NQ * Q_BYTES - (n + 1) * 8;
        const uint32_t s = (uint32_t)(left / SLOT);
        return s < kMostSlots ? s : kMostSlots;
    }
    static size_t smem(uint32_t slots, uint32_t n) { return 1024 + NQ * Q_BYTES + (size_t)slots * SLOT + (n + 1) * 8; }
};

// Place in the ring's order of the keys (values) of tile j of n. Two tiles of rows need K0 V0 K1 V1 ..., one needs K0 K1 V0 K2 V1 ...
__device__ __forceinline__ uint32_t key_place(bool two, uint32_t j) { return two ? 2 * j : j < 2 ? j : 2 * j - 1; }
__device__ __forceinline__ uint32_t value_place(bool two, uint32_t j, uint32_t n) { return two ? 2 * j + 1 : j + 1 < n ? 2 * j + 2 : 2 * n - 1; }

template <typename T>
__host__ __device__ constexpr uint32_t idesc(uint32_t n, bool b_mn);
template <>
__host__ __device__ constexpr uint32_t idesc<__nv_bfloat16>(uint32_t n, bool b_mn) {
    return umma::idesc_bf16_mn(kTileRows, n, false, b_mn);
}
template <>
__host__ __device__ constexpr uint32_t idesc<__half>(uint32_t n, bool b_mn) {
    return umma::idesc_bf16_mn(kTileRows, n, false, b_mn) & ~((1u << 7) | (1u << 10));  // the types' fields: 0 for f16
}
// Operands of 128-byte swizzled rows: `group` bytes from eight rows (keys) to the next eight; keys run along m or n, or along k
// with `atom` bytes from 64 dimensions to the next.
__device__ __forceinline__ uint64_t desc_rows(uint32_t addr, uint32_t group) {
    return (uint64_t)((addr & 0x3ffff) >> 4) | (1ull << 16) | ((uint64_t)(group >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_columns(uint32_t addr, uint32_t group, uint32_t atom) {
    return (uint64_t)((addr & 0x3ffff) >> 4) | ((uint64_t)(atom >> 4) << 16) | ((uint64_t)(group >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <typename T, int D>
__global__ void __launch_bounds__(kTileThreads, 1)
    k_attention_tile(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnArgs a,
                     uint32_t slots, int32_t *error_word) {
    using namespace umma;
    using G = Tile<D>;
    extern __shared__ uint8_t raw[];
    // ring; queries of each tile of rows; scores and weights of score buffer 0, of buffer 1 when it is the second tile's, and of
    // buffer 1 when it is the first's; end of a unit for each tile of rows; products with values that a rescale waits for
    __shared__ __align__(8) uint64_t bars[2 * kMostSlots + 2 + 3 + 3 + 2 + 2 + 1];
    __shared__ unsigned long long scan[32];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int dead;
    __shared__ Cut cuts[2];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = (smem_addr(raw) + 1023) & ~1023u, q_s = base, ring = q_s + G::NQ * G::Q_BYTES;
    unsigned long long *at = reinterpret_cast<unsigned long long *>(raw + (ring + slots * G::SLOT - smem_addr(raw)));
    const uint32_t full = smem_addr(bars), empty = full + kMostSlots * 8, q_full = empty + kMostSlots * 8, s_full = q_full + 16,
                   p_full = s_full + 24, fin = p_full + 24, o_done = fin + 16, drained = o_done + 16;
    if (tid == 0) {
        dead = 0;
        for (uint32_t i = 0; i < slots; ++i) {
            bar_init(full + i * 8, 1);
            bar_init(empty + i * 8, 1);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            bar_init(q_full + i * 8, 4);
            bar_init(fin + i * 8, 1);
            bar_init(o_done + i * 8, 1);
        }
        for (uint32_t i = 0; i < 3; ++i) {
            bar_init(s_full + i * 8, 1);
            bar_init(p_full + i * 8, 4);
        }
        bar_init(drained, 1);
        bar_init_fence();
    }
    if (warp == kIssueWarp) tmem_alloc(smem_addr(&tmem_slot), 512);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_launch();
    pdl_wait();
    const uint64_t total = lay_line(a, at, scan, error_word);
    const uint32_t pieces = total ? pieces_of(total, gridDim.x, a.least) : 0;
    const Line line{a, at, a.op.n_requests};
    Walk w;
    w.at.x = w.end = 0;
    if (blockIdx.x < pieces) {
        if (warp < 2) {
            const Cut c = cut_at(a.shape, line, total, pieces, blockIdx.x + warp, a.least);
            if (lane == 0) cuts[warp] = c;
        }
        __syncthreads();
        w.at = cuts[0];
        w.end = cuts[1].x;
    }
    bool ok = true;
    if (warp >= kLoadWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
        if (warp == kLoadWarp) {
            const uint32_t per = kTileKeys / a.box, box_bytes = a.box * G::CH * 128;
            uint32_t n = 0;  // slots filled
            for (; ok && walk_unit(a.shape, line, w); walk_on(a.shape, line, w)) {
                const int32_t *table = table_row(a, w.at.request);
                const bool two = w.u.rows > kTileRows;
                const uint32_t tiles = w.tile1 - w.tile0;
                uint32_t kj = 0, vj = 0;  // the next tile of each
                for (uint32_t i = 0; ok && i < 2 * tiles; ++i) {
                    const bool is_k = kj < tiles && key_place(two, kj) == i;
                    const uint32_t j = is_k ? kj++ : vj++;
                    const uint32_t token = (w.u.tile0 + w.tile0 + j) * kTileKeys + lane * a.box;
                    int32_t page = -1;
                    bool mine = lane < per && token < w.u.hi && token + a.box > w.u.lo;
                    if (mine) mine = page_at(a, table, token, page, error_word);
                    const uint32_t copies = __popc(__ballot_sync(0xffffffffu, mine));
                    for (uint32_t h = 0; h < G::HALVES; ++h, ++n) {
                        const uint32_t s = n % slots, round = n / slots;
                        if (round > 0 && !(ok = __all_sync(0xffffffffu, bar_wait(empty + s * 8, (round - 1) & 1, &dead)))) break;
                        if (lane == 0) bar_expect(full + s * 8, copies * box_bytes);
                        __syncwarp();
                        if (mine)
                            load_box(ring + s * G::SLOT + lane * box_bytes, is_k ? &map_k : &map_v, full + s * 8, (int)(h * G::CH),
                                     (int)(token % a.op.kv.page_tokens / 8), box_step(a, page, w.at.head));
                    }
                }
            }
            if (!ok && lane == 0)  // leave no copy in flight behind
                for (uint32_t s = 0; s < slots && s < n; ++s) bar_drain(full + s * 8, ((n - 1 - s) / slots) & 1);
        } else if (warp == kIssueWarp) {
            constexpr uint32_t idesc_s = idesc<T>(kTileKeys, false), idesc_o = idesc<T>(G::N_O, true);
            const bool leader = elect_one();  // one thread throughout: a commit covers what its own thread issued
            uint32_t ring0 = 0, units[2] = {0, 0}, weights[3] = {0, 0, 0};
            for (; ok && walk_unit(a.shape, line, w); walk_on(a.shape, line, w)) {
                const bool two = w.u.rows > kTileRows;
                const uint32_t tiles = w.tile1 - w.tile0, steps = two ? 2 * tiles : tiles;
                if (!tiles) continue;
                auto slot_full = [&](uint32_t place, uint32_t h) {
                    const uint32_t n = ring0 + place * G::HALVES + h;
                    return __all_sync(0xffffffffu, bar_wait(full + n % slots * 8, (n / slots) & 1, &dead));
                };
                auto slot_of = [&](uint32_t place, uint32_t h) { return (ring0 + place * G::HALVES + h) % slots; };
                auto scores = [&](uint32_t i) {
                    const uint32_t j = two ? i >> 1 : i, t = two ? i & 1 : 0, place = key_place(two, j);
                    for (uint32_t h = 0; h < G::HALVES; ++h)
                        if (!slot_full(place, h)) return false;
                    fence_after();
                    if (leader) {
                        uint64_t dq = desc_rows(q_s + t * G::Q_BYTES, 1024);
#pragma unroll
                        for (uint32_t h = 0; h < G::HALVES; ++h) {
                            uint64_t dk = desc_rows(ring + slot_of(place, h) * G::SLOT, G::CH * 1024);
                            asm volatile("" : "+l"(dq), "+l"(dk));  // formed here, not kept for the whole unit
#pragma unroll
                            for (uint32_t k = 0; k < G::CH * 4; ++k)
                                mma_f16(tmem + (i & 1) * kTileKeys, dq + ((h * G::CH + k / 4) * (kTileRows * 128) + k % 4 * 32) / 16,
                                        dk + (k / 4 * 1024 + k % 4 * 32) / 16, idesc_s, h > 0 || k > 0);
                        }
                        commit(s_full + (two ? i & 1 : (i & 1) * 2) * 8);
                        if (!two || t == 1)
                            for (uint32_t h = 0; h < G::HALVES; ++h) commit(empty + slot_of(place, h) * 8);
                    }
                    __syncwarp();
                    return true;
                };
                ok = __all_sync(0xffffffffu, bar_wait(q_full, units[0] & 1, &dead) && (!two || bar_wait(q_full + 8, units[1] & 1, &dead)));
                ++units[0];
                if (two) ++units[1];
                fence_after();
                ok = ok && scores(0) && (steps < 2 || scores(1));
                for (uint32_t i = 0; ok && i < steps; ++i) {
                    const uint32_t j = two ? i >> 1 : i, t = two ? i & 1 : 0, b = two ? i & 1 : (i & 1) * 2, place = value_place(two, j, tiles);
                    if (!(ok = __all_sync(0xffffffffu, bar_wait(p_full + b * 8, weights[b] & 1, &dead)))) break;
                    ++weights[b];
                    for (uint32_t h = 0; ok && h < G::HALVES; ++h) ok = slot_full(place, h);
                    if (!ok) break;
                    const uint32_t key0 = (w.u.tile0 + w.tile0 + j) * kTileKeys;
                    if (t == 0 && (key0 < w.u.lo || key0 + kTileKeys > w.u.hi)) {
                        // values in places that no row sees may be anything, and 0 times that is not 0
                        for (uint32_t r = 0; r < kTileKeys; ++r) {
                            if (key0 + r >= w.u.lo && key0 + r < w.u.hi) continue;
                            for (uint32_t h = 0; h < G::HALVES; ++h)
                                if (lane < G::CH * 8)
                                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(ring + slot_of(place, h) * G::SLOT +
                                                                                                  (r >> 3) * (G::CH * 1024) + (lane >> 3) * 1024 +
                                                                                                  (r & 7) * 128 + (lane & 7) * 16),
                                                 "r"(0)
                                                 : "memory");
                        }
                        proxy_fence();
                        __syncwarp();
                    }
                    fence_after();
                    if (leader) {
#pragma unroll
                        for (uint32_t h = 0; h < G::HALVES; ++h) {
                            uint64_t dv = desc_columns(ring + slot_of(place, h) * G::SLOT, G::CH * 1024, 1024);
                            asm volatile("" : "+l"(dv));
#pragma unroll
                            for (uint32_t k = 0; k < kTileKeys / 16; ++k)
                                mma_f16_ts(tmem + 256 + t * D + h * 128, tmem + (i & 1) * kTileKeys + k * 8, dv + k * (2 * G::CH * 1024 / 16), idesc_o,
                                           j > 0 || k > 0);
                        }
                        if (!two || t == 1)
                            for (uint32_t h = 0; h < G::HALVES; ++h) commit(empty + slot_of(place, h) * 8);
                        if (!two) commit(o_done + (i & 1) * 8);
                        if (j + 1 == tiles) commit(fin + t * 8);
                    }
                    __syncwarp();
                    if (i + 2 < steps) ok = scores(i + 2);
                }
                ring0 += 2 * tiles * G::HALVES;
            }
            if (!ok) {
                if (leader) commit(drained);
                __syncwarp();
                bar_drain(drained, 0);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegisters));
        const uint32_t t = warp >> 2, row = tid & 127, lanes = ((warp & 3) * 32) << 16;  // tile of rows, row in it
        const float c = a.c;
        bool shares = false;
        uint32_t units = 0, seen[2] = {0, 0}, done[2] = {0, 0};
        for (; ok && walk_unit(a.shape, line, w); walk_on(a.shape, line, w)) {
            const bool two = w.u.rows > kTileRows;
            const uint32_t tiles = w.tile1 - w.tile0, group = a.shape.group;
            if (w.begins && !w.ends) {
                shares = true;
                if (tid == 0)
                    a.shared[blockIdx.x] = Shared{sharers(total, pieces, blockIdx.x, w.at.start + w.u.cost), w.at.request, w.at.head, w.u.row0, w.u.rows};
            }
            const uint32_t in = t * kTileRows + row, r = w.u.row0 + in;
            const bool live = in < w.u.rows;
            const uint32_t token = w.q.q0 + r / group, head = w.at.head * group + r % group;
            float ref = -INFINITY;
            f32x2 sums[2] = {0, 0};
            if (tiles && (t == 0 || two)) {
                {  // queries; the products of the unit before have finished
                    const uint4 *q = reinterpret_cast<const uint4 *>((const T *)a.op.q + (uint64_t)token * a.op.q_token_stride +
                                                                     (uint64_t)head * a.op.q_head_stride);
                    const uint32_t d = q_s + t * G::Q_BYTES + row * 128;
#pragma unroll
                    for (uint32_t i = 0; i < D / 8; ++i) {
                        const uint4 x = live ? q[i] : make_uint4(0, 0, 0, 0);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(d + i / 8 * (kTileRows * 128) + ((i % 8 ^ (row & 7)) << 4)),
                                     "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w)
                                     : "memory");
                    }
                    proxy_fence();
                    __syncwarp();
                    if (lane == 0) bar_arrive(q_full + t * 8);
                }
                uint32_t lo = 0, hi = 0;
                if (live) key_range(a.shape, w.q, r, r + 1, lo, hi);
                const bool idle = !__any_sync(0xffffffffu, live);
                for (uint32_t j = 0; j < tiles; ++j) {
                    const uint32_t buf = two ? t : j & 1, b = two ? t : (j & 1) * 2, o = j & 1;  // score buffer, its barriers
                    uint32_t &phase = seen[!two && o];
                    if (!(ok = __all_sync(0xffffffffu, bar_wait(s_full + b * 8, phase & 1, &dead)))) break;
                    ++phase;
                    fence_after();
                    if (!idle) {
                        float s[kTileKeys];
#pragma unroll
                        for (uint32_t k = 0; k < kTileKeys; k += 32) tmem_ld32(tmem + buf * kTileKeys + k + lanes, s + k);
                        tmem_ld_wait();
                        const uint32_t key0 = (w.u.tile0 + w.tile0 + j) * kTileKeys;
                        if (__any_sync(0xffffffffu, key0 < lo || key0 + kTileKeys > hi)) {
#pragma unroll
                            for (uint32_t k = 0; k < kTileKeys; ++k)
                                if (key0 + k < lo || key0 + k >= hi) s[k] = -INFINITY;
                        }
                        float m4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                        for (uint32_t k = 4; k < kTileKeys; k += 8)
#pragma unroll
                            for (uint32_t x = 0; x < 4; ++x)
                                m4[x] = k + 4 + x < kTileKeys ? fmaxf(fmaxf(m4[x], s[k + x]), s[(k + 4 + x) % kTileKeys]) : fmaxf(m4[x], s[k + x]);
                        const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * c;
                        const bool grow = mx > ref + 8.f || (ref == -INFINITY && mx > ref);
                        if (__any_sync(0xffffffffu, grow)) {
                            const float f = grow ? ex2(ref - mx) : 1.f;  // ref = -inf: 0, and nothing but zeros was added
                            if (grow) ref = mx;
                            const f32x2 ff = pack2(f, f);
                            sums[0] = mul2(sums[0], ff);
                            sums[1] = mul2(sums[1], ff);
                            if (j > 0) {
                                // The output belongs to the product of the key tile before. With two tiles of rows that one has finished: it was
                                // issued before the scores that this warp waited for. With one, the scores are a tile ahead of it.
                                if (!two) {
                                    const uint32_t before = o ^ 1;
                                    if (!(ok = __all_sync(0xffffffffu, bar_wait(o_done + before * 8, (done[before] - 1) & 1, &dead)))) break;
                                    fence_after();
                                }
#pragma unroll 1
                                for (uint32_t d = 0; d < D; d += 16) {
                                    float v[16];
                                    tmem_ld16(tmem + 256 + t * D + d + lanes, v);
                                    tmem_ld_wait();
#pragma unroll
                                    for (int i = 0; i < 16; ++i) v[i] *= f;
                                    tmem_st16(tmem + 256 + t * D + d + lanes, v);
                                }
                            }
                        }
                        const float m = ref == -INFINITY ? 0.f : ref;
                        const f32x2 cc = pack2(c, c), mm = pack2(-m, -m), one = pack2(1.f, 1.f);
#pragma unroll
                        for (uint32_t k0 = 0; k0 < kTileKeys; k0 += 32) {
                            uint32_t p[16];
#pragma unroll
                            for (uint32_t k = 0; k < 32; k += 2) {
                                float x, y;
                                unpack2(fma2(pack2(s[k0 + k], s[k0 + k + 1]), cc, mm), x, y);
                                x = ex2(x);
                                y = ex2(y);
                                sums[k / 2 & 1] = fma2(pack2(x, y), one, sums[k / 2 & 1]);
                                p[k / 2] = pack_pair<T>(x, y);
                            }
                            tmem_st16(tmem + buf * kTileKeys + k0 / 2 + lanes, reinterpret_cast<const float *>(p));
                        }
                        tmem_st_wait();
                        fence_before();
                    }
                    if (!two) ++done[o];
                    __syncwarp();
                    if (lane == 0) bar_arrive(p_full + b * 8);
                }
                if (!ok) break;
                if (!(ok = __all_sync(0xffffffffu, bar_wait(fin + t * 8, units & 1, &dead)))) break;
                ++units;
                fence_after();
            }
            if (t > 0 && !two) continue;
            float sum, x[4];
            unpack2(sums[0], x[0], x[1]);
            unpack2(sums[1], x[2], x[3]);
            sum = (x[0] + x[1]) + (x[2] + x[3]);
            if (w.begins && w.ends) {
                float inv = 0.f;
                if (sum != 0.f) {
                    if (a.op.sinks && live) sum += ex2(fmaf(a.op.sinks[head], 1.4426950408889634f, -ref));
                    inv = 1.0f / sum;
                }
                T *out = (T *)a.op.out + (uint64_t)token * a.op.out_token_stride + (uint64_t)head * a.op.out_head_stride;
#pragma unroll 1
                for (uint32_t d = 0; d < D; d += 32) {
                    float v[32];
                    tmem_ld32(tmem + 256 + t * D + d + lanes, v);
                    tmem_ld_wait();
                    if (live) {
#pragma unroll
                        for (uint32_t i = 0; i < 32; i += 8)
                            *reinterpret_cast<uint4 *>(out + d + i) =
                                sum == 0.f ? make_uint4(0, 0, 0, 0)
                                           : make_uint4(pack_pair<T>(v[i] * inv, v[i + 1] * inv), pack_pair<T>(v[i + 2] * inv, v[i + 3] * inv),
                                                        pack_pair<T>(v[i + 4] * inv, v[i + 5] * inv), pack_pair<T>(v[i + 6] * inv, v[i + 7] * inv));
                    }
                }
            } else {
                const uint32_t BR = G::NQ * kTileRows;
                float *slot = a.partial + (blockIdx.x * 2ull + (w.begins ? 1 : 0)) * slot_floats(BR, D);
                slot[in] = ref;
                slot[BR + in] = sum;
                float4 *part = reinterpret_cast<float4 *>(slot + 2 * BR);
                if (tiles)
#pragma unroll 1
                    for (uint32_t d = 0; d < D; d += 16) {
                        float v[16];
                        tmem_ld16(tmem + 256 + t * D + d + lanes, v);
                        tmem_ld_wait();
#pragma unroll
                        for (uint32_t i = 0; i < 16; i += 4) part[((d + i) / 4) * BR + in] = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                    }
            }
            fence_before();  // the next unit's products write the output
        }
        if (!shares && tid == 0) a.shared[blockIdx.x].sharers = 0;
    }
    __syncwarp();
    __syncthreads();
    if (warp == kIssueWarp) {
        fence_after();
        tmem_free(tmem, 512);
    }
    if (tid == 0 && dead) *error_word = DEV_ERR_WAIT_TIMEOUT;
}

template <typename T, int D>
ctox_status tile_launch(ctox_ctx *ctx, AttnArgs &a) {
    using G = Tile<D>;
    a.box = kTileKeys;
    while (a.op.kv.page_tokens % a.box) a.box /= 2;
    CUtensorMap mk, mv;
    EX(cache_map(ctx, &mk, a.op, a.op.kv.k, a.box, G::CH));
    EX(cache_map(ctx, &mv, a.op, a.op.kv.v, a.box, G::CH));
    const size_t room = (size_t)ctx->max_smem_optin - 1024;  // static shared memory
    const uint32_t slots = G::slots(room, a.op.n_requests);
    const size_t smem = G::smem(slots, a.op.n_requests);
    auto kernel = k_attention_tile<T, D>;
    CTOX_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    CTOX_CUDA(ctx, launch_pdl(kernel, dim3((uint32_t)ctx->sm_count), dim3(kTileThreads), smem, ctx->stream, mk, mv, a, slots, ctx->dev_error));
    return CTOX_OK;
}
template <typename T>
ctox_status tile_launch(ctox_ctx *ctx, AttnArgs &a) {
    return a.op.dim == 64 ? tile_launch<T, 64>(ctx, a) : a.op.dim == 128 ? tile_launch<T, 128>(ctx, a) : tile_launch<T, 256>(ctx, a);
}

}  // namespace

uint32_t tile_block_rows(uint32_t dim) { return dim == 256 ? kTileRows : 2 * kTileRows; }

ctox_status launch_attention_tile(ctox_ctx *ctx, AttnArgs &a) {
    a.shape.block_rows = tile_block_rows(a.op.dim);
    a.shape.half_rows = kTileRows;
    a.shape.key_tile = kTileKeys;
    return a.op.kv.dtype == CTOX_BF16 ? tile_launch<__nv_bfloat16>(ctx, a) : tile_launch<__half>(ctx, a);
}

}  // namespace paged
}  // namespace ctox
