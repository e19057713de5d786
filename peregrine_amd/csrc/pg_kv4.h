// The paged key/value cache in 4 bits: layout and the device functions that its kernels share.
//
// A row is one head of one token, keys and values alike: codes n of 0 .. 15 with a centre z and a step d, both bfloat16,
// value = z + d (n - 7.5).  The step is one per row and not one per 32 channels: it then multiplies a whole score (keys) or
// a whole probability (values), so the matrix cores take the codes as they are and no value is ever dequantised.
//
// A block holds block_size tokens (a power of two, 16 .. 256) of every key head.  Its record for one head, bytes:
//   key codes [block_size][D / 2], value codes [block_size][D / 2], key (z, d) [block_size], value (z, d) [block_size]
// with D = head_dim up to 64, 128 or 256 (codes behind head_dim are 0), two codes a byte with the even channel in the low
// half, and z in the low 16 bits of its word.  Heads of a block follow one another, then the next block.
// Its summary for one head: int8 hi[D], lo[D] (the most and least of each channel over the block's keys, in units of
// `scale`), scale f32, 12 bytes unused.  scale = inf marks a block that holds a row that is not finite.
#pragma once
#include "pg_internal.h"

// The position of what is in no block: beyond every query, and so far under 2^31 that a tile's places behind it are still counted in 32
// bits.  A table holds no more tokens than that.
constexpr int KV4_NOWHERE = 0x7fffff00;
constexpr size_t PG_KV4_MAX_TOKENS = KV4_NOWHERE;

struct pg_paged_kv4 {
    uint8_t *data, *sums;
    size_t num_blocks, block_size, heads, head_dim;
    int D, shift;  // stored channels of a row, log2(block_size)
    mutable pg_dev_block mem, sums_mem;
    int device;
    void touch(const pg_ctx *ctx) const { mem.touch(ctx); sums_mem.touch(ctx); }
    pg_status use(const char *fn, const pg_ctx *ctx) const {
        PG_CHECK_ARG(ctx->device == device, "%s: a cache on device %d, a context on device %d", fn, device, ctx->device);
        touch(ctx);
        return PG_OK;
    }
};

// What a kernel needs to know of a cache.
struct kv4_view {
    uint8_t *data, *sums;
    int num_blocks, heads, head_dim, shift;
};
inline kv4_view kv4_view_of(const pg_paged_kv4 *c) {
    return {c->data, c->sums, (int)c->num_blocks, (int)c->heads, (int)c->head_dim, c->shift};
}
// A step's requests as its kernels read them.
struct kv4_batch {
    const int *starts, *lens, *table;
    int batch, tokens, max_blocks;
};

template <int D>
struct kv4_rec {
    static constexpr int ROW = D / 2;
    static __host__ __device__ size_t bytes(int shift) { return (size_t)(D + 8) << shift; }
    static __host__ __device__ size_t v(int shift) { return (size_t)ROW << shift; }
    static __host__ __device__ size_t k_meta(int shift) { return (size_t)D << shift; }
    static __host__ __device__ size_t v_meta(int shift) { return (size_t)(D + 4) << shift; }
    static constexpr size_t SUM = 2 * D + 16;
};

__device__ __forceinline__ float kv4_z(uint32_t meta) { return __builtin_bit_cast(float, meta << 16); }
__device__ __forceinline__ float kv4_d(uint32_t meta) { return __builtin_bit_cast(float, meta & 0xffff0000u); }

// What a request of the batch asks of a step, made safe: rows outside the packed array and lengths outside the table are cut.
struct kv4_request {
    int first, rows, len;  // first packed row, rows, tokens in the cache (the rows among them: they are the last)
};
__device__ __forceinline__ kv4_request kv4_request_of(const kv4_batch &ba, int from, int to, int len, int shift) {
    kv4_request r = {from, to - from, (int)min((long)max(len, 0), (long)ba.max_blocks << shift)};
    if (from < 0 || to < from || from > ba.tokens) r.rows = 0;
    return r;
}
__device__ __forceinline__ kv4_request kv4_request_at(const kv4_batch &ba, int b, int shift) { return kv4_request_of(ba, ba.starts[b], ba.starts[b + 1], ba.lens[b], shift); }

// The request that packed row t belongs to and what it asks, or -1: a lane looks at a request, so that up to 64 of them cost one
// memory latency.  The whole wavefront asks.
__device__ __forceinline__ int kv4_find(const kv4_batch &ba, int t, int shift, kv4_request &r) {
    const int lane = threadIdx.x & 63;
    for (int at = 0; at < ba.batch; at += 64) {
        const int i = min(at + lane, ba.batch - 1);
        const int from = ba.starts[i], to = ba.starts[i + 1], len = ba.lens[i];
        const uint64_t mine = __ballot(at + lane < ba.batch && from <= t && t < to);
        if (mine) {
            const int who = __builtin_ctzll(mine);
            r = kv4_request_of(ba, __builtin_amdgcn_readlane(from, who), __builtin_amdgcn_readlane(to, who), __builtin_amdgcn_readlane(len, who), shift);
            return r.rows > 0 ? at + who : -1;
        }
    }
    return -1;
}

// Sums and maxima across lanes without LDS: DPP moves within 16, swaps of rows and halves beyond.
struct kv4_add { __device__ float operator()(float a, float b) const { return a + b; } };
struct kv4_max { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct kv4_umax { __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; } };
struct kv4_iadd { __device__ int operator()(int a, int b) const { return a + b; } };
template <class T, class F>
__device__ __forceinline__ T over_16(T v, F f) {  // lanes of a row of 16
    const auto move = [](T x, auto ctrl) { return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, false)); };
    v = f(v, move(v, std::integral_constant<int, 0xB1>{}));   // quad_perm [1,0,3,2]
    v = f(v, move(v, std::integral_constant<int, 0x4E>{}));   // quad_perm [2,3,0,1]
    v = f(v, move(v, std::integral_constant<int, 0x141>{}));  // row_half_mirror
    return f(v, move(v, std::integral_constant<int, 0x140>{}));  // row_mirror
}
template <class T, class F>
__device__ __forceinline__ T over_rows(T v, F f) {  // lane and lane ^ 16
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    return f(__builtin_bit_cast(T, (unsigned)r[0]), __builtin_bit_cast(T, (unsigned)r[1]));
}
template <class T, class F>
__device__ __forceinline__ T over_halves(T v, F f) {  // lane and lane ^ 32
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    return f(__builtin_bit_cast(T, (unsigned)r[0]), __builtin_bit_cast(T, (unsigned)r[1]));
}
template <class T, class F>
__device__ __forceinline__ T over_wave(T v, F f) { return over_halves(over_rows(over_16(v, f), f), f); }

pg_status pg_kv4_check_step(const char *fn, const pg_paged_kv4 *c, size_t num_q_heads, size_t batch, size_t tokens, size_t max_blocks);
