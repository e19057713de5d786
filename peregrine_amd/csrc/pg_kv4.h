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

struct pg_paged_kv4 {
    uint8_t *data, *sums;
    size_t num_blocks, block_size, heads, head_dim;
    int D, shift;  // stored channels of a row, log2(block_size)
    mutable pg_dev_block mem, sums_mem;
    void touch(const pg_ctx *ctx) const { mem.touch(ctx); sums_mem.touch(ctx); }
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

// The request that packed row t belongs to (starts ascending, batch + 1 of them), or -1; the whole wavefront asks.
__device__ __forceinline__ int kv4_request_of(const int *__restrict__ starts, int batch, int t) {
    int below = 0;
    for (int i = threadIdx.x & 63; i - (int)(threadIdx.x & 63) <= batch; i += 64)
        below += __popcll(__ballot(i <= batch && starts[min(i, batch)] <= t));
    return below >= 1 && below <= batch ? below - 1 : -1;
}

// What a request of the batch asks of a step, made safe: rows outside the packed array and lengths outside the table are cut.
struct kv4_request {
    int first, rows, len;  // first packed row, rows, tokens in the cache (the rows among them: they are the last)
};
__device__ __forceinline__ kv4_request kv4_request_at(const kv4_batch &ba, int b, int shift) {
    kv4_request r;
    r.first = ba.starts[b];
    r.rows = ba.starts[b + 1] - r.first;
    const long most = (long)ba.max_blocks << shift;
    r.len = (int)min((long)max(ba.lens[b], 0), most);
    if (r.first < 0 || r.rows < 0 || r.first > ba.tokens) r.rows = 0;
    return r;
}

pg_status pg_kv4_check_step(const char *fn, const pg_paged_kv4 *c, size_t num_q_heads, size_t batch, size_t tokens, size_t max_blocks);
