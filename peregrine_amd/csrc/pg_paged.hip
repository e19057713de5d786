// Block tables made on the GPU, and the paged key/value cache in 4 bits: its memory, the append, the read-back, the
// blocks' summaries.
#include <math.h>
#include <new>
#include "pg_kv4.h"

namespace {

// ---- block tables ---------------------------------------------------------------------------

__device__ __forceinline__ int blocks_of(long tokens, int shift) { return (int)((tokens + (1l << shift) - 1) >> shift); }

// Sums over the threads below this one in a workgroup of 1024, and over all of them, of two numbers; part: 32 words of LDS.
__device__ __forceinline__ void below_sums(long &a, long &b, long *part, long *all_a, long *all_b) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    long s = a, t = b;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const long u = __shfl_up(s, d), v = __shfl_up(t, d);
        if (lane >= d) s += u, t += v;
    }
    __syncthreads();
    if (lane == 63) part[wave] = s, part[16 + wave] = t;
    __syncthreads();
    long below_a = 0, below_b = 0, sum_a = 0, sum_b = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        const long p = part[w], q = part[16 + w];
        below_a += w < wave ? p : 0, below_b += w < wave ? q : 0;
        sum_a += p, sum_b += q;
    }
    *all_a = sum_a, *all_b = sum_b;
    a = below_a + s - a, b = below_b + t - b;
}

// The last of n ascending numbers that is at most v (the first is).
__device__ __forceinline__ int last_upto(const int *at, int n, int v) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (at[mid] <= v) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// The slot of position pos in block phys, -1 where that is no block (its number could wrap to another block's slot).
__device__ __forceinline__ int slot_of(int phys, int pos, int shift, int num_blocks) {
    return (unsigned)phys < (unsigned)num_blocks ? phys << shift | (pos & ((1 << shift) - 1)) : -1;
}

// The requests in runs of 1024, a thread a request: rows and needs are prefix sums.  Needs are counted whether they are met or
// not, so those that are met come first: a granted request's new blocks begin at the sum of the needs before it, and new entries
// and slots are flat lists, a thread a place, the request by bisection in LDS.  A slot in a new block comes from the free list like
// the entry itself, so nothing waits for what this launch writes.  A few loads behind one another bound it: 256 decoding
// requests 6.0 us, 13.4 with a wavefront a request for entries and slots; 200 prompts with 223 000 slots 10.4 us on 55 workgroups.
// Workgroup w does the slots of rows 4096 w .. and on; the first does everything else, and may write lengths and count over their
// inputs if it is the only one (slots = null: no slots, slot_map_kernel does them).
__global__ __launch_bounds__(1024) void extend_tables_kernel(const int *seq_lens, const int *new_lens, int batch, int shift, const int *free_list, const int *free_count,
                                                             int num_blocks, int *table, int max_blocks, int *lens_out, int *free_out, int *starts, int *granted,
                                                             int *slots, int max_tokens) {
    __shared__ long part[32];
    __shared__ int first_row[1024], base_pos[1024], old_blocks[1024], first_need[1024];
    __shared__ uint8_t fine[1024];
    __shared__ int handed;
    const int have_free = min(max(*free_count, 0), num_blocks), tid = threadIdx.x;
    const bool all_else = blockIdx.x == 0;
    const long from_row = (long)blockIdx.x * 4096, to_row = min(from_row + 4096, (long)max_tokens);
    const long most = (long)max_blocks << shift;
    long rows_before = 0, needs_before = 0;  // of the runs before this one
    if (tid == 0) handed = 0;
    for (int at = 0; at < batch; at += 1024) {
        const int b = at + tid, run = min(1024, batch - at);
        const int len = b < batch ? max(seq_lens[b], 0) : 0, add = b < batch ? max(new_lens[b], 0) : 0;
        const bool fits = (long)len + add <= most;
        const int have = blocks_of(len, shift);
        const int need = b < batch && fits ? blocks_of((long)len + add, shift) - have : 0;
        long row = add, before = need, rows_all, needs_all;
        below_sums(row, before, part, &rows_all, &needs_all);
        row += rows_before, before += needs_before;
        const bool ok = b < batch && fits && (need == 0 || before + need <= have_free);
        first_row[tid] = (int)min(row, (long)max_tokens);
        base_pos[tid] = len;
        old_blocks[tid] = have;
        first_need[tid] = (int)min(before, (long)num_blocks);
        fine[tid] = ok;
        if (ok && need) atomicMax(&handed, (int)(before + need));
        if (all_else && b < batch) {
            starts[b] = (int)min(row, (long)max_tokens);
            granted[b] = ok;
            lens_out[b] = ok ? len + add : len;
        }
        __syncthreads();
        for (int e = (int)min(needs_before, (long)num_blocks) + 1024 * blockIdx.x + tid; e < handed; e += 1024 * gridDim.x) {
            const int i = last_upto(first_need, run, e);
            table[(size_t)(at + i) * max_blocks + old_blocks[i] + e - first_need[i]] = free_list[have_free - 1 - e];
        }
        if (slots) {
            const int upto = (int)min(min(rows_before + rows_all, (long)max_tokens), to_row);
            const int from = (int)max(min(rows_before, (long)max_tokens), from_row);
            int pos[4], phys[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {  // a thread's four places' loads go out together
                const int j = from + tid + 1024 * u;
                pos[u] = -1, phys[u] = 0;
                if (j < upto) {
                    const int i = last_upto(first_row, run, j), p = base_pos[i] + j - first_row[i], block = p >> shift;
                    if (fine[i]) {
                        const int *from_list = free_list + (have_free - 1 - (first_need[i] + block - old_blocks[i]));
                        phys[u] = *(block < old_blocks[i] ? table + (size_t)(at + i) * max_blocks + block : from_list);
                        pos[u] = p;
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int j = from + tid + 1024 * u;
                if (j < upto) slots[j] = pos[u] < 0 ? -1 : slot_of(phys[u], pos[u], shift, num_blocks);
            }
        }
        rows_before += rows_all;
        needs_before += needs_all;
        __syncthreads();
    }
    const int rows = (int)min(rows_before, (long)max_tokens);
    if (all_else && tid == 0) {
        starts[batch] = rows;
        *free_out = have_free - handed;
    }
    if (slots)
        for (int j = max(rows, (int)from_row) + tid; j < to_row; j += 1024) slots[j] = -1;
}

// The slot map over the chip: a thread a row, its request by bisection.  lens are those after the step; a granted request's rows
// begin new_lens before them -- not so many rows before them as it has, which max_tokens may have cut.
__global__ __launch_bounds__(256) void slot_map_kernel(const int *__restrict__ starts, const int *__restrict__ lens, const int *__restrict__ new_lens, int batch, int shift,
                                                       const int *__restrict__ table, int max_blocks, const int *__restrict__ granted, int *__restrict__ slots, int max_tokens,
                                                       int num_blocks) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= max_tokens) return;
    int slot = -1;
    if (t < starts[batch]) {
        int lo = 0, hi = batch - 1;  // the last request that starts at or before t
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (starts[mid] <= t) lo = mid;
            else hi = mid - 1;
        }
        if (granted[lo]) {
            const int pos = lens[lo] - max(new_lens[lo], 0) + (t - starts[lo]);
            slot = slot_of(table[(size_t)lo * max_blocks + (pos >> shift)], pos, shift, num_blocks);
        }
    }
    slots[t] = slot;
}

// Blocks of flagged requests back to the free list, requests and their blocks in ascending order.
__global__ __launch_bounds__(1024) void release_tables_kernel(const int *release, int *seq_lens, int batch, int shift, int *table, int max_blocks, int *free_list,
                                                              int *free_count, int num_blocks) {
    __shared__ long part[32];
    __shared__ int valid[1024], first[1024];
    const int tid = threadIdx.x, lane = tid & 63;
    int top = min(max(*free_count, 0), num_blocks);
    for (int at = 0; at < batch; at += 1024) {
        const int run = min(1024, batch - at);
        for (int i = tid >> 6; i < run; i += 16) {
            int n = 0;
            if (release[at + i]) {
                const int blocks = min(blocks_of(max(seq_lens[at + i], 0), shift), max_blocks);
                for (int j = lane; j - lane < blocks; j += 64) {
                    const int e = j < blocks ? table[(size_t)(at + i) * max_blocks + j] : -1;
                    n += __popcll(__ballot(e >= 0 && e < num_blocks));
                }
            }
            if (lane == 0) valid[i] = n;
        }
        __syncthreads();
        long all, mine = tid < run ? valid[tid] : 0, none = 0, no_sum;
        below_sums(mine, none, part, &all, &no_sum);
        first[tid] = (int)min(mine, (long)num_blocks);  // (tables that share blocks can hold more than 31 bits count)
        __syncthreads();
        for (int i = tid >> 6; i < run; i += 16)
            if (release[at + i]) {
                int to = top + first[i];
                const int blocks = min(blocks_of(max(seq_lens[at + i], 0), shift), max_blocks);
                for (int j = lane; j - lane < blocks; j += 64) {
                    int *entry = &table[(size_t)(at + i) * max_blocks + (j < blocks ? j : 0)];
                    const int e = j < blocks ? *entry : -1;
                    const bool good = e >= 0 && e < num_blocks;
                    const uint64_t mask = __ballot(good);
                    const int place = to + __popcll(mask & ((1ull << lane) - 1));
                    if (good && place < num_blocks) free_list[place] = e;
                    if (j < blocks) *entry = -1;
                    to += __popcll(mask);
                }
                if (lane == 0) seq_lens[at + i] = 0;
            }
        top = (int)min(top + all, (long)num_blocks);
        __syncthreads();
    }
    if (tid == 0) *free_count = top;
}

// ---- rows -----------------------------------------------------------------------------------

// v over the L lanes of a row (8, 16 or 32), in each of them: DPP moves within 16 lanes, a swap of half rows across.
template <int L, class F>
__device__ __forceinline__ uint32_t row_all(uint32_t v, F f) {
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));   // quad_perm [1,0,3,2]
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));   // quad_perm [2,3,0,1]
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, false));  // row_half_mirror
    if (L >= 16) v = f(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, false));  // row_mirror
    if (L >= 32) v = f(v, (uint32_t)__shfl_xor((int)v, 16));
    return v;
}
struct row_min {
    __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return __builtin_bit_cast(uint32_t, fminf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b))); }
};
struct row_max {
    __device__ uint32_t operator()(uint32_t a, uint32_t b) const { return __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b))); }
};

// Eight channels of a row a lane, D / 8 lanes a row, TWO rows a lane half a workgroup's apart: both rows' loads are on their way before
// anything is known of their slots.  Bound by memory: a row's 4 D bytes in, D / 2 + 4 out; 15 400 tokens of 8 heads of 128 in 34 us
// (4.2 TB/s).
template <int D, bool WIDE>
__global__ __launch_bounds__(256) void kv4_append_kernel(const float *__restrict__ k, const float *__restrict__ v, kv4_view c, size_t token_stride, size_t head_stride,
                                                         int tokens, const int *__restrict__ slots) {
    using R = kv4_rec<D>;
    constexpr int L = D / 8, TWO = 2;
    const int lane = threadIdx.x & (L - 1), i0 = lane * 8;
    float a[TWO][8];
    int slot[TWO], head[TWO], side[TWO];
#pragma unroll
    for (int u = 0; u < TWO; ++u) {
        const unsigned row = (blockIdx.x * TWO + u) * (256 / L) + threadIdx.x / L;  // (a launch has under 2^31 of them)
        side[u] = row & 1;
        const unsigned th = row >> 1, token = th / (unsigned)c.heads;
        head[u] = (int)(th % (unsigned)c.heads);
        const bool there = token < (unsigned)tokens;  // (every lane stays for its row's sums)
        slot[u] = there ? slots[token] : -1;
        const float *x = (side[u] ? v : k) + (size_t)(there ? token : 0) * token_stride + head[u] * head_stride;
        if (WIDE) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i0 + 4 * h < c.head_dim) f = *reinterpret_cast<const float4 *>(x + i0 + 4 * h);
                a[u][4 * h] = f.x, a[u][4 * h + 1] = f.y, a[u][4 * h + 2] = f.z, a[u][4 * h + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) a[u][i] = i0 + i < c.head_dim ? x[i0 + i] : 0.f;
        }
    }
#pragma unroll
    for (int u = 0; u < TWO; ++u) {
        float lo = INFINITY, hi = -INFINITY;
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i0 + i < c.head_dim) {
                lo = fminf(lo, a[u][i]);
                hi = fmaxf(hi, a[u][i]);
                top = max(top, __builtin_bit_cast(uint32_t, a[u][i]) & 0x7fffffffu);  // (of magnitudes the bits are in order, NaN last)
            }
        lo = __builtin_bit_cast(float, row_all<L>(__builtin_bit_cast(uint32_t, lo), row_min{}));
        hi = __builtin_bit_cast(float, row_all<L>(__builtin_bit_cast(uint32_t, hi), row_max{}));
        top = row_all<L>(top, [](uint32_t p, uint32_t q) { return max(p, q); });
        uint32_t zb = __builtin_bit_cast(uint32_t, 0.5f * lo + 0.5f * hi);
        zb = (zb + 0x7fffu + ((zb >> 16) & 1)) & 0xffff0000u;  // to bfloat16, to nearest even
        const float z = __builtin_bit_cast(float, zb);
        const float h = fmaxf(hi - z, z - lo);
        // up to the next bfloat16, so that 7.5 steps reach both ends; not so small that 1 / d is infinite
        const uint32_t db = (__builtin_bit_cast(uint32_t, h * (1.0f / 7.5f)) + 0xffffu) & 0xffff0000u;
        const float d = h == 0.f ? 0.f : fmaxf(__builtin_bit_cast(float, db), 7.52316385e-37f);  // 2^-120
        const float r = h == 0.f ? 0.f : 1.0f / d;
        const bool bad = top >= 0x7f800000u || !(h <= 3.402823466e38f);
        uint32_t codes = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float n = fminf(fmaxf(rintf((a[u][i] - z) * r + 7.5f), 0.f), 15.f);
            codes |= (i0 + i < c.head_dim && !bad ? (uint32_t)n : 0u) << (4 * i);
        }
        if (slot[u] < 0 || (slot[u] >> c.shift) >= c.num_blocks) continue;
        uint8_t *rec = c.data + ((size_t)(slot[u] >> c.shift) * c.heads + head[u]) * R::bytes(c.shift);
        const int at = slot[u] & ((1 << c.shift) - 1);
        *reinterpret_cast<uint32_t *>(rec + (side[u] ? R::v(c.shift) : 0) + (size_t)at * R::ROW + lane * 4) = codes;
        if (lane == 0)
            reinterpret_cast<uint32_t *>(rec + (side[u] ? R::v_meta(c.shift) : R::k_meta(c.shift)))[at] =
                bad ? 0x7fc07fc0u : (zb >> 16) | (__builtin_bit_cast(uint32_t, d) & 0xffff0000u);
    }
}

// The rows of the named slots as the values they stand for; rows of a slot that is none are 0.  Bound by memory: 17 000 tokens of 8
// heads of 128 in 27 us (5.8 TB/s).
template <int D>
__global__ __launch_bounds__(256) void kv4_read_kernel(const int *__restrict__ slots, float *__restrict__ k, kv4_view c, int n, float *__restrict__ v) {
    using R = kv4_rec<D>;
    constexpr int L = D / 8;
    const int lane = threadIdx.x & (L - 1);
    const unsigned row = blockIdx.x * (256 / L) + threadIdx.x / L;  // (a launch has under 2^31 of them)
    const int side = row & 1;
    const unsigned th = row >> 1, token = th / (unsigned)c.heads;
    const int head = (int)(th % (unsigned)c.heads);
    if (token >= (unsigned)n) return;
    const int slot = slots[token];
    const bool live = slot >= 0 && (slot >> c.shift) < c.num_blocks;
    const uint8_t *rec = c.data + ((size_t)(live ? slot >> c.shift : 0) * c.heads + head) * R::bytes(c.shift);
    const int at = live ? slot & ((1 << c.shift) - 1) : 0;
    const uint32_t codes = *reinterpret_cast<const uint32_t *>(rec + (side ? R::v(c.shift) : 0) + (size_t)at * R::ROW + lane * 4);
    const uint32_t meta = reinterpret_cast<const uint32_t *>(rec + (side ? R::v_meta(c.shift) : R::k_meta(c.shift)))[at];
    const float z = kv4_z(meta), d = kv4_d(meta);
    float *out = (side ? v : k) + ((size_t)token * c.heads + head) * c.head_dim;
    float a[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = live ? d * ((float)((codes >> (4 * i)) & 15) - 7.5f) + z : 0.f;
    const int i0 = lane * 8;
    if ((c.head_dim & 3) == 0 && ((uintptr_t)out & 15) == 0) {
        if (i0 < c.head_dim) *reinterpret_cast<float4 *>(out + i0) = make_float4(a[0], a[1], a[2], a[3]);
        if (i0 + 4 < c.head_dim) *reinterpret_cast<float4 *>(out + i0 + 4) = make_float4(a[4], a[5], a[6], a[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i0 + i < c.head_dim) out[i0 + i] = a[i];
    }
}

// The summaries of the blocks that a step's rows lie in: a wavefront an (item, head).  Request b has the items from (its first row
// >> shift) + 2 b on -- its r rows lie in at most (r >> shift) + 2 blocks, so no two requests share one -- and those without a block
// have nothing to do.  A block's least and most are order-independent, so a block that two requests share gets the same bits from both.
template <int D>
__global__ __launch_bounds__(256) void kv4_summarise_kernel(kv4_batch ba, kv4_view c) {
    using R = kv4_rec<D>;
    constexpr int L = D / 8, G = 64 / L;  // lanes a row, rows at a time
    const int item = blockIdx.x, lane = threadIdx.x & (L - 1), group = (threadIdx.x & 63) / L;
    int b = -1;
    kv4_request rq = {0, 0, 0};
    for (int at = 0; at < ba.batch; at += 64) {  // a lane a request, with what it asks, so that nothing of it is loaded again
        const int i = at + (threadIdx.x & 63), j = min(i, ba.batch - 1);
        const int from = ba.starts[j], to = ba.starts[j + 1], len = ba.lens[j];
        const uint64_t upto = __ballot(i < ba.batch && (long)(from >> c.shift) + 2 * i <= item);
        if (!upto) break;
        const int last = 63 - __builtin_clzll(upto);
        b = at + last;
        rq = kv4_request_of(ba, __builtin_amdgcn_readlane(from, last), __builtin_amdgcn_readlane(to, last), __builtin_amdgcn_readlane(len, last), c.shift);
        if (last < 63) break;
    }
    if (rq.rows == 0) return;
    const int bs = 1 << c.shift, first = max(rq.len - rq.rows, 0), block = (first >> c.shift) + item - ((rq.first >> c.shift) + 2 * b);
    if (block < 0 || (long)block << c.shift >= rq.len) return;
    const int phys = ba.table[(size_t)b * ba.max_blocks + block], count = min(bs, rq.len - (block << c.shift));
    if (phys < 0 || phys >= c.num_blocks) return;
    for (int head = blockIdx.y * 4 + (threadIdx.x >> 6); head < c.heads; head += gridDim.y * 4) {
        const size_t at = (size_t)phys * c.heads + head;
        const uint8_t *rec = c.data + at * R::bytes(c.shift);
        const uint32_t *meta = reinterpret_cast<const uint32_t *>(rec + R::k_meta(c.shift));
        float lo[8], hi[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) lo[i] = INFINITY, hi[i] = -INFINITY;
        bool bad = false;
        for (int j0 = group; j0 < count; j0 += 8 * G) {  // eight tokens' loads go out together
            uint32_t codes[8], m[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int j = min(j0 + u * G, count - 1);  // (the last again does no harm)
                codes[u] = *reinterpret_cast<const uint32_t *>(rec + (size_t)j * R::ROW + lane * 4);
                m[u] = meta[j];
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float z = kv4_z(m[u]), d = kv4_d(m[u]);
                bad |= !(d == d);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = d * ((float)((codes[u] >> (4 * i)) & 15) - 7.5f) + z;
                    lo[i] = fminf(lo[i], x);
                    hi[i] = fmaxf(hi[i], x);
                }
            }
        }
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int s = L; s < 64; s <<= 1) {
                lo[i] = fminf(lo[i], __shfl_xor(lo[i], s));
                hi[i] = fmaxf(hi[i], __shfl_xor(hi[i], s));
            }
            if (lane * 8 + i < c.head_dim) most = fmaxf(most, fmaxf(fabsf(lo[i]), fabsf(hi[i])));
        }
        most = over_wave(most, kv4_max{});
        bad = __ballot(bad) != 0;
        const float r = bad || most < 7.88860905e-31f ? 0.f : 1.0f / most * 127.f;  // 2^-100
        uint32_t h4[2] = {0, 0}, l4[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane * 8 + i < c.head_dim && !bad) {
                h4[i >> 2] |= (uint32_t)(uint8_t)(int8_t)rintf(hi[i] * r) << (8 * (i & 3));
                l4[i >> 2] |= (uint32_t)(uint8_t)(int8_t)rintf(lo[i] * r) << (8 * (i & 3));
            }
        uint8_t *s = c.sums + at * R::SUM;
        if (group == 0) {
            *reinterpret_cast<uint2 *>(s + lane * 8) = make_uint2(h4[0], h4[1]);
            *reinterpret_cast<uint2 *>(s + D + lane * 8) = make_uint2(l4[0], l4[1]);
            if (lane == 0) *reinterpret_cast<float *>(s + 2 * D) = bad ? INFINITY : most * (1.0f / 127.f);
        }
    }
}

// Least and most of each channel of the named blocks, as their summaries hold them; 0 where the block is none.  A workgroup a block,
// a wavefront a head at a time.
template <int D>
__global__ __launch_bounds__(256) void kv4_read_sums_kernel(const int *__restrict__ blocks, float *__restrict__ lo, kv4_view c, float *__restrict__ hi) {
    const int phys = blocks[blockIdx.x];
    const bool there = phys >= 0 && phys < c.num_blocks;
    for (int head = threadIdx.x >> 6; head < c.heads; head += 4) {
        const uint8_t *s = c.sums + ((size_t)(there ? phys : 0) * c.heads + head) * kv4_rec<D>::SUM;
        const float scale = there ? *reinterpret_cast<const float *>(s + 2 * D) : 0.f;
        const size_t at = ((size_t)blockIdx.x * c.heads + head) * c.head_dim;
        for (int ch = threadIdx.x & 63; ch < c.head_dim; ch += 64) {
            lo[at + ch] = there ? (float)(int8_t)s[D + ch] * scale : 0.f;
            hi[at + ch] = there ? (float)(int8_t)s[ch] * scale : 0.f;
        }
    }
}

__global__ __launch_bounds__(256) void kv4_clear_kernel(uint4 *p, size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) p[i] = make_uint4(0, 0, 0, 0);
}

constexpr size_t ROWS_A_LAUNCH = 1u << 30;  // rows (token, head, side) of an append or a read-back in one launch: 32 bits count them

int log2_of(size_t v) {
    int s = 0;
    while (((size_t)1 << s) < v) ++s;
    return s;
}

template <class F>
pg_status with_width(int D, F f) {
    if (D == 64) return f(std::integral_constant<int, 64>{});
    if (D == 128) return f(std::integral_constant<int, 128>{});
    return f(std::integral_constant<int, 256>{});
}

pg_status check_tables(const char *fn, size_t batch, size_t block_size, size_t num_blocks, size_t max_blocks) {
    PG_CHECK_ARG(block_size >= 16 && block_size <= 256 && (block_size & (block_size - 1)) == 0,
                 "%s: a block of %zu tokens (16, 32, 64, 128 or 256)", fn, block_size);
    PG_CHECK_ARG(batch < (1u << 24) && num_blocks * block_size < (1ull << 31) && num_blocks < (1ull << 31), "%s: %zu requests, %zu blocks of %zu: out of range", fn, batch,
                 num_blocks, block_size);
    PG_CHECK_ARG(max_blocks > 0 && max_blocks < (1ull << 31) && max_blocks * block_size < (1ull << 31), "%s: tables of %zu blocks: out of range", fn, max_blocks);
    return PG_OK;
}

// A request's tokens as a table on the host holds them: a length within the table, blocks of the pool.
pg_status check_request(const char *fn, size_t b, int32_t len, const int32_t *table, size_t block_size, size_t max_blocks, size_t num_blocks) {
    PG_CHECK_ARG(len >= 0 && (size_t)len <= max_blocks * block_size, "%s: request %zu has %d tokens, its table room for %zu", fn, b, len, max_blocks * block_size);
    const size_t used = ((size_t)len + block_size - 1) / block_size;
    for (size_t j = 0; j < used; ++j)
        PG_CHECK_ARG(table[j] >= 0 && (size_t)table[j] < num_blocks, "%s: request %zu's block %zu is %d of %zu", fn, b, j, table[j], num_blocks);
    return PG_OK;
}

}  // namespace

pg_status pg_kv4_check_step(const char *fn, const pg_paged_kv4 *c, size_t num_q_heads, size_t batch, size_t tokens, size_t max_blocks) {
    PG_CHECK_ARG(c != nullptr, "%s: null cache", fn);
    PG_CHECK_ARG(num_q_heads > 0 && num_q_heads % c->heads == 0 && num_q_heads <= 65535, "%s: %zu query heads over %zu key heads", fn, num_q_heads, c->heads);
    PG_CHECK_ARG(batch <= 65535, "%s: %zu requests (65535 at most)", fn, batch);
    PG_CHECK_ARG(tokens < (1ull << 31) && max_blocks > 0 && max_blocks < (1ull << 31) && max_blocks * c->block_size <= PG_KV4_MAX_TOKENS,
                 "%s: %zu rows, tables of %zu blocks: out of range", fn, tokens, max_blocks);
    return PG_OK;
}

PG_API pg_status pg_block_tables_extend_dev(pg_ctx *ctx, const int32_t *seq_lens_dev, const int32_t *new_lens_dev, size_t batch, size_t block_size,
                                            const int32_t *free_list_dev, const int32_t *free_count_dev, size_t num_blocks, int32_t *block_table_dev, size_t max_blocks,
                                            int32_t *seq_lens_out_dev, int32_t *free_count_out_dev, int32_t *query_start_dev, int32_t *granted_dev, int32_t *slots_dev,
                                            size_t max_tokens) {
    PG_TRY(pg_use(ctx));
    PG_TRY(check_tables("pg_block_tables_extend", batch, block_size, num_blocks, max_blocks));
    PG_CHECK_ARG(max_tokens < (1ull << 31), "pg_block_tables_extend: %zu rows: out of range", max_tokens);
    PG_CHECK_ARG(free_count_dev && free_count_out_dev && query_start_dev && (num_blocks == 0 || free_list_dev) && (max_tokens == 0 || slots_dev) &&
                     (batch == 0 || (seq_lens_dev && new_lens_dev && block_table_dev && seq_lens_out_dev && granted_dev)),
                 "pg_block_tables_extend: null pointer");
    const int shift = log2_of(block_size);
    // One launch, every workgroup with its own sums, unless outputs lie over what the others would still read, or the sums of very
    // many requests are not worth repeating.
    const bool in_place = pg_overlap(seq_lens_dev, batch * 4, seq_lens_out_dev, batch * 4) || free_count_dev == free_count_out_dev;
    const size_t parts = std::max<size_t>(1, (max_tokens + 4095) / 4096);
    const bool here = parts == 1 || (!in_place && batch <= 4096);
    PG_TRY(pg_launch(ctx, "extend_tables_kernel", extend_tables_kernel, dim3((unsigned)(here ? parts : 1)), dim3(1024), 0, seq_lens_dev, new_lens_dev, (int)batch, shift,
                     free_list_dev, free_count_dev, (int)num_blocks, block_table_dev, (int)max_blocks, seq_lens_out_dev, free_count_out_dev, query_start_dev, granted_dev,
                     here ? slots_dev : nullptr, (int)max_tokens));
    if (here) return PG_OK;
    return pg_launch(ctx, "slot_map_kernel", slot_map_kernel, dim3((unsigned)((max_tokens + 255) / 256)), dim3(256), 0, query_start_dev, seq_lens_out_dev,
                     new_lens_dev, (int)batch, shift, block_table_dev, (int)max_blocks, granted_dev, slots_dev, (int)max_tokens, (int)num_blocks);
}

PG_API pg_status pg_block_tables_release_dev(pg_ctx *ctx, const int32_t *release_dev, int32_t *seq_lens_dev, size_t batch, size_t block_size, int32_t *block_table_dev,
                                             size_t max_blocks, int32_t *free_list_dev, int32_t *free_count_dev, size_t num_blocks) {
    PG_TRY(pg_use(ctx));
    PG_TRY(check_tables("pg_block_tables_release", batch, block_size, num_blocks, max_blocks));
    if (batch == 0) return PG_OK;
    PG_CHECK_ARG(release_dev && seq_lens_dev && block_table_dev && free_list_dev && free_count_dev, "pg_block_tables_release: null pointer");
    return pg_launch(ctx, "release_tables_kernel", release_tables_kernel, dim3(1), dim3(1024), 0, release_dev, seq_lens_dev, (int)batch, log2_of(block_size), block_table_dev,
                     (int)max_blocks, free_list_dev, free_count_dev, (int)num_blocks);
}

PG_API pg_status pg_block_tables_extend(pg_ctx *ctx, const int32_t *seq_lens, const int32_t *new_lens, size_t batch, size_t block_size, const int32_t *free_list,
                                        const int32_t *free_count, size_t num_blocks, int32_t *block_table, size_t max_blocks, int32_t *seq_lens_out,
                                        int32_t *free_count_out, int32_t *query_start, int32_t *granted, int32_t *slots, size_t max_tokens) {
    PG_TRY(pg_use(ctx));
    PG_TRY(check_tables("pg_block_tables_extend", batch, block_size, num_blocks, max_blocks));
    PG_CHECK_ARG(max_tokens < (1ull << 31), "pg_block_tables_extend: %zu rows: out of range", max_tokens);
    PG_CHECK_ARG(free_count && free_count_out && query_start && (num_blocks == 0 || free_list) && (max_tokens == 0 || slots) &&
                     (batch == 0 || (seq_lens && new_lens && block_table && seq_lens_out && granted)),
                 "pg_block_tables_extend: null pointer");
    PG_CHECK_ARG(*free_count >= 0 && (size_t)*free_count <= num_blocks, "pg_block_tables_extend: %d free blocks of %zu", *free_count, num_blocks);
    size_t rows = 0;
    for (size_t b = 0; b < batch; ++b) {
        PG_CHECK_ARG(seq_lens[b] >= 0 && new_lens[b] >= 0, "pg_block_tables_extend: request %zu has %d tokens and %d new ones", b, seq_lens[b], new_lens[b]);
        PG_TRY(check_request("pg_block_tables_extend", b, seq_lens[b], block_table + b * max_blocks, block_size, max_blocks, num_blocks));
        rows += (size_t)new_lens[b];
    }
    PG_CHECK_ARG(rows <= max_tokens, "pg_block_tables_extend: %zu new tokens, a slot map of %zu", rows, max_tokens);
    for (int32_t i = 0; i < *free_count; ++i)
        PG_CHECK_ARG(free_list[i] >= 0 && (size_t)free_list[i] < num_blocks, "pg_block_tables_extend: free block %d of %zu", free_list[i], num_blocks);
    const size_t w = sizeof(int32_t);
    pg_dev_block lens, adds, list, count, table, out;
    PG_TRY(pg_host_in(ctx, seq_lens, batch * w, lens));
    PG_TRY(pg_host_in(ctx, new_lens, batch * w, adds));
    PG_TRY(pg_host_in(ctx, free_list, num_blocks * w, list));
    PG_TRY(pg_host_in(ctx, free_count, w, count));
    PG_TRY(pg_host_in(ctx, block_table, batch * max_blocks * w, table));
    const size_t part = pg_round_up(batch + 1, 64);  // (each output begins on a line of its own)
    PG_TRY(out.alloc(ctx, (4 * part + max_tokens) * w));
    int32_t *o = out.as<int32_t>();
    PG_TRY(pg_block_tables_extend_dev(ctx, lens.as<int32_t>(), adds.as<int32_t>(), batch, block_size, list.as<int32_t>(), count.as<int32_t>(), num_blocks,
                                      table.as<int32_t>(), max_blocks, o, o + part, o + 2 * part, o + 3 * part, o + 4 * part, max_tokens));
    PG_TRY(pg_host_out(ctx, block_table, table.p, batch * max_blocks * w));
    PG_TRY(pg_host_out(ctx, seq_lens_out, o, batch * w));
    PG_TRY(pg_host_out(ctx, free_count_out, o + part, w));
    PG_TRY(pg_host_out(ctx, query_start, o + 2 * part, (batch + 1) * w));
    PG_TRY(pg_host_out(ctx, granted, o + 3 * part, batch * w));
    return pg_host_out(ctx, slots, o + 4 * part, max_tokens * w);
}

PG_API pg_status pg_block_tables_release(pg_ctx *ctx, const int32_t *release, int32_t *seq_lens, size_t batch, size_t block_size, int32_t *block_table, size_t max_blocks,
                                         int32_t *free_list, int32_t *free_count, size_t num_blocks) {
    PG_TRY(pg_use(ctx));
    PG_TRY(check_tables("pg_block_tables_release", batch, block_size, num_blocks, max_blocks));
    if (batch == 0) return PG_OK;
    PG_CHECK_ARG(release && seq_lens && block_table && free_list && free_count, "pg_block_tables_release: null pointer");
    PG_CHECK_ARG(*free_count >= 0 && (size_t)*free_count <= num_blocks, "pg_block_tables_release: %d free blocks of %zu", *free_count, num_blocks);
    size_t back = (size_t)*free_count;
    for (size_t b = 0; b < batch; ++b)
        if (release[b]) {
            PG_TRY(check_request("pg_block_tables_release", b, seq_lens[b], block_table + b * max_blocks, block_size, max_blocks, num_blocks));
            back += ((size_t)seq_lens[b] + block_size - 1) / block_size;
        }
    PG_CHECK_ARG(back <= num_blocks, "pg_block_tables_release: %zu free blocks of %zu: one is given back twice", back, num_blocks);
    const size_t w = sizeof(int32_t);
    pg_dev_block flags, lens, table, list, count;
    PG_TRY(pg_host_in(ctx, release, batch * w, flags));
    PG_TRY(pg_host_in(ctx, seq_lens, batch * w, lens));
    PG_TRY(pg_host_in(ctx, block_table, batch * max_blocks * w, table));
    PG_TRY(pg_host_in(ctx, free_list, num_blocks * w, list));
    PG_TRY(pg_host_in(ctx, free_count, w, count));
    PG_TRY(pg_block_tables_release_dev(ctx, flags.as<int32_t>(), lens.as<int32_t>(), batch, block_size, table.as<int32_t>(), max_blocks, list.as<int32_t>(),
                                       count.as<int32_t>(), num_blocks));
    PG_TRY(pg_host_out(ctx, seq_lens, lens.p, batch * w));
    PG_TRY(pg_host_out(ctx, block_table, table.p, batch * max_blocks * w));
    PG_TRY(pg_host_out(ctx, free_list, list.p, num_blocks * w));
    return pg_host_out(ctx, free_count, count.p, w);
}

// ---- the cache ------------------------------------------------------------------------------

PG_API pg_status pg_paged_kv4_create(pg_ctx *ctx, size_t num_blocks, size_t block_size, size_t num_kv_heads, size_t head_dim, pg_paged_kv4 **out) {
    PG_TRY(pg_use(ctx));
    PG_CHECK_ARG(out != nullptr, "pg_paged_kv4_create: null output");
    *out = nullptr;
    PG_TRY(check_tables("pg_paged_kv4_create", 0, block_size, num_blocks, 1));
    PG_CHECK_ARG(num_blocks > 0 && num_kv_heads > 0 && num_kv_heads < 65536 && head_dim > 0 && head_dim <= 256,
                 "pg_paged_kv4_create: %zu blocks, %zu key heads of %zu: out of range (head_dim <= 256)", num_blocks, num_kv_heads, head_dim);
    PG_TRY(pg_refuse_capture(ctx, "pg_paged_kv4_create"));
    pg_paged_kv4 *c = new (std::nothrow) pg_paged_kv4{};
    if (!c) return pg_fail(PG_ENOMEM, "pg_paged_kv4_create: out of host memory");
    c->num_blocks = num_blocks, c->block_size = block_size, c->heads = num_kv_heads, c->head_dim = head_dim;
    c->D = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
    c->device = ctx->device;
    c->shift = log2_of(block_size);
    const size_t records = num_blocks * num_kv_heads, bytes = records * block_size * (c->D + 8), sums = records * (2 * c->D + 16);
    pg_status st = c->mem.alloc(ctx, bytes);
    if (st == PG_OK) st = c->sums_mem.alloc(ctx, sums);
    if (st == PG_OK) {
        c->data = c->mem.as<uint8_t>();
        c->sums = c->sums_mem.as<uint8_t>();
        st = pg_launch(ctx, "kv4_clear_kernel", kv4_clear_kernel, dim3(2048), dim3(256), 0, c->mem.as<uint4>(), bytes / 16);
    }
    if (st == PG_OK) st = pg_launch(ctx, "kv4_clear_kernel", kv4_clear_kernel, dim3(1024), dim3(256), 0, c->sums_mem.as<uint4>(), sums / 16);
    if (st != PG_OK) {
        delete c;
        return st;
    }
    *out = c;
    return PG_OK;
}

PG_API void pg_paged_kv4_free(pg_ctx *ctx, pg_paged_kv4 *c) {
    if (!c) return;
    if (ctx) {
        (void)pg_use(ctx);
        c->touch(ctx);
        if (c->mem.foreign || c->sums_mem.foreign) (void)hipStreamSynchronize(ctx->stream);
    }
    delete c;
}

PG_API pg_status pg_paged_kv4_info(const pg_paged_kv4 *c, size_t *num_blocks, size_t *block_size, size_t *num_kv_heads, size_t *head_dim, size_t *bytes) {
    PG_CHECK_ARG(c != nullptr, "pg_paged_kv4_info: null cache");
    if (num_blocks) *num_blocks = c->num_blocks;
    if (block_size) *block_size = c->block_size;
    if (num_kv_heads) *num_kv_heads = c->heads;
    if (head_dim) *head_dim = c->head_dim;
    if (bytes) *bytes = c->num_blocks * c->heads * (c->block_size * (c->D + 8) + 2 * c->D + 16);
    return PG_OK;
}

PG_API pg_status pg_paged_kv4_append_dev(pg_ctx *ctx, pg_paged_kv4 *c, const float *k_dev, const float *v_dev, size_t token_stride, size_t head_stride, size_t tokens,
                                         const int32_t *slots_dev) {
    PG_TRY(pg_use(ctx));
    PG_CHECK_ARG(c != nullptr, "pg_paged_kv4_append: null cache");
    if (tokens == 0) return PG_OK;
    PG_CHECK_ARG(k_dev && v_dev && slots_dev, "pg_paged_kv4_append: null pointer");
    PG_CHECK_ARG(tokens < (1ull << 31) && token_stride < (1ull << 40) && head_stride < (1ull << 40), "pg_paged_kv4_append: %zu rows: out of range", tokens);
    PG_TRY(c->use("pg_paged_kv4_append", ctx));
    const bool wide = c->head_dim % 4 == 0 && token_stride % 4 == 0 && head_stride % 4 == 0 && (((uintptr_t)k_dev | (uintptr_t)v_dev) & 15) == 0;
    return with_width(c->D, [&](auto w) -> pg_status {
        constexpr int D = decltype(w)::value, PER = 2 * 256 / (D / 8);
        const size_t most = ROWS_A_LAUNCH / (2 * c->heads);  // tokens a launch
        for (size_t at = 0; at < tokens; at += most) {
            const size_t n = std::min(most, tokens - at);
            PG_TRY(pg_launch(ctx, "kv4_append_kernel", wide ? kv4_append_kernel<D, true> : kv4_append_kernel<D, false>, dim3((unsigned)((n * c->heads * 2 + PER - 1) / PER)),
                             dim3(256), 0, k_dev + at * token_stride, v_dev + at * token_stride, kv4_view_of(c), token_stride, head_stride, (int)n, slots_dev + at));
        }
        return PG_OK;
    });
}

PG_API pg_status pg_paged_kv4_read_dev(pg_ctx *ctx, const pg_paged_kv4 *c, const int32_t *slots_dev, size_t n, float *k_dev, float *v_dev) {
    PG_TRY(pg_use(ctx));
    PG_CHECK_ARG(c != nullptr, "pg_paged_kv4_read: null cache");
    if (n == 0) return PG_OK;
    PG_CHECK_ARG(slots_dev && k_dev && v_dev, "pg_paged_kv4_read: null pointer");
    PG_CHECK_ARG(n < (1ull << 31), "pg_paged_kv4_read: %zu rows: out of range", n);
    PG_TRY(c->use("pg_paged_kv4_read", ctx));
    return with_width(c->D, [&](auto w) -> pg_status {
        constexpr int D = decltype(w)::value, PER = 256 / (D / 8);
        const size_t most = ROWS_A_LAUNCH / (2 * c->heads), width = c->heads * c->head_dim;
        for (size_t at = 0; at < n; at += most) {
            const size_t m = std::min(most, n - at);
            PG_TRY(pg_launch(ctx, "kv4_read_kernel", kv4_read_kernel<D>, dim3((unsigned)((m * c->heads * 2 + PER - 1) / PER)), dim3(256), 0, slots_dev + at, k_dev + at * width,
                             kv4_view_of(c), (int)m, v_dev + at * width));
        }
        return PG_OK;
    });
}

PG_API pg_status pg_paged_kv4_summarise_dev(pg_ctx *ctx, pg_paged_kv4 *c, const int32_t *query_start_dev, const int32_t *seq_lens_dev, size_t batch, size_t tokens,
                                            const int32_t *block_table_dev, size_t max_blocks) {
    PG_TRY(pg_use(ctx));
    PG_CHECK_ARG(c != nullptr, "pg_paged_kv4_summarise: null cache");
    PG_TRY(pg_kv4_check_step("pg_paged_kv4_summarise", c, c->heads, batch, tokens, max_blocks));
    if (tokens == 0 || batch == 0) return PG_OK;
    PG_CHECK_ARG(query_start_dev && seq_lens_dev && block_table_dev, "pg_paged_kv4_summarise: null pointer");
    if ((tokens >> c->shift) + 2 * batch >= (1u << 24)) return pg_fail(PG_EUNSUPPORTED, "pg_paged_kv4_summarise: %zu rows are more than a launch takes", tokens);
    PG_TRY(c->use("pg_paged_kv4_summarise", ctx));
    const kv4_batch ba = {query_start_dev, seq_lens_dev, block_table_dev, (int)batch, (int)tokens, (int)max_blocks};
    return with_width(c->D, [&](auto w) -> pg_status {
        return pg_launch(ctx, "kv4_summarise_kernel", kv4_summarise_kernel<decltype(w)::value>, dim3((unsigned)((tokens >> c->shift) + 2 * batch), (unsigned)((c->heads + 3) / 4)),
                         dim3(256), 0, ba,
                         kv4_view_of(c));
    });
}

PG_API pg_status pg_paged_kv4_read_summaries_dev(pg_ctx *ctx, const pg_paged_kv4 *c, const int32_t *blocks_dev, size_t n, float *lo_dev, float *hi_dev) {
    PG_TRY(pg_use(ctx));
    PG_CHECK_ARG(c != nullptr, "pg_paged_kv4_read_summaries: null cache");
    if (n == 0) return PG_OK;
    PG_CHECK_ARG(blocks_dev && lo_dev && hi_dev, "pg_paged_kv4_read_summaries: null pointer");
    PG_CHECK_ARG(n < (1ull << 24), "pg_paged_kv4_read_summaries: %zu blocks: out of range", n);
    PG_TRY(c->use("pg_paged_kv4_read_summaries", ctx));
    return with_width(c->D, [&](auto w) -> pg_status {
        return pg_launch(ctx, "kv4_read_sums_kernel", kv4_read_sums_kernel<decltype(w)::value>, dim3((unsigned)n), dim3(256), 0, blocks_dev, lo_dev, kv4_view_of(c), hi_dev);
    });
}

// ---- host arrays ----------------------------------------------------------------------------

PG_API pg_status pg_paged_kv4_append(pg_ctx *ctx, pg_paged_kv4 *c, const float *k, const float *v, size_t tokens, const int32_t *slots) {
    PG_TRY(pg_use(ctx));
    PG_CHECK_ARG(c != nullptr, "pg_paged_kv4_append: null cache");
    if (tokens == 0) return PG_OK;
    PG_CHECK_ARG(k && v && slots, "pg_paged_kv4_append: null pointer");
    PG_CHECK_ARG(tokens < (1ull << 31), "pg_paged_kv4_append: %zu rows: out of range", tokens);
    std::vector<int32_t> order;
    try {
        order.assign(slots, slots + tokens);
    } catch (const std::bad_alloc &) {
        return pg_fail(PG_ENOMEM, "pg_paged_kv4_append: out of host memory");
    }
    std::sort(order.begin(), order.end());
    for (size_t i = 0; i < tokens; ++i) {
        PG_CHECK_ARG(order[i] >= -1 && order[i] < (int64_t)(c->num_blocks * c->block_size), "pg_paged_kv4_append: slot %d of %zu", order[i], c->num_blocks * c->block_size);
        PG_CHECK_ARG(i == 0 || order[i] == -1 || order[i] != order[i - 1], "pg_paged_kv4_append: slot %d is named twice", order[i]);
    }
    const size_t row = c->heads * c->head_dim, bytes = tokens * row * sizeof(float);
    pg_dev_block dk, dv, ds;
    PG_TRY(pg_host_in(ctx, k, bytes, dk));
    PG_TRY(pg_host_in(ctx, v, bytes, dv));
    PG_TRY(pg_host_in(ctx, slots, tokens * sizeof(int32_t), ds));
    PG_TRY(pg_paged_kv4_append_dev(ctx, c, dk.as<float>(), dv.as<float>(), row, c->head_dim, tokens, ds.as<int32_t>()));
    PG_HIP(hipStreamSynchronize(ctx->stream));
    return PG_OK;
}

PG_API pg_status pg_paged_kv4_read(pg_ctx *ctx, const pg_paged_kv4 *c, const int32_t *slots, size_t n, float *k, float *v) {
    PG_TRY(pg_use(ctx));
    PG_CHECK_ARG(c != nullptr, "pg_paged_kv4_read: null cache");
    if (n == 0) return PG_OK;
    PG_CHECK_ARG(slots && k && v, "pg_paged_kv4_read: null pointer");
    for (size_t i = 0; i < n; ++i)
        PG_CHECK_ARG(slots[i] >= 0 && (size_t)slots[i] < c->num_blocks * c->block_size, "pg_paged_kv4_read: slot %d of %zu", slots[i], c->num_blocks * c->block_size);
    const size_t bytes = n * c->heads * c->head_dim * sizeof(float);
    pg_dev_block ds, dk, dv;
    PG_TRY(pg_host_in(ctx, slots, n * sizeof(int32_t), ds));
    PG_TRY(dk.alloc(ctx, bytes));
    PG_TRY(dv.alloc(ctx, bytes));
    PG_TRY(pg_paged_kv4_read_dev(ctx, c, ds.as<int32_t>(), n, dk.as<float>(), dv.as<float>()));
    PG_TRY(pg_host_out(ctx, k, dk.p, bytes));
    return pg_host_out(ctx, v, dv.p, bytes);
}
