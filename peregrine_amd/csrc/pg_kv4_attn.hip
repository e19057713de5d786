// Attention over the paged cache in 4 bits, and over the blocks of it that a score selects for each query.
//
// With a key row's values z + d (n - 7.5) a score is  d (q . (n - 8)) + (z + d / 2) sum(q):  a product of small whole
// numbers, which the int8 matrix cores do exactly once q is in fixed point (23 bits under its row's largest, as three digits of
// 8), and two FMAs.  With a value row's the output is  sum_t (p_t d_t) (n_t - 7.5) + sum_t p_t z_t:  the f16 matrix cores
// take n - 7.5 as it is and p_t d_t as two f16 (22 bits, ending 2^-34 under the row's largest).  No key or value is
// dequantised; one pass over the rows keeps the running maximum and sum of the softmax.
//
// The lanes' operands come straight from the rows as they lie in memory.  S^T = K Q^T: a lane holds 16 bytes of one of 16
// tokens' keys, (x & 0x0f0f0f0f) and (x >> 4 & 0x0f0f0f0f) are 8 int8 channels in an order that the digits of q share.
// The scores come out with a query row a lane and 4 tokens in it, which is how O^T = V^T P^T takes its probabilities, so
// none crosses a lane.  For V a lane loads 8 tokens' word of 8 channels; the pair of one channel of two tokens is a byte
// permute, a mask and an FMA away.
#include <math.h>
#include <new>
#include "pg_kv4.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float Q_UNITS = 127 * 65536.f;  // the largest of a query row in fixed point
constexpr float P_TOP = 1024.f;          // what a row's largest p d so far is scaled to (over half of it, not all)
constexpr float P_MOST = 32768.f;        // ... and may grow to before the running maximum follows
constexpr float P_SUM = 65536.f;         // what a lane's p of a tile may sum to before it does: sums of p z over 2^20 keys stay finite for values up to 2^90
constexpr float CODE = 1.f / 512.f;      // the value operand is (n - 7.5) / 512: its low codes are f16 subnormals on their way

struct kv4_attn {
    const float *q;
    size_t q_token, q_head;
    kv4_view c;
    kv4_batch ba;
    const int *selected;  // [tokens][heads][top], or null
    int top;
    float scale, cap;
    int mask, window, sinks, group, q_heads, max_query, splits, row_tiles, by_length;
    float *part, *out;
};

// A wavefront's 16 query rows (row = lane & 15) as the B operands of the score products.
template <int D>
struct q_rows {
    static constexpr int NJ = D / 64;
    i32x4 digit[3][NJ];
    int sum_hi2, sum_hi1, sum_lo;  // -8 times the sums of each digit over the row: (n - 8) for n
    float unit, sum;               // value of a unit, sum of the row in units
};

// Over the four lanes of a row (lane & 15).
__device__ __forceinline__ float over_groups(float v) { return over_halves(over_rows(v, kv4_add{}), kv4_add{}); }
__device__ __forceinline__ int over_groups(int v) { return over_halves(over_rows(v, kv4_iadd{}), kv4_iadd{}); }
__device__ __forceinline__ float max_groups(float v) { return over_halves(over_rows(v, kv4_max{}), kv4_max{}); }

// N channels of a query row from channel d on, zeros where there is no row (x null) or channel.  wide: by 16 bytes, for rows that
// are aligned and end at such a word -- every lane has a row or a part of one of its own, so that a load costs by the lines that it
// touches and four times the bytes are nearly free (a wavefront of 32 rows of 128: 64 loads of 4 bytes took 20 us where a CU had
// eight of them).  `some` is read where nothing is, so that no load stands behind a branch.
struct query_rows {
    const float *some;
    int head_dim;
    bool wide;
};
template <int N>
__device__ __forceinline__ void take_channels(const query_rows &qr, const float *x, int d, float *a) {
    if (qr.wide) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const bool there = x && d + i < qr.head_dim;
            const float4 v = *reinterpret_cast<const float4 *>(there ? x + d + i : qr.some);
            a[i] = there ? v.x : 0.f, a[i + 1] = there ? v.y : 0.f, a[i + 2] = there ? v.z : 0.f, a[i + 3] = there ? v.w : 0.f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool there = x && d + i < qr.head_dim;
            const float v = *(there ? x + d + i : qr.some);
            a[i] = there ? v : 0.f;
        }
    }
}
__device__ __forceinline__ query_rows rows_of(const float *q, size_t q_token, size_t q_head, int head_dim) {
    return {q, head_dim, (((uintptr_t)q | q_token * 4 | q_head * 4 | (size_t)head_dim * 4) & 15) == 0};
}

// First channel of the 16 that lane group g holds for the j-th product.
template <int D>
__device__ __forceinline__ constexpr int q_base(int j, int g) {
    return D == 64 ? 16 * g : 128 * (j >> 1) + 32 * g + 16 * (j & 1);
}

// This lane's channels of a query row in fixed point, as words of which byte b is digit b (signed, -128 .. 127), in the order of
// the key operand: even channels of 8, then the odd ones.  x + 0x808080 has the digits plus 128 in its bytes.
template <int D>
struct q_fixed {
    static constexpr int NJ = D / 64;
    int y[NJ][16];
    float unit, sum;  // value of a unit (NaN for a row that is not finite), the row's sum in units
};
// x: the row, or null (zeros).
template <int D>
__device__ __forceinline__ void fix_q(const query_rows &qr, const float *x, int g, q_fixed<D> &r) {
    constexpr int NJ = D / 64;
    float in[NJ][16], a[NJ][16];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NJ; ++j) take_channels<16>(qr, x, q_base<D>(j, g), in[j]);
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            a[j][e] = in[j][8 * (e >> 3) + 2 * (e & 3) + (e >> 2 & 1)];
            top = max(top, __builtin_bit_cast(uint32_t, a[j][e]) & 0x7fffffffu);  // (of magnitudes the bits are in order, NaN last)
        }
    top = over_halves(over_rows(top, kv4_umax{}), kv4_umax{});
    const bool bad = top >= 0x7f800000u;
    const float most = __builtin_bit_cast(float, top);
    const float inv = bad || most < 7.88860905e-31f ? 0.f : Q_UNITS / most;  // under 2^-100: scores of 0
    int sum = 0;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int v = bad ? 0 : (int)rintf(a[j][e] * inv);
            sum += v;
            r.y[j][e] = (v + 0x808080) ^ 0x808080;
        }
    r.unit = bad ? __builtin_nanf("") : most / Q_UNITS;
    r.sum = over_groups((float)sum);
}
// Byte `digit` of four words, in one.
__device__ __forceinline__ int pick_digit(const int *y, uint32_t sel) {  // sel = (4 + digit) << 8 | digit
    const uint32_t lo = __builtin_amdgcn_perm((uint32_t)y[1], (uint32_t)y[0], sel), hi = __builtin_amdgcn_perm((uint32_t)y[3], (uint32_t)y[2], sel);
    return (int)__builtin_amdgcn_perm(hi, lo, 0x05040100u);
}
__device__ __forceinline__ int sum_bytes(int x, int s) { return __builtin_amdgcn_sdot4(x, 0x01010101, s, false); }

template <int D>
__device__ __forceinline__ void load_q(const query_rows &qr, const float *x, int g, q_rows<D> &r) {
    q_fixed<D> f;
    fix_q<D>(qr, x, g, f);
    int s[3] = {0, 0, 0};
#pragma unroll
    for (int j = 0; j < D / 64; ++j)
#pragma unroll
        for (int p = 0; p < 3; ++p)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                r.digit[p][j][w] = pick_digit(&f.y[j][4 * w], 0x0400u + 0x0101u * p);
                s[p] = sum_bytes(r.digit[p][j][w], s[p]);
            }
    r.sum_hi2 = -8 * over_groups(s[2]), r.sum_hi1 = -8 * over_groups(s[1]), r.sum_lo = -8 * over_groups(s[0]);
    r.unit = f.unit;
    r.sum = f.sum;
}

// 32 tokens of one key head as they lie in memory: two runs of 16, each within a block.
template <int D>
struct kv_tile {
    static constexpr int NC = D == 256 ? 2 : 1;
    uint32_t k[2][NC][4];  // (D = 64: two words)
    uint32_t v[2][4][NC];
    uint4 km[2], vm[2];
    int pos[2];  // position of a run's first token; beyond every query where there is none
};

template <int D>
__device__ __forceinline__ void load_tile(const uint8_t *const (&rec)[2], const int (&at)[2], int shift, int lane, kv_tile<D> &t) {
    using R = kv4_rec<D>;
    const int row = lane & 15, g = lane >> 4;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const uint8_t *kp = rec[s] + (size_t)at[s] * R::ROW;
        const uint8_t *vp = kp + R::v(shift);
        const uint32_t ko = row * R::ROW + g * (D == 64 ? 8 : 16);
        if (D == 64) {
            const uint2 x = *reinterpret_cast<const uint2 *>(kp + ko);
            t.k[s][0][0] = x.x, t.k[s][0][1] = x.y, t.k[s][0][2] = t.k[s][0][3] = 0;
        } else {
#pragma unroll
            for (int c = 0; c < kv_tile<D>::NC; ++c) {
                const uint4 x = *reinterpret_cast<const uint4 *>(kp + ko + 64 * c);
                t.k[s][c][0] = x.x, t.k[s][c][1] = x.y, t.k[s][c][2] = x.z, t.k[s][c][3] = x.w;
            }
        }
        const uint32_t vo = 4 * g * R::ROW + (D == 64 ? row >> 1 : row) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < kv_tile<D>::NC; ++c) t.v[s][i][c] = *reinterpret_cast<const uint32_t *>(vp + vo + i * R::ROW + 64 * c);
        t.km[s] = *reinterpret_cast<const uint4 *>(rec[s] + R::k_meta(shift) + 4 * (size_t)at[s] + 16 * g);
        t.vm[s] = *reinterpret_cast<const uint4 *>(rec[s] + R::v_meta(shift) + 4 * (size_t)at[s] + 16 * g);
    }
}

// Lets products of the matrix cores end before accumulators are read behind a loop.  Straight code needs none of it, but where a
// branch stands between a product and its first reader the compiler counts the wait along one of the two ways only, and the
// hardware does not count: so nothing branches between the scores' products and their readers either (masks are without one).
__device__ __forceinline__ void settle_all() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7");
    __builtin_amdgcn_sched_barrier(0);
}

// What a row's p d are scaled by on their way to two f16: P_TOP over the power of two above `peak`, the largest p d that the row has
// seen.  By weight, not by the largest step: the low half ends at 2^-25, which is 2^-34 of the peak, so a large value row takes bits from
// the others only as far as it outweighs them in the output too.  A peak under 2^-118 is taken as that, so that the power is finite.
__device__ __forceinline__ float norm_over(float peak) {
    return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, P_TOP) + (127u << 23) - max((__builtin_bit_cast(uint32_t, peak) & 0x7f800000u) + 0x00800000u, 10u << 23));
}
// 1 / (norm CODE), and f now / before, of such powers of two: by their exponents, so that nothing in between leaves f32's range.
__device__ __forceinline__ float back_from(float norm) { return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, 1.f / CODE) + (127u << 23) - __builtin_bit_cast(uint32_t, norm)); }
__device__ __forceinline__ float rescaled(float f, float now, float before) {
    return __builtin_ldexpf(f, (__builtin_bit_cast(int, now) - __builtin_bit_cast(int, before)) >> 23);
}

// The running softmax of a wavefront's 16 rows: O^T in the accumulators (this lane's row, channels of D / 4 in a run).
template <int D>
struct softmax_rows {
    static constexpr int NV = D / 16;
    f32x4 o[NV];
    float m, l, zsum;  // maximum (log2), sums over this lane's tokens
    bool set;          // whether m is one (the same in a row's four lanes)
    float peak, norm;  // the largest p d seen when the maximum last moved or p d outgrew its scale, and that scale (the same too)
};

__device__ __forceinline__ uint32_t meta_at(const uint4 &m, int i) { return i == 0 ? m.x : i == 1 ? m.y : i == 2 ? m.z : m.w; }

struct row_view {
    int pos;              // this lane's row sees keys up to here (-1: no row)
    int window, sinks;    // and, where window >= 0, from window behind it or below sinks
};

template <int D, bool CAP>
__device__ __forceinline__ void take_tile(bool masked, const kv_tile<D> &t, const q_rows<D> &q, softmax_rows<D> &a, const row_view &rv, float c1, float sq, float cap_log2e, float inv_cap,
                                          int lane) {
    constexpr int NJ = D / 64, NV = D / 16, NC = kv_tile<D>::NC;
    const int g = lane >> 4;
    float s[8], dv[8], zv[8];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        i32x4 hi, lo;
        i32x4 k8[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const uint32_t x = t.k[r][j >> 1][2 * (j & 1)], y = t.k[r][j >> 1][2 * (j & 1) + 1];
            k8[j] = i32x4{(int)(x & 0x0f0f0f0fu), (int)(x >> 4 & 0x0f0f0f0fu), (int)(y & 0x0f0f0f0fu), (int)(y >> 4 & 0x0f0f0f0fu)};
        }
        hi = i32x4{q.sum_hi2, q.sum_hi2, q.sum_hi2, q.sum_hi2};
        lo = i32x4{q.sum_lo, q.sum_lo, q.sum_lo, q.sum_lo};
#pragma unroll
        for (int j = 0; j < NJ; ++j) hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(k8[j], q.digit[2][j], hi, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < NJ; ++j) lo = __builtin_amdgcn_mfma_i32_16x16x64_i8(k8[j], q.digit[0][j], lo, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) hi[i] = (hi[i] << 8) + q.sum_hi1;  // |hi| < 2^26: 256 channels of 15 x 128 x 256 at most
#pragma unroll
        for (int j = 0; j < NJ; ++j) hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(k8[j], q.digit[1][j], hi, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = fmaf((float)hi[i], 256.f, (float)lo[i]);
            const uint32_t km = meta_at(t.km[r], i), vm = meta_at(t.vm[r], i);
            const float d = kv4_d(km), w = fmaf(0.5f, d, kv4_z(km));
            float y;
            if (CAP) y = fmaf(cap_log2e, tanhf(fmaf(d * c1, x, w * sq) * inv_cap), -a.m);
            else y = fmaf(d * c1, x, fmaf(w, sq, -a.m));
            s[4 * r + i] = y;
            zv[4 * r + i] = kv4_z(vm);
            dv[4 * r + i] = kv4_d(vm);
        }
    }
    if (masked)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int key = t.pos[i >> 2] + 4 * g + (i & 3), far = rv.pos - key;
            const bool seen = (far >= 0) & ((rv.window < 0) | (far <= rv.window) | (key < rv.sinks));
            s[i] = seen ? s[i] : -INFINITY;
            zv[i] = seen ? zv[i] : 0.f;  // what is masked may be anything
            dv[i] = seen ? dv[i] : 0.f;
        }
    float p[8], pd[8], sum;
    auto weigh = [&] {
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i] = __builtin_amdgcn_exp2f(s[i]);
            sum += p[i];
            pd[i] = p[i] * dv[i];
        }
    };
    weigh();
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(uint32_t, pd[i] * a.norm));  // (none is negative: the bits are in order, NaN last)
    bool off = top > __builtin_bit_cast(uint32_t, P_MOST) || !(sum < P_SUM);  // (a NaN is off too)
    if (!a.set) off = true;
    {
        if (__ballot(off)) {
            // The slow way: the rows' maxima and scales follow, what was summed is brought to them.
            float at = s[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) at = fmaxf(at, s[i]);
            at = max_groups(at);
            float f = 1.f, shift = 0.f;
            if (at > -INFINITY && (!a.set || at > 0.f)) {
                f = a.set ? __builtin_amdgcn_exp2f(-at) : 1.f;
                shift = at;
                a.m += at;
                a.set = true;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] -= shift;
            weigh();
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) most = fmaxf(most, pd[i]);  // (a NaN is passed over)
            a.peak = fmaxf(a.peak * f, max_groups(most));
            const float norm = norm_over(a.peak), fo = rescaled(f, norm, a.norm);
            a.norm = norm;
            a.l *= f;
            a.zsum *= f;
#pragma unroll
            for (int n = 0; n < NV; ++n) a.o[n] *= fo;
        }
    }
    a.l += sum;
    float zs = 0.f, minus = -1.f;
    asm("" : "+s"(minus));  // (not a subtraction, so that one instruction takes the f16 as it is)
    f16x8 ph, pl;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        zs = fmaf(p[i], zv[i], zs);
        pd[i] *= a.norm;
        ph[i] = (_Float16)pd[i];
    }
    a.zsum += zs;
#pragma unroll
    for (int i = 0; i < 8; ++i) pl[i] = (_Float16)fmaf((float)ph[i], minus, pd[i]);
    // Values: of two tokens' words the byte that holds two channels, beside each other in 16 bits each.
    const f16x2 low_by = {(_Float16)32768.f, (_Float16)32768.f}, high_by = {(_Float16)2048.f, (_Float16)2048.f};
    const f16x2 centre = {(_Float16)(-7.5f * CODE), (_Float16)(-7.5f * CODE)};
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int b = 0; b < (D == 64 ? 2 : 4); ++b) {
            uint32_t sel = 0x0c040c00u + 0x00010001u * b;
            if (D == 64) sel += (lane & 1) ? 0x00020002u : 0u;  // an odd row's channels are in the word's upper half
            f16x8 even, odd;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const uint32_t x = __builtin_amdgcn_perm(t.v[h >> 1][2 * (h & 1) + 1][c], t.v[h >> 1][2 * (h & 1)][c], sel);
                const f16x2 e = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, x & 0x000f000fu), low_by, centre);
                const f16x2 o = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, x & 0x00f000f0u), high_by, centre);
                even[2 * h] = e[0], even[2 * h + 1] = e[1];
                odd[2 * h] = o[0], odd[2 * h + 1] = o[1];
            }
            const int n = (D == 64 ? 0 : 8 * c) + 2 * b;
            a.o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, ph, a.o[n], 0, 0, 0);
            a.o[n + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, ph, a.o[n + 1], 0, 0, 0);
            a.o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, pl, a.o[n], 0, 0, 0);
            a.o[n + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, pl, a.o[n + 1], 0, 0, 0);
        }
}

// The requests in the order of their lengths, the longest first (of equal ones the first): where there are more workgroups than run
// at once, a long request that comes last would have the chip to itself.  128 requests of up to 12000 tokens: 219 instead of 235
// us; a workgroup's own counting, at 256 requests the most, takes half a microsecond.  The whole workgroup of 256 asks.
constexpr int RANKED = 256;
__device__ __forceinline__ int by_length(const kv4_batch &ba, int rank) {
    __shared__ __attribute__((aligned(16))) uint32_t keys[RANKED];
    __shared__ int chosen;
    const int tid = threadIdx.x;
    const uint32_t mine = tid < ba.batch ? (uint32_t)min(max(ba.lens[tid], 0), 0xffffff) << 8 | (uint32_t)(RANKED - 1 - tid) : 0u;
    keys[tid] = mine;
    if (tid == 0) chosen = 0;
    __syncthreads();
    int before = 0;
    for (int j = 0; j < ba.batch; j += 4) {
        const uint4 k = *reinterpret_cast<const uint4 *>(&keys[j]);
        before += (k.x > mine) + (k.y > mine) + (k.z > mine) + (k.w > mine);
    }
    if (tid < ba.batch && before == rank) chosen = tid;
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(chosen);
}

// How many of a list of `top` entries there are to look at: of ascending ones no more than the row has blocks (`own`), but all where
// others are left out ahead of one that counts.  The whole wavefront asks, each for the same answer.
__device__ __forceinline__ int entries_upto(const int *picked, int top, int own, int lane) {
    bool behind = false;
    for (int i = own + lane; i < top; i += 64) behind |= picked[i] >= 0;
    return __ballot(behind) ? top : min(top, own);
}

// One workgroup: 16 query rows of one key head (the rows of a request's tokens and of the head's group, token by token; or
// with SELECTED the group's rows of one token) over one of `splits` runs of their keys, its four wavefronts every fourth
// tile of 32 tokens.
template <int D, bool CAP, bool SELECTED>
__global__ __launch_bounds__(256, D == 64 || (D == 128 && !CAP) ? 3 : 2) void kv4_rows_kernel(kv4_attn A) {
    using R = kv4_rec<D>;
    constexpr int STRIDE = D + 4;
    __shared__ float so[4][16][STRIDE];
    __shared__ float sm[4][16], sl[4][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4;
    unsigned id = blockIdx.x;
    const int split = id % A.splits;
    id /= A.splits;
    const int rt = id % A.row_tiles;
    id /= A.row_tiles;
    const int head = id % A.c.heads;
    const int unit = !SELECTED && A.by_length ? by_length(A.ba, id / A.c.heads) : id / A.c.heads;
    const int shift = A.c.shift, bs = 1 << shift;

    kv4_request rq;
    const int b = SELECTED ? kv4_find(A.ba, unit, shift, rq) : unit;
    if (SELECTED && b < 0) return;
    if (!SELECTED) rq = kv4_request_at(A.ba, b, shift);
    const int tok0 = SELECTED ? unit - rq.first : 0;
    const int rows = SELECTED ? A.group : min(min(rq.rows, A.max_query), A.ba.tokens - rq.first) * A.group;
    const int r0 = rt * 16;
    if (r0 >= rows || (SELECTED && (unsigned)tok0 >= (unsigned)rq.rows)) return;
    const int behind = rq.len - rq.rows;  // position of the request's first row
    auto token_of = [&](int r) { return SELECTED ? tok0 : r / A.group; };
    auto pos_of = [&](int r) { return A.mask == PG_MASK_NONE ? rq.len - 1 : behind + token_of(r); };
    const int r = r0 + (lane & 15), last = min(r0 + 15, rows - 1);
    const bool live = r < rows;
    const int low_pos = pos_of(r0), high_pos = pos_of(last);
    const bool windowed = A.mask == PG_MASK_CAUSAL_SLIDING_WINDOW;
    const row_view rv = {live ? pos_of(r) : -1, windowed ? A.window : -1, A.sinks};

    // The tiles that any row can see.
    int near = 0, sink_tiles = 0, tiles;
    const int *picked = nullptr;
    if (SELECTED) {
        picked = A.selected + ((size_t)unit * A.c.heads + head) * A.top;
        const int blocks = high_pos < 0 ? 0 : entries_upto(picked, A.top, (high_pos >> shift) + 1, lane);
        tiles = (int)((((long)blocks << shift) + 31) >> 5);
    } else {
        const int to = max(high_pos + 1, 0);
        const int from = windowed ? max((long)low_pos - A.window, 0l) : 0;
        near = from >> 5;
        sink_tiles = windowed ? min((int)(((long)A.sinks + 31) >> 5), near) : 0;
        tiles = to > 0 ? sink_tiles + ((to + 31) >> 5) - near : 0;
    }
    const int per = (tiles + A.splits - 1) / A.splits, begin = split * per, end = min(begin + per, tiles);

    const int *table = A.ba.table + (size_t)b * A.ba.max_blocks;
    auto fetch = [&](int tile, kv_tile<D> &t) {
        const uint8_t *rec[2];
        int at[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            int phys = -1, pos = KV4_NOWHERE;
            if (SELECTED) {
                const int v = 32 * tile + 16 * s, e = v >> shift;
                if (e < A.top) {
                    const int block = picked[e], before = e ? picked[e - 1] : -1;
                    if (block > before && block >= 0 && block <= high_pos >> shift) {
                        pos = (block << shift) + (v & (bs - 1));
                        phys = table[block];
                    }
                }
            } else {
                const int p = 32 * (tile < sink_tiles ? tile : tile - sink_tiles + near) + 16 * s;
                if (p <= high_pos) {
                    pos = p;
                    phys = table[p >> shift];
                }
            }
            phys = __builtin_amdgcn_readfirstlane(phys);
            pos = __builtin_amdgcn_readfirstlane(pos);
            if ((unsigned)phys >= (unsigned)A.c.num_blocks) phys = 0, pos = KV4_NOWHERE;
            t.pos[s] = pos;
            at[s] = pos & (bs - 1);
            if (pos == KV4_NOWHERE) at[s] = 0;
            rec[s] = A.c.data + ((size_t)phys * A.c.heads + head) * R::bytes(shift);
        }
        load_tile<D>(rec, at, shift, lane, t);
    };
    kv_tile<D> t;
    int tile = begin + wave;
    if (tile < end) fetch(tile, t);  // on its way while the queries are made ready
    q_rows<D> q;
    load_q<D>(rows_of(A.q, A.q_token, A.q_head, A.c.head_dim), live ? A.q + (size_t)(rq.first + token_of(r)) * A.q_token + (size_t)(head * A.group + (SELECTED ? r : r % A.group)) * A.q_head : nullptr, g, q);
    const float c1 = q.unit * A.scale * (CAP ? 1.f : LOG2E), sq = q.sum * c1;
    const float cap_log2e = CAP ? A.cap * LOG2E : 0.f, inv_cap = CAP ? 1.f / A.cap : 0.f;

    softmax_rows<D> a;
#pragma unroll
    for (int n = 0; n < D / 16; ++n) a.o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    a.m = 0.f, a.l = 0.f, a.zsum = 0.f, a.set = false, a.peak = 0.f, a.norm = norm_over(0.f);

    auto take = [&] {
        const bool whole = max(t.pos[0], t.pos[1]) + 15 <= low_pos && (!windowed || high_pos - min(t.pos[0], t.pos[1]) <= A.window);
        take_tile<D, CAP>(!whole, t, q, a, rv, c1, sq, cap_log2e, inv_cap, lane);
    };
    while (tile < end) {
        take();
        tile += 4;
        if (tile < end) fetch(tile, t);
    }

    settle_all();
    // Four wavefronts' sums into one.
    a.l = over_groups(a.l);
    a.zsum = over_groups(a.zsum);
    const float back = back_from(a.norm);
    constexpr int RUN = D / 4;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
            const int d = D == 256 ? 128 * (n >> 3) + 32 * g + 8 * i + (n & 7) : RUN * g + (D / 16) * i + n;
            so[wave][lane & 15][d] = fmaf(a.o[n][i], back, a.zsum);
        }
    if (g == 0) {
        sm[wave][lane] = a.set ? a.m : a.l == 0.f ? -INFINITY : 0.f;  // (an unset maximum with a sum: NaN scores, which stay)
        sl[wave][lane] = a.l;
    }
    __syncthreads();
    const int row = threadIdx.x >> 4, part = threadIdx.x & 15;
    if (r0 + row >= rows) return;
    float m = fmaxf(fmaxf(sm[0][row], sm[1][row]), fmaxf(sm[2][row], sm[3][row])), w[4], l = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = sm[i][row] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[i][row] - m);
        l += w[i] * sl[i][row];  // (a weight of 0 drops no NaN; where nothing was seen the sums are 0)
    }
    float *out;
    float by = 1.f;
    if (A.splits > 1) {
        float *base = A.part + (size_t)blockIdx.x * (16 * D + 32);
        out = base + row * D;
        if (part == 0) base[16 * D + row] = m, base[16 * D + 16 + row] = l;
    } else {
        const int rr = r0 + row;
        out = A.out + ((size_t)(rq.first + token_of(rr)) * A.q_heads + head * A.group + (SELECTED ? rr : rr % A.group)) * A.c.head_dim;
        by = l == 0.f ? 0.f : 1.f / l;
    }
    const int most = A.splits > 1 ? D : A.c.head_dim;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
        const int d = part + 16 * i;
        float v = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) v += w[j] * so[j][row][d];
        if (d < most) out[d] = v * by;
    }
}

// ---- up to eight rows -----------------------------------------------------------------------
// A decoding step has a group's rows alone (4 or 8 for most models), and 16 columns of scores are mostly padding then: the
// exponentials and everything else that is done by score would be done four times too often.  Here the digits of q are rows
// of one product instead of three products, 64 tokens at a time: S = Q K^T with rows (digit, head) and columns the
// tokens of a run.  A lane then has four heads' scores of one digit, and two swaps between lane halves and two between
// quarters of four runs' results leave it all three digits of one token of its own: 64 tokens x 4 heads are four scores
// a lane.  For O^T = V^T P^T the probabilities cross the lanes once, through LDS, as f16: columns (high half, head), (low
// half, head), so that one product takes both.

template <int D>
struct kv_tile64 {
    static constexpr int NC = D == 256 ? 2 : 1, KW = D == 64 ? 2 : 4;
    uint32_t k[4][NC][KW];
    uint32_t v[4][4][NC];
    uint32_t km[2], vm[2];  // of this lane's tokens
    int pos[4];
};

// Row HB of a wavefront: HB = 4 or 8 heads (rows of the caller), digits of q as rows of A.
template <int D, int HB>
struct q_few {
    static constexpr int NJ = D / 64, SETS = HB == 4 ? 1 : 2;
    i32x4 digit[SETS][NJ];
    i32x4 start[SETS];      // -8 times the sums of the digits: (n - 8) for n
    float unit[4], sum[4];  // of this lane's heads
};

template <int D, int HB>
__device__ __forceinline__ void load_q_few(const query_rows &qr, const float *x, int lane, q_few<D, HB> &r) {
    constexpr int NJ = D / 64, SETS = HB == 4 ? 1 : 2;
    const int g = lane >> 4, row = lane & 15;
    q_fixed<D> f;
    fix_q<D>(qr, x, g, f);
    // HB = 4: rows 0-3 the high digit, 4-7 the middle one, 8-11 the low one, 12-15 nothing
    // HB = 8: rows 0-7 high, 8-15 middle; second set: rows 0-7 low, 8-15 nothing
    const int digit0 = HB == 4 ? 2 - (row >> 2) : 2 - (row >> 3);
    const uint32_t sel0 = digit0 < 0 ? 0x0c0cu : 0x0400u + 0x0101u * (uint32_t)digit0, sel1 = row < 8 ? 0x0400u : 0x0c0cu;
    int s0 = 0, s1 = 0;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            s0 = sum_bytes(r.digit[0][j][w] = pick_digit(&f.y[j][4 * w], sel0), s0);
            if (SETS == 2) s1 = sum_bytes(r.digit[SETS - 1][j][w] = pick_digit(&f.y[j][4 * w], sel1), s1);
        }
    s0 = -8 * over_groups(s0);
    if (SETS == 2) s1 = -8 * over_groups(s1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r.start[0][i] = __shfl(s0, 4 * g + i);
        if (SETS == 2) r.start[SETS - 1][i] = __shfl(s1, 4 * g + i);
        const int from = HB == 4 ? i : 4 * (g & 1) + i;
        r.unit[i] = __shfl(f.unit, from);
        r.sum[i] = __shfl(f.sum, from);
    }
}

// Lanes 32-63 of a with lanes 0-31 of b; lanes 16-31 and 48-63 of a with lanes 0-15 and 32-47 of b.
__device__ __forceinline__ void swap_halves(int &a, int &b) {
    const auto r = __builtin_amdgcn_permlane32_swap((unsigned)a, (unsigned)b, false, false);
    a = (int)r[0], b = (int)r[1];
}
__device__ __forceinline__ void swap_quarters(int &a, int &b) {
    const auto r = __builtin_amdgcn_permlane16_swap((unsigned)a, (unsigned)b, false, false);
    a = (int)r[0], b = (int)r[1];
}

template <int D>
struct softmax_few {
    f32x4 o[D / 16];                  // O^T: this lane's column, channels of D / 4 in a run
    float m[4], l[4], zsum[4];        // of this lane's heads; the sums over this lane's tokens
    bool set[4];
    float peak[4];                    // their largest p d when last looked for (its scale is made again for each tile: registers count)
};

// What lanes of a wavefront wrote to LDS is there for its others.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

constexpr int P_ROW = 72;  // f16 from one row of probabilities to the next: 64 and a shift of four banks

template <int HB, class F>
__device__ __forceinline__ float over_heads(float v, F f) {  // over the lanes that have this lane's heads
    v = over_16(v, f);
    if (HB == 4) v = over_rows(v, f);
    return over_halves(v, f);
}

template <int D, int HB, bool CAP>
__device__ __forceinline__ void take_tile64(bool masked, const kv_tile64<D> &t, const q_few<D, HB> &q, softmax_few<D> &a, const int (&row_pos)[4], int window, int sinks,
                                            const float (&c1)[4], const float (&sq)[4], float cap_log2e, float inv_cap, int lane, _Float16 *pbuf) {
    constexpr int NJ = D / 64, NC = kv_tile64<D>::NC, SETS = HB == 4 ? 1 : 2, NT = HB / 4;  // NT: tokens a lane
    const int g = lane >> 4, c = lane & 15;
    i32x4 acc[SETS][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int s = 0; s < SETS; ++s) acc[s][u] = q.start[s];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const uint32_t x = t.k[u][j >> 1][2 * (j & 1)], y = t.k[u][j >> 1][2 * (j & 1) + 1];
            const i32x4 k8 = {(int)(x & 0x0f0f0f0fu), (int)(x >> 4 & 0x0f0f0f0fu), (int)(y & 0x0f0f0f0fu), (int)(y >> 4 & 0x0f0f0f0fu)};
#pragma unroll
            for (int s = 0; s < SETS; ++s) acc[s][u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(q.digit[s][j], k8, acc[s][u], 0, 0, 0);
        }
    }
    float s[NT][4], dv[NT], zv[NT];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (HB == 4) {
            int x0 = acc[0][0][i], x1 = acc[0][1][i], x2 = acc[0][2][i], x3 = acc[0][3][i];
            swap_halves(x0, x2);
            swap_halves(x1, x3);
            swap_quarters(x0, x1);
            swap_quarters(x2, x3);
            s[0][i] = fmaf((float)((x0 << 8) + x1), 256.f, (float)x2);
        } else {
#pragma unroll
            for (int p = 0; p < NT; ++p) {
                int x0 = acc[0][2 * p][i], x1 = acc[0][2 * p + 1][i], y0 = acc[SETS - 1][2 * p][i], y1 = acc[SETS - 1][2 * p + 1][i];
                swap_halves(x0, x1);
                swap_halves(y0, y1);
                s[p][i] = fmaf((float)((x0 << 8) + x1), 256.f, (float)y0);
            }
        }
    }
#pragma unroll
    for (int p = 0; p < NT; ++p) {
        const float d = kv4_d(t.km[p]), w = fmaf(0.5f, d, kv4_z(t.km[p]));
        zv[p] = kv4_z(t.vm[p]);
        dv[p] = kv4_d(t.vm[p]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (CAP) s[p][i] = fmaf(cap_log2e, tanhf(fmaf(d * c1[i], s[p][i], w * sq[i]) * inv_cap), -a.m[i]);
            else s[p][i] = fmaf(d * c1[i], s[p][i], fmaf(w, sq[i], -a.m[i]));
        }
    }
    if (masked)
#pragma unroll
        for (int p = 0; p < NT; ++p) {
            const int run = HB == 4 ? (g == 0 ? t.pos[0] : g == 1 ? t.pos[1] : g == 2 ? t.pos[2] : t.pos[3]) : (g < 2 ? t.pos[2 * p] : t.pos[2 * p + 1]);
            bool any = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = run + c, far = row_pos[i] - key;
                const bool seen = (far >= 0) & ((window < 0) | (far <= window) | (key < sinks));
                s[p][i] = seen ? s[p][i] : -INFINITY;
                any |= seen;
            }
            zv[p] = any ? zv[p] : 0.f;  // what no row sees may be anything; a row's own mask is on its probability below
            dv[p] = any ? dv[p] : 0.f;
        }
    float pd[NT][4], sum[4], zs[4], total;
    auto weigh_as = [&](auto masked_) {
        constexpr bool MASKED = decltype(masked_)::value;
        total = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sum[i] = zs[i] = 0.f;
#pragma unroll
            for (int p = 0; p < NT; ++p) {
                const float pr = __builtin_amdgcn_exp2f(s[p][i]);
                const bool none = MASKED && s[p][i] == -INFINITY;  // (a token that another row sees may be NaN)
                sum[i] += pr;
                zs[i] = fmaf(pr, none ? 0.f : zv[p], zs[i]);
                pd[p][i] = pr * (none ? 0.f : dv[p]);
            }
            total += sum[i];
        }
    };
    auto weigh = [&] {
        if (masked) weigh_as(std::true_type{});
        else weigh_as(std::false_type{});
    };
    weigh();
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int p = 0; p < NT; ++p) top = max(top, __builtin_bit_cast(uint32_t, pd[p][i] * norm_over(a.peak[i])));  // (none is negative: the bits are in order, NaN last)
    bool off = top > __builtin_bit_cast(uint32_t, P_MOST) || !(total < P_SUM);  // (a NaN is off too)
    off |= !(a.set[0] && a.set[1] && a.set[2] && a.set[3]);
    if (__ballot(off)) {
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float at = s[0][i];
            if (NT == 2) at = fmaxf(at, s[NT - 1][i]);
            at = over_heads<HB>(at, kv4_max{});
            f[i] = 1.f;
            if (at > -INFINITY && (!a.set[i] || at > 0.f)) {
                f[i] = a.set[i] ? __builtin_amdgcn_exp2f(-at) : 1.f;
                a.m[i] += at;
                a.set[i] = true;
#pragma unroll
                for (int p = 0; p < NT; ++p) s[p][i] -= at;
            }
            a.l[i] *= f[i];
            a.zsum[i] *= f[i];
        }
        weigh();
        float fo = 1.f;  // of the column's head, from a lane that has it
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float most = fmaxf(0.f, pd[0][i]);  // (a NaN is passed over)
            if (NT == 2) most = fmaxf(most, pd[NT - 1][i]);
            const float before = norm_over(a.peak[i]);
            a.peak[i] = fmaxf(a.peak[i] * f[i], over_heads<HB>(most, kv4_max{}));
            const float fs = rescaled(f[i], norm_over(a.peak[i]), before);
            const float fi = HB == 4 ? fs : __shfl(fs, 16 * (c >> 2 & 1));
            fo = (c & 3) == i ? fi : fo;
        }
#pragma unroll
        for (int n = 0; n < D / 16; ++n) a.o[n] *= fo;
    }
    float minus = -1.f;
    asm("" : "+s"(minus));  // (not a subtraction, so that one instruction takes the f16 as it is)
    // Probabilities to LDS: row (half, head), the tokens of 32 in the order in which the value operand's lanes have them.
#pragma unroll
    for (int p = 0; p < NT; ++p) {
        const int u = HB == 4 ? g : 2 * p + (g >> 1);
        const int at = 32 * (u >> 1) + 8 * (c >> 2) + 4 * (u & 1) + (c & 3);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int head = HB == 4 ? i : 4 * (g & 1) + i;
            const float x = pd[p][i] * norm_over(a.peak[i]);
            const _Float16 hi = (_Float16)x;
            pbuf[head * P_ROW + at] = hi;
            pbuf[(HB + head) * P_ROW + at] = (_Float16)fmaf((float)hi, minus, x);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) a.l[i] += sum[i], a.zsum[i] += zs[i];
    wave_fence();
    const f16x2 low_by = {(_Float16)32768.f, (_Float16)32768.f}, high_by = {(_Float16)2048.f, (_Float16)2048.f};
    const f16x2 centre = {(_Float16)(-7.5f * CODE), (_Float16)(-7.5f * CODE)};
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const f16x8 ph = *reinterpret_cast<const f16x8 *>(pbuf + (c & (2 * HB - 1)) * P_ROW + 32 * w + 8 * g);
#pragma unroll
        for (int cc = 0; cc < NC; ++cc)
#pragma unroll
            for (int b = 0; b < (D == 64 ? 2 : 4); ++b) {
                uint32_t sel = 0x0c040c00u + 0x00010001u * b;
                if (D == 64) sel += (lane & 1) ? 0x00020002u : 0u;
                f16x8 even, odd;
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const uint32_t x = __builtin_amdgcn_perm(t.v[2 * w + (h >> 1)][2 * (h & 1) + 1][cc], t.v[2 * w + (h >> 1)][2 * (h & 1)][cc], sel);
                    const f16x2 e = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, x & 0x000f000fu), low_by, centre);
                    const f16x2 o = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, x & 0x00f000f0u), high_by, centre);
                    even[2 * h] = e[0], even[2 * h + 1] = e[1];
                    odd[2 * h] = o[0], odd[2 * h + 1] = o[1];
                }
                const int n = (D == 64 ? 0 : 8 * cc) + 2 * b;
                a.o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, ph, a.o[n], 0, 0, 0);
                a.o[n + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, ph, a.o[n + 1], 0, 0, 0);
            }
    }
    __builtin_amdgcn_wave_barrier();
}

// As kv4_rows_kernel, for up to HB rows of a unit: one row tile, wavefronts every fourth tile of 64 tokens.  Bound by memory where
// contexts are long: 128 requests of 7500 tokens, 8 key heads of 128, a group of 4 198 to 200 us (5.2 TB/s; loads alone 5.5, a
// copy 4.8), of 8 201 to 205.  Three workgroups a CU where the registers reach (with 8 rows they do not: 26 spilled, 347 us).
template <int D, int HB, bool CAP, bool SELECTED>
__global__ __launch_bounds__(256, D == 64 || (D == 128 && HB == 4) ? 3 : 2) void kv4_few_kernel(kv4_attn A) {
    using R = kv4_rec<D>;
    constexpr int STRIDE = D + 4;
    __shared__ __attribute__((aligned(16))) char lds[4 * 2 * HB * STRIDE * 4 > 4 * 2 * HB * P_ROW * 2 ? 4 * 2 * HB * STRIDE * 4 : 4 * 2 * HB * P_ROW * 2];
    __shared__ float sm[4][HB], sl[4][HB], sz[4][HB], sback[4][HB];
    // Eight rows of 256 leave no registers for what a tile needs once of each row (factors, position, digits' sums): it waits in LDS, as
    // spilled registers come back behind the tile's own loads.  64 requests of 4000 tokens, 4 key heads: 59 us (75 spilled), capped
    // logits 60 (87).
    constexpr bool LEAN = D == 256 && HB == 8;
    __shared__ __attribute__((aligned(16))) float of_rows[4][3][LEAN ? 2 : 1][4], of_digits[4][2][LEAN ? 4 : 1][4];
    auto so = reinterpret_cast<float(*)[2 * HB][STRIDE]>(lds);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    unsigned id = blockIdx.x;
    const int split = id % A.splits;
    id /= A.splits;
    const int head = id % A.c.heads;
    const int unit = !SELECTED && A.by_length ? by_length(A.ba, id / A.c.heads) : id / A.c.heads;
    const int shift = A.c.shift, bs = 1 << shift;

    kv4_request rq;
    const int b = SELECTED ? kv4_find(A.ba, unit, shift, rq) : unit;
    if (SELECTED && b < 0) return;
    if (!SELECTED) rq = kv4_request_at(A.ba, b, shift);
    const int tok0 = SELECTED ? unit - rq.first : 0;
    const int rows = SELECTED ? A.group : min(min(rq.rows, A.max_query), A.ba.tokens - rq.first) * A.group;
    if (rows <= 0 || (SELECTED && (unsigned)tok0 >= (unsigned)rq.rows)) return;
    const int behind = rq.len - rq.rows;
    auto token_of = [&](int r) { return SELECTED ? tok0 : r / A.group; };
    auto pos_of = [&](int r) { return A.mask == PG_MASK_NONE ? rq.len - 1 : behind + token_of(r); };
    const int low_pos = pos_of(0), high_pos = pos_of(rows - 1);
    const bool windowed = A.mask == PG_MASK_CAUSAL_SLIDING_WINDOW;
    const int window = windowed ? A.window : -1;

    int near = 0, sink_tiles = 0, tiles;
    const int *picked = nullptr;
    if (SELECTED) {
        picked = A.selected + ((size_t)unit * A.c.heads + head) * A.top;
        const int blocks = high_pos < 0 ? 0 : entries_upto(picked, A.top, (high_pos >> shift) + 1, lane);
        tiles = (int)((((long)blocks << shift) + 63) >> 6);
    } else {
        const int to = max(high_pos + 1, 0);
        const int from = windowed ? max((long)low_pos - A.window, 0l) : 0;
        near = from >> 6;
        sink_tiles = windowed ? min((int)(((long)A.sinks + 63) >> 6), near) : 0;
        tiles = to > 0 ? sink_tiles + ((to + 63) >> 6) - near : 0;
    }
    const int per = (tiles + A.splits - 1) / A.splits, begin = split * per, end = min(begin + per, tiles);

    const int *table = A.ba.table + (size_t)b * A.ba.max_blocks;
    auto fetch = [&](int tile, kv_tile64<D> &t) {
        const uint8_t *rec[4];
        int at[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            int phys = -1, pos = KV4_NOWHERE;
            if (SELECTED) {
                const int v = 64 * tile + 16 * u, e = v >> shift;
                if (e < A.top) {
                    const int block = picked[e], before = e ? picked[e - 1] : -1;
                    if (block > before && block >= 0 && block <= high_pos >> shift) {
                        pos = (block << shift) + (v & (bs - 1));
                        phys = table[block];
                    }
                }
            } else {
                const int p = 64 * (tile < sink_tiles ? tile : tile - sink_tiles + near) + 16 * u;
                if (p <= high_pos) {
                    pos = p;
                    phys = table[p >> shift];
                }
            }
            phys = __builtin_amdgcn_readfirstlane(phys);
            pos = __builtin_amdgcn_readfirstlane(pos);
            if ((unsigned)phys >= (unsigned)A.c.num_blocks) phys = 0, pos = KV4_NOWHERE;
            t.pos[u] = pos;
            at[u] = pos == KV4_NOWHERE ? 0 : pos & (bs - 1);
            rec[u] = A.c.data + ((size_t)phys * A.c.heads + head) * R::bytes(shift);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint8_t *kp = rec[u] + (size_t)at[u] * R::ROW, *vp = kp + R::v(shift);
            const uint32_t ko = c * R::ROW + g * (D == 64 ? 8 : 16);
#pragma unroll
            for (int cc = 0; cc < kv_tile64<D>::NC; ++cc) {
                if (D == 64) {
                    const uint2 x = *reinterpret_cast<const uint2 *>(kp + ko);
                    t.k[u][cc][0] = x.x, t.k[u][cc][1] = x.y;
                } else {
                    const uint4 x = *reinterpret_cast<const uint4 *>(kp + ko + 64 * cc);
                    t.k[u][cc][0] = x.x, t.k[u][cc][1] = x.y, t.k[u][cc][kv_tile64<D>::KW - 2] = x.z, t.k[u][cc][kv_tile64<D>::KW - 1] = x.w;
                }
            }
            const uint32_t vo = 4 * g * R::ROW + (D == 64 ? c >> 1 : c) * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int cc = 0; cc < kv_tile64<D>::NC; ++cc) t.v[u][i][cc] = *reinterpret_cast<const uint32_t *>(vp + vo + i * R::ROW + 64 * cc);
        }
#pragma unroll
        for (int p = 0; p < HB / 4; ++p) {
            // this lane's token: HB = 4 of run g, HB = 8 of run 2 p + (g >> 1)
            const uint8_t *r0 = HB == 4 ? (g < 2 ? (g == 0 ? rec[0] : rec[1]) : (g == 2 ? rec[2] : rec[3])) : (g < 2 ? rec[2 * p] : rec[2 * p + 1]);
            const int a0 = HB == 4 ? (g < 2 ? (g == 0 ? at[0] : at[1]) : (g == 2 ? at[2] : at[3])) : (g < 2 ? at[2 * p] : at[2 * p + 1]);
            const uint32_t *mp = reinterpret_cast<const uint32_t *>(r0 + R::k_meta(shift)) + a0 + c;
            t.km[p] = mp[0];
            t.vm[p] = mp[(size_t)1 << shift];
        }
    };
    kv_tile64<D> t;
    int tile = begin + wave;
    if (tile < end) fetch(tile, t);  // on its way while the queries are made ready
    q_few<D, HB> q;
    float c1[4], sq[4];
    int row_pos[4];
    {
        const int r = HB == 4 ? c & 3 : c & 7;
        load_q_few<D, HB>(rows_of(A.q, A.q_token, A.q_head, A.c.head_dim), r < rows ? A.q + (size_t)(rq.first + token_of(r)) * A.q_token + (size_t)(head * A.group + (SELECTED ? r : r % A.group)) * A.q_head : nullptr,
                          lane, q);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int mine = HB == 4 ? i : 4 * (g & 1) + i;
            c1[i] = q.unit[i] * A.scale * (CAP ? 1.f : LOG2E);
            sq[i] = q.sum[i] * c1[i];
            row_pos[i] = mine < rows ? pos_of(mine) : -1;
        }
    }
    if (LEAN && c == 0 && g < HB / 4) {
        *reinterpret_cast<f32x4 *>(of_rows[wave][0][g]) = f32x4{c1[0], c1[1], c1[2], c1[3]};
        *reinterpret_cast<f32x4 *>(of_rows[wave][1][g]) = f32x4{sq[0], sq[1], sq[2], sq[3]};
        *reinterpret_cast<i32x4 *>(of_rows[wave][2][g]) = i32x4{row_pos[0], row_pos[1], row_pos[2], row_pos[3]};
    }
    if (LEAN && c == 0)
#pragma unroll
        for (int k = 0; k < 2; ++k) *reinterpret_cast<i32x4 *>(of_digits[wave][k][g]) = q.start[k * (q_few<D, HB>::SETS - 1)];
    wave_fence();
    const float cap_log2e = CAP ? A.cap * LOG2E : 0.f, inv_cap = CAP ? 1.f / A.cap : 0.f;

    softmax_few<D> a;
#pragma unroll
    for (int n = 0; n < D / 16; ++n) a.o[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) a.m[i] = a.l[i] = a.zsum[i] = a.peak[i] = 0.f, a.set[i] = false;
    _Float16 *pbuf = reinterpret_cast<_Float16 *>(lds) + wave * 2 * HB * P_ROW;

    auto take = [&] {
        if constexpr (LEAN) {
#pragma unroll
            for (int k = 0; k < 2; ++k) q.start[k] = *reinterpret_cast<const i32x4 *>(of_digits[wave][k][g]);
            const f32x4 x = *reinterpret_cast<const f32x4 *>(of_rows[wave][0][g & 1]), y = *reinterpret_cast<const f32x4 *>(of_rows[wave][1][g & 1]);
            const i32x4 p = *reinterpret_cast<const i32x4 *>(of_rows[wave][2][g & 1]);
#pragma unroll
            for (int i = 0; i < 4; ++i) c1[i] = x[i], sq[i] = y[i], row_pos[i] = p[i];
        }
        const int far = max(max(t.pos[0], t.pos[1]), max(t.pos[2], t.pos[3])), close = min(min(t.pos[0], t.pos[1]), min(t.pos[2], t.pos[3]));
        const bool whole = far + 15 <= low_pos && (!windowed || high_pos - close <= A.window);
        take_tile64<D, HB, CAP>(!whole, t, q, a, row_pos, window, A.sinks, c1, sq, cap_log2e, inv_cap, lane, pbuf);
    };
    while (tile < end) {
        take();
        tile += 4;
        if (tile < end) fetch(tile, t);
    }

    settle_all();
    // Four wavefronts' sums, and each column's two halves, into one.
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a.l[i] = over_heads<HB>(a.l[i], kv4_add{});
        a.zsum[i] = over_heads<HB>(a.zsum[i], kv4_add{});
    }
    __syncthreads();  // (the probabilities' memory is the sums')
    constexpr int RUN = D / 4;
    if (c < 2 * HB)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int n = 0; n < D / 16; ++n) {
                const int d = D == 256 ? 128 * (n >> 3) + 32 * g + 8 * i + (n & 7) : RUN * g + (D / 16) * i + n;
                so[wave][c][d] = a.o[n][i];
            }
    if (c == 0 && g < HB / 4)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int h = 4 * g + i;
            sm[wave][h] = a.set[i] ? a.m[i] : a.l[i] == 0.f ? -INFINITY : 0.f;
            sl[wave][h] = a.l[i];
            sz[wave][h] = a.zsum[i];
            sback[wave][h] = back_from(norm_over(a.peak[i]));
        }
    __syncthreads();
    constexpr int TPR = 256 / HB;
    const int row = threadIdx.x / TPR, part = threadIdx.x % TPR;
    if (row >= rows) return;
    float m = fmaxf(fmaxf(sm[0][row], sm[1][row]), fmaxf(sm[2][row], sm[3][row])), w[4], l = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = sm[i][row] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[i][row] - m);
        l += w[i] * sl[i][row];  // (a weight of 0 drops no NaN; where nothing was seen the sums are 0)
    }
    float *out;
    float by = 1.f;
    if (A.splits > 1) {
        float *base = A.part + (size_t)blockIdx.x * (HB * D + 32);
        out = base + row * D;
        if (part == 0) base[HB * D + row] = m, base[HB * D + 16 + row] = l;
    } else {
        out = A.out + ((size_t)(rq.first + token_of(row)) * A.q_heads + head * A.group + (SELECTED ? row : row % A.group)) * A.c.head_dim;
        by = l == 0.f ? 0.f : 1.f / l;
    }
    const int most = A.splits > 1 ? D : A.c.head_dim;
#pragma unroll
    for (int i = 0; i < D / TPR; ++i) {
        const int d = part + TPR * i;
        float v = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) v += w[j] * fmaf(so[j][row][d] + so[j][HB + row][d], sback[j][row], sz[j][row]);
        if (d < most) out[d] = v * by;
    }
}

// ---- prompts --------------------------------------------------------------------------------
// With many rows the keys' and values' way from codes to operands is what 16 rows at a time would pay for again and again.
// Here a workgroup has eight wavefronts of 16 rows and makes the operands of 64 tokens once, in LDS, in the order in
// which the lanes take them (four wavefronts the keys', four the values'); the next 64 tokens' codes are on their way meanwhile, and the
// two buffers take turns, one barrier a tile.  Scores and probabilities as in kv4_rows_kernel.  What bounds it is the arithmetic on
// scores: about 17 instructions for each of 16 x 64 beside 112 products of the matrix cores.  Heads of 256: the last 2048 rows of 8192, 16
// heads, 470 us (512 TFLOP/s of one product each).
template <int D>
struct prompt_lds {
    static constexpr int K = 64 * D, V = 128 * D;  // bytes of a tile's operands
    alignas(16) uint8_t k[2][K];
    alignas(16) uint8_t v[2][V];
    alignas(16) float meta[2][4][64];  // key step, key z + d / 2, value step, value z
};

template <bool CAP>
__global__ __launch_bounds__(512, 2) void kv4_prompt_kernel(kv4_attn A) {
    constexpr int D = 256, NW = 8, NJ = D / 64, NV = D / 16, NC = 2;
    using R = kv4_rec<D>;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_raw[];
    auto &lds = *reinterpret_cast<prompt_lds<D> *>(lds_raw);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    // The heads next to each other: workgroups go to the XCDs in turn, and a head's rows share its keys in one L2.  The last rows,
    // which see the most keys, first.
    unsigned id = blockIdx.x;
    const int head = id % A.c.heads;
    id /= A.c.heads;
    const int split = id % A.splits;
    id /= A.splits;
    const int groups = (A.row_tiles + NW - 1) / NW;
    const int group = groups - 1 - id % groups;
    const int b = id / groups;
    const int shift = A.c.shift, bs = 1 << shift;
    const kv4_request rq = kv4_request_at(A.ba, b, shift);
    const int rows = min(min(rq.rows, A.max_query), A.ba.tokens - rq.first) * A.group;
    const int r0 = group * 16 * NW;
    if (r0 >= rows) return;
    const int behind = rq.len - rq.rows;
    auto pos_of = [&](int r) { return A.mask == PG_MASK_NONE ? rq.len - 1 : behind + r / A.group; };
    const int mine = r0 + wave * 16;  // this wavefront's first row
    const int last_row = min(r0 + 16 * NW, rows) - 1, my_last = min(mine + 16, rows) - 1;
    const int group_low = pos_of(r0), group_high = pos_of(last_row);
    const int low_pos = pos_of(min(mine, last_row)), high_pos = mine < rows ? pos_of(my_last) : -1;
    const bool windowed = A.mask == PG_MASK_CAUSAL_SLIDING_WINDOW;
    const int window = windowed ? A.window : -1;
    const int to = max(group_high + 1, 0), from = windowed ? (int)max((long)group_low - A.window, 0l) : 0;
    const int near = from >> 6, sink_tiles = windowed ? min((int)(((long)A.sinks + 63) >> 6), near) : 0;
    const int tiles = to > 0 ? sink_tiles + ((to + 63) >> 6) - near : 0;
    const int per = (tiles + A.splits - 1) / A.splits, begin = split * per, end = min(begin + per, tiles);

    // A tile's codes on their way to LDS: a thread has one token's chunk of keys (4 threads a token), and words of values
    // for one half of the tile and one half of each word's channels.
    struct {
        uint4 k[NC];
        uint32_t v[8][NC], km, vm;
    } st;
    const int *table = A.ba.table + (size_t)b * A.ba.max_blocks;
    auto first_of = [&](int tile) { return 64 * (tile < sink_tiles ? tile : tile - sink_tiles + near); };
    auto rec_of = [&](int run, int tile, int &at) {  // record and place of a run of 16 tokens (some block where there is none)
        const int p = first_of(tile) + 16 * run;
        int phys = p <= group_high ? table[p >> shift] : -1;
        at = p & (bs - 1);
        if ((unsigned)phys >= (unsigned)A.c.num_blocks) phys = 0;
        return A.c.data + ((size_t)phys * A.c.heads + head) * R::bytes(shift);
    };
    const int k_token = tid >> 2, k_chunk = tid & 3, v_half = wave & 1, v_part = wave >> 1 & 1;
    const bool does_k = wave < 4;
    auto fetch = [&](int tile) {
        if (does_k) {
            int at;
            // (the wavefront's keys are one run: tokens 16 wave .. 16 wave + 15)
            const uint8_t *rec = rec_of(wave, tile, at);
            const uint8_t *kp = rec + (size_t)(at + (k_token & 15)) * R::ROW + k_chunk * 16;
#pragma unroll
            for (int cc = 0; cc < NC; ++cc) st.k[cc] = *reinterpret_cast<const uint4 *>(kp + 64 * cc);
            if (lane < 16) {
                st.km = reinterpret_cast<const uint32_t *>(rec + R::k_meta(shift))[at + lane];
                st.vm = reinterpret_cast<const uint32_t *>(rec + R::v_meta(shift))[at + lane];
            }
            return;
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            int va;
            const uint8_t *vp = rec_of(2 * v_half + r, tile, va);
            vp += R::v(shift) + (size_t)(va + 4 * g) * R::ROW + c * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int cc = 0; cc < NC; ++cc) st.v[4 * r + i][cc] = *reinterpret_cast<const uint32_t *>(vp + i * R::ROW + 64 * cc);
        }
    };
    auto store = [&](int buf) {
        if (does_k) {
            // keys: product j of a run, lanes (chunk, token) in the order of the operand
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const uint32_t x = j & 1 ? st.k[j >> 1].z : st.k[j >> 1].x, y = j & 1 ? st.k[j >> 1].w : st.k[j >> 1].y;
                *reinterpret_cast<i32x4 *>(&lds.k[buf][((wave * NJ + j) * 64 + 16 * k_chunk + (k_token & 15)) * 16]) =
                    i32x4{(int)(x & 0x0f0f0f0fu), (int)(x >> 4 & 0x0f0f0f0fu), (int)(y & 0x0f0f0f0fu), (int)(y >> 4 & 0x0f0f0f0fu)};
            }
            if (lane < 16) {
                const float d = kv4_d(st.km);
                lds.meta[buf][0][16 * wave + lane] = d;
                lds.meta[buf][1][16 * wave + lane] = fmaf(0.5f, d, kv4_z(st.km));
                lds.meta[buf][2][16 * wave + lane] = kv4_d(st.vm);
                lds.meta[buf][3][16 * wave + lane] = kv4_z(st.vm);
            }
            return;
        }
        const f16x2 low_by = {(_Float16)32768.f, (_Float16)32768.f}, high_by = {(_Float16)2048.f, (_Float16)2048.f};
        const f16x2 centre = {(_Float16)(-7.5f * CODE), (_Float16)(-7.5f * CODE)};
#pragma unroll
        for (int cc = 0; cc < NC; ++cc)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int b2 = 2 * v_part + q;
                const uint32_t sel = 0x0c040c00u + 0x00010001u * b2;
                f16x8 even, odd;
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const uint32_t x = __builtin_amdgcn_perm(st.v[2 * h + 1][cc], st.v[2 * h][cc], sel);
                    const f16x2 e = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, x & 0x000f000fu), low_by, centre);
                    const f16x2 o = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, x & 0x00f000f0u), high_by, centre);
                    even[2 * h] = e[0], even[2 * h + 1] = e[1];
                    odd[2 * h] = o[0], odd[2 * h + 1] = o[1];
                }
                const int n = 8 * cc + 2 * b2;
                *reinterpret_cast<f16x8 *>(&lds.v[buf][((v_half * NV + n) * 64 + lane) * 16]) = even;
                *reinterpret_cast<f16x8 *>(&lds.v[buf][((v_half * NV + n + 1) * 64 + lane) * 16]) = odd;
            }
    };
    if (begin < end) fetch(begin);

    q_rows<D> q;
    const int r = mine + c;
    const bool live = r < rows;
    load_q<D>(rows_of(A.q, A.q_token, A.q_head, A.c.head_dim), live ? A.q + (size_t)(rq.first + r / A.group) * A.q_token + (size_t)(head * A.group + r % A.group) * A.q_head : nullptr, g, q);
    const float c1 = q.unit * A.scale * (CAP ? 1.f : LOG2E);
    const float sq = q.sum * c1;
    const int row_pos = live ? pos_of(r) : -1;
    const float cap_log2e = CAP ? A.cap * LOG2E : 0.f, inv_cap = CAP ? 1.f / A.cap : 0.f;
    f32x4 o[NV];
    float m = 0.f, l = 0.f, zsum = 0.f, peak = 0.f, norm = norm_over(0.f);
    bool set = false;
#pragma unroll
    for (int n = 0; n < NV; ++n) o[n] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto take = [&](bool masked, const int (&run_pos)[4], int buf) {
#pragma unroll 1
        for (int w = 0; w < 2; ++w) {
            const int pos0 = w ? run_pos[2] : run_pos[0], pos1 = w ? run_pos[3] : run_pos[1];
            float s[8], dv[8], zv[8];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int run = 2 * w + r;
                i32x4 k8[NJ];
#pragma unroll
                for (int j = 0; j < NJ; ++j) k8[j] = *reinterpret_cast<const i32x4 *>(&lds.k[buf][((run * NJ + j) * 64 + lane) * 16]);
                const f32x4 kd = *reinterpret_cast<const f32x4 *>(&lds.meta[buf][0][16 * run + 4 * g]), kw = *reinterpret_cast<const f32x4 *>(&lds.meta[buf][1][16 * run + 4 * g]);
                const f32x4 vd = *reinterpret_cast<const f32x4 *>(&lds.meta[buf][2][16 * run + 4 * g]), vz = *reinterpret_cast<const f32x4 *>(&lds.meta[buf][3][16 * run + 4 * g]);
                i32x4 hi = {q.sum_hi2, q.sum_hi2, q.sum_hi2, q.sum_hi2}, lo = {q.sum_lo, q.sum_lo, q.sum_lo, q.sum_lo};
#pragma unroll
                for (int j = 0; j < NJ; ++j) hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(k8[j], q.digit[2][j], hi, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < NJ; ++j) lo = __builtin_amdgcn_mfma_i32_16x16x64_i8(k8[j], q.digit[0][j], lo, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) hi[i] = (hi[i] << 8) + q.sum_hi1;
#pragma unroll
                for (int j = 0; j < NJ; ++j) hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(k8[j], q.digit[1][j], hi, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = fmaf((float)hi[i], 256.f, (float)lo[i]);
                    float y;
                    if (CAP) y = fmaf(cap_log2e, tanhf(fmaf(kd[i] * c1, x, kw[i] * sq) * inv_cap), -m);
                    else y = fmaf(kd[i] * c1, x, fmaf(kw[i], sq, -m));
                    s[4 * r + i] = y;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) dv[4 * r + i] = vd[i], zv[4 * r + i] = vz[i];
            }
            if (masked) {
                // What lies behind the rows' last position, or in no block, may be anything, and so may masked tokens.
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int key = (i < 4 ? pos0 : pos1) + 4 * g + (i & 3), far = row_pos - key;
                    const bool seen = (far >= 0) & ((window < 0) | (far <= window) | (key < A.sinks));
                    s[i] = seen ? s[i] : -INFINITY;
                    dv[i] = seen ? dv[i] : 0.f;
                    zv[i] = seen ? zv[i] : 0.f;
                }
            }
            float p[8], pd[8], sum;
            auto weigh = [&] {
                sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    p[i] = __builtin_amdgcn_exp2f(s[i]);
                    sum += p[i];
                    pd[i] = p[i] * dv[i];
                }
            };
            weigh();
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(uint32_t, pd[i] * norm));
            const bool off = !set || top > __builtin_bit_cast(uint32_t, P_MOST) || !(sum < P_SUM);
            if (__ballot(off)) {
                float at = s[0];
#pragma unroll
                for (int i = 1; i < 8; ++i) at = fmaxf(at, s[i]);
                at = max_groups(at);
                float f = 1.f;
                if (at > -INFINITY && (!set || at > 0.f)) {
                    f = set ? __builtin_amdgcn_exp2f(-at) : 1.f;
                    m += at;
                    set = true;
#pragma unroll
                    for (int i = 0; i < 8; ++i) s[i] -= at;
                }
                l *= f;
                zsum *= f;
                weigh();
                float most = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) most = fmaxf(most, pd[i]);  // (a NaN is passed over)
                peak = fmaxf(peak * f, max_groups(most));
                const float next = norm_over(peak), fo = rescaled(f, next, norm);
                norm = next;
#pragma unroll
                for (int n = 0; n < NV; ++n) o[n] *= fo;
            }
            f16x8 ph, pl;
            float minus = -1.f;
            asm("" : "+s"(minus));  // (not a subtraction, so that one instruction takes the f16 as it is)
            l += sum;
            float zs = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                zs = fmaf(p[i], zv[i], zs);
                pd[i] *= norm;
                ph[i] = (_Float16)pd[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) pl[i] = (_Float16)fmaf((float)ph[i], minus, pd[i]);
            zsum += zs;
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const f16x8 v = *reinterpret_cast<const f16x8 *>(&lds.v[buf][((w * NV + n) * 64 + lane) * 16]);
                o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph, o[n], 0, 0, 0);
                o[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl, o[n], 0, 0, 0);
            }
        }
    };
    if (begin < end) store(0);
    __syncthreads();
    for (int tile = begin; tile < end; ++tile) {
        const int buf = (tile - begin) & 1, first = first_of(tile);
        if (tile + 1 < end) fetch(tile + 1);
        if (first <= high_pos) {
            int run_pos[4];  // of each run's first token, beyond every row where the run lies in no block
            bool there = true;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int p = first + 16 * r;
                const bool ok = (p <= group_high) & ((unsigned)table[min(p, group_high) >> shift] < (unsigned)A.c.num_blocks);
                run_pos[r] = ok ? p : KV4_NOWHERE;
                there &= ok;
            }
            take(!there || first + 63 > low_pos || (windowed && high_pos - first > window), run_pos, buf);
        }
        if (tile + 1 < end) store(buf ^ 1);
        __syncthreads();
    }

    settle_all();
    const float back = back_from(norm);
    const float ls = over_groups(l), zs = over_groups(zsum);
    if (r >= rows) return;
    float *out;
    float by = 1.f;
    if (A.splits > 1) {
        const size_t tile = ((size_t)b * A.c.heads + head) * A.row_tiles + r / 16;
        float *base = A.part + (tile * A.splits + split) * (16 * D + 32);
        out = base + c * D;
        if (g == 0) base[16 * D + c] = set ? m : ls == 0.f ? -INFINITY : 0.f, base[16 * D + 16 + c] = ls;
    } else {
        out = A.out + ((size_t)(rq.first + r / A.group) * A.q_heads + head * A.group + r % A.group) * A.c.head_dim;
        by = ls == 0.f ? 0.f : 1.f / ls;
    }
    const int most = A.splits > 1 ? D : A.c.head_dim;
    const bool wide = (most & 3) == 0 && ((uintptr_t)out & 15) == 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < NV; n += 4) {
            const int d = 128 * (n >> 3) + 32 * g + 8 * i + (n & 7);
            const float4 y = make_float4(fmaf(o[n][i], back, zs) * by, fmaf(o[n + 1][i], back, zs) * by, fmaf(o[n + 2][i], back, zs) * by, fmaf(o[n + 3][i], back, zs) * by);
            if (wide) {
                if (d < most) *reinterpret_cast<float4 *>(out + d) = y;
            } else {
                if (d < most) out[d] = y.x;
                if (d + 1 < most) out[d + 1] = y.y;
                if (d + 2 < most) out[d + 2] = y.z;
                if (d + 3 < most) out[d + 3] = y.w;
            }
        }
}

// The same for heads up to 128 on 32 x 32 products: a wavefront has 32 rows, so each operand that it takes from LDS serves twice the
// rows.  Keys go through the f16 matrix cores too, against q as two f16 (scaled by a power of two to 512 .. 1024 at the row's
// largest): two more products a step than with three int8 digits on half the depth, and four instructions a score less, of
// which there are 16 a lane.  Lanes and operands: A and B of a product hold 8 values of its 16 deep side, row or column lane & 31;
// a result's registers i are rows (i & 3) + 8 (i >> 2) + 4 (lane >> 5), which makes the probabilities of registers 8 s .. 8 s + 7
// the B operand of step s once the values' tokens stand in that order.  2048 rows at 16384, 32 heads of 128: 1095 us (471 TFLOP/s of one
// product each, twice that executed); vector instructions 51 %, matrix products 40 % of the cycles, which do not overlap much better.
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int D>
struct prompt32_lds {
    static constexpr int K = 128 * D, V = 128 * D;  // bytes of 64 tokens' operands
    alignas(16) uint8_t k[2][K];
    alignas(16) uint8_t v[2][V];
    alignas(16) float meta[2][4][64];  // key step, key centre, value step, value centre
};

template <int D, bool CAP>
__global__ __launch_bounds__(256, 2) void kv4_prompt32_kernel(kv4_attn A) {
    using R = kv4_rec<D>;
    constexpr int KS = D / 16, DT = D / 32, W = D / 8, KW = D / 32;  // steps of a score, tiles of channels, words of a row, words a lane stages
    extern __shared__ __attribute__((aligned(16))) uint8_t lds_raw[];
    auto &lds = *reinterpret_cast<prompt32_lds<D> *>(lds_raw);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, c = lane & 31;
    // The heads next to each other: workgroups go to the XCDs in turn, and a head's rows share its keys in one L2.  The last rows,
    // which see the most keys, first.
    unsigned id = blockIdx.x;
    const int head = id % A.c.heads;
    id /= A.c.heads;
    const int split = id % A.splits;
    id /= A.splits;
    const int groups = (A.row_tiles + 7) / 8;
    const int group = groups - 1 - id % groups;
    const int b = id / groups;
    const int shift = A.c.shift, bs = 1 << shift;
    const kv4_request rq = kv4_request_at(A.ba, b, shift);
    const int rows = min(min(rq.rows, A.max_query), A.ba.tokens - rq.first) * A.group;
    const int r0 = group * 128;
    if (r0 >= rows) return;
    const int behind = rq.len - rq.rows;
    auto pos_of = [&](int r) { return A.mask == PG_MASK_NONE ? rq.len - 1 : behind + r / A.group; };
    const int mine = r0 + wave * 32, last_row = min(r0 + 128, rows) - 1;
    const int group_low = pos_of(r0), group_high = pos_of(last_row);
    const int low_pos = pos_of(min(mine, last_row)), high_pos = mine < rows ? pos_of(min(mine + 32, rows) - 1) : -1;
    const bool windowed = A.mask == PG_MASK_CAUSAL_SLIDING_WINDOW;
    const int window = windowed ? A.window : -1;
    const int to = max(group_high + 1, 0), from = windowed ? (int)max((long)group_low - A.window, 0l) : 0;
    const int near = from >> 6, sink_tiles = windowed ? min((int)(((long)A.sinks + 63) >> 6), near) : 0;
    const int tiles = to > 0 ? sink_tiles + ((to + 63) >> 6) - near : 0;
    const int per = (tiles + A.splits - 1) / A.splits, begin = split * per, end = min(begin + per, tiles);

    const int *table = A.ba.table + (size_t)b * A.ba.max_blocks;
    auto first_of = [&](int tile) { return 64 * (tile < sink_tiles ? tile : tile - sink_tiles + near); };
    // A tile on its way: the blocks of its four runs first (a tile ahead of the codes), then its codes in registers -- a lane has one
    // token's chunk of keys, and words of eight tokens' values, those of run `wave` in the order that the products take them.
    int phys[4], run_pos[4], next_pos[4];
    auto look = [&](int tile) {
        const int first = first_of(tile);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int p = first + 16 * r;
            phys[r] = table[min(p, group_high) >> shift];
            if (p > group_high) phys[r] = -1;
        }
    };
    uint32_t ck[KW], cv[8], cm = 0;
    auto fetch = [&](int tile) {
        const int first = first_of(tile);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const bool ok = (unsigned)phys[r] < (unsigned)A.c.num_blocks;
            next_pos[r] = ok ? first + 16 * r : KV4_NOWHERE;
            phys[r] = ok ? phys[r] : 0;
        }
        const int of_lane = lane < 32 ? (lane < 16 ? phys[0] : phys[1]) : (lane < 48 ? phys[2] : phys[3]);
        const int at = (first + lane) & (bs - 1);
        const uint8_t *rec = A.c.data + ((size_t)of_lane * A.c.heads + head) * R::bytes(shift);
        const uint8_t *kp = rec + (uint32_t)(at * R::ROW) + wave * (4 * KW);
        if (D == 64) {
            const uint2 x = *reinterpret_cast<const uint2 *>(kp);
            ck[0] = x.x, ck[1] = x.y;
        } else {
            const uint4 x = *reinterpret_cast<const uint4 *>(kp);
            ck[0] = x.x, ck[1] = x.y, ck[KW - 2] = x.z, ck[KW - 1] = x.w;
        }
        if (wave < 2) cm = reinterpret_cast<const uint32_t *>(rec + (wave ? R::v_meta(shift) : R::k_meta(shift)))[at];
        const int my_phys = wave < 2 ? (wave == 0 ? phys[0] : phys[1]) : (wave == 2 ? phys[2] : phys[3]);
        const uint8_t *vp = A.c.data + ((size_t)my_phys * A.c.heads + head) * R::bytes(shift) + R::v(shift) + (size_t)((first + 16 * wave) & (bs - 1)) * R::ROW;
        const uint32_t vo = 4 * half * R::ROW + (c & (W - 1)) * 4;
#pragma unroll
        for (int e = 0; e < 8; ++e) cv[e] = *reinterpret_cast<const uint32_t *>(vp + vo + ((e & 3) + 8 * (e >> 2)) * R::ROW);
    };
    const f16x2 low_by = {(_Float16)32768.f, (_Float16)32768.f}, high_by = {(_Float16)2048.f, (_Float16)2048.f};
    const f16x2 centre = {(_Float16)(-7.5f * CODE), (_Float16)(-7.5f * CODE)};
    const bool upper = c / W & 1;  // which of a byte's channels this lane's rows of values are
    const uint32_t v_mask = upper ? 0x00f000f0u : 0x000f000fu;
    const f16x2 v_by = upper ? high_by : low_by;
    auto store = [&](int buf) {
#pragma unroll
        for (int i = 0; i < KW; ++i) {
            const int word = KW * wave + i;
            const uint32_t x = ck[i], y = x >> 8;
            const f16x2 p0 = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, x & 0x000f000fu), low_by, centre);
            const f16x2 p1 = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, x & 0x00f000f0u), high_by, centre);
            const f16x2 p2 = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, y & 0x000f000fu), low_by, centre);
            const f16x2 p3 = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, y & 0x00f000f0u), high_by, centre);
            *reinterpret_cast<f16x8 *>(&lds.k[buf][((half * KS + (word >> 1)) * 64 + c + 32 * (word & 1)) * 16]) = f16x8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
        }
        if (wave < 2) {
            lds.meta[buf][2 * wave][lane] = kv4_d(cm);
            lds.meta[buf][2 * wave + 1][lane] = kv4_z(cm);
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            uint32_t sel = 0x0c040c00u + 0x00010001u * (D == 64 ? 2 * dt : dt);
            if (D == 64) sel += 0x00010001u * (c >> 4);
            f16x8 x;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const f16x2 y = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, __builtin_amdgcn_perm(cv[2 * h + 1], cv[2 * h], sel) & v_mask), v_by, centre);
                x[2 * h] = y[0], x[2 * h + 1] = y[1];
            }
            *reinterpret_cast<f16x8 *>(&lds.v[buf][((wave * DT + dt) * 64 + lane) * 16]) = x;
        }
    };
    if (begin < end) {
        look(begin);
        fetch(begin);
        look(min(begin + 1, end - 1));
    }

    // The rows: lane (row c, half) has channels 8 (2 step + half) .. + 7 in the keys' order.
    f16x8 qh[KS], ql[KS];
    float c1, sq;
    const int r = mine + c;
    const bool live = r < rows;
    {
        const float *x = live ? A.q + (size_t)(rq.first + r / A.group) * A.q_token + (size_t)(head * A.group + r % A.group) * A.q_head : nullptr;
        const query_rows qr = rows_of(A.q, A.q_token, A.q_head, A.c.head_dim);
        float in[KS][8], a[KS][8], sum = 0.f;
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < KS; ++k) take_channels<8>(qr, x, 8 * (2 * k + half), in[k]);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                a[k][e] = in[k][(e >> 1) + 4 * (e & 1)];
                top = max(top, __builtin_bit_cast(uint32_t, a[k][e]) & 0x7fffffffu);
            }
        top = over_halves(top, kv4_umax{});
        const bool bad = top >= 0x7f800000u, none = bad || top < 0x0d800000u;  // 2^-100: scores of 0
        // to 512 .. 1024 (1 / CODE, which the keys' operands are short of) by a power of two: 2^109 .. 2^-118 for 2^-100 .. 2^127
        const uint32_t exponent = none ? 127u << 23 : top & 0x7f800000u;
        const float by = none ? 0.f : __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, 1.f / CODE) + (127u << 23) - exponent), back = __builtin_bit_cast(float, exponent);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = bad ? 0.f : a[k][e] * by;
                sum += y;
                qh[k][e] = (_Float16)y;
                ql[k][e] = (_Float16)(y - (float)qh[k][e]);
            }
        sum = over_halves(sum, kv4_add{});
        const float unit = bad ? __builtin_nanf("") : back * A.scale * (CAP ? 1.f : LOG2E);
        c1 = unit;
        sq = sum * CODE * unit;
    }
    const int row_pos = live ? pos_of(r) : -1;
    const float cap_log2e = CAP ? A.cap * LOG2E : 0.f, inv_cap = CAP ? 1.f / A.cap : 0.f;
    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
    float m = 0.f, l = 0.f, zsum = 0.f, peak = 0.f, norm = norm_over(0.f);
    bool set = false;

    auto take = [&](bool masked, int buf) {
#pragma unroll 1
        for (int w = 0; w < 2; ++w) {
            const int pos0 = w ? run_pos[2] : run_pos[0], pos1 = w ? run_pos[3] : run_pos[1];
            f32x16 x;
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = 0.f;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const f16x8 key = *reinterpret_cast<const f16x8 *>(&lds.k[buf][((w * KS + k) * 64 + lane) * 16]);
                x = __builtin_amdgcn_mfma_f32_32x32x16_f16(key, qh[k], x, 0, 0, 0);
                x = __builtin_amdgcn_mfma_f32_32x32x16_f16(key, ql[k], x, 0, 0, 0);
            }
            float s[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x4 kd = *reinterpret_cast<const f32x4 *>(&lds.meta[buf][0][32 * w + 8 * j + 4 * half]), kz = *reinterpret_cast<const f32x4 *>(&lds.meta[buf][1][32 * w + 8 * j + 4 * half]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float y;
                    if (CAP) y = fmaf(cap_log2e, tanhf(fmaf(kd[i] * c1, x[4 * j + i], kz[i] * sq) * inv_cap), -m);
                    else y = fmaf(kd[i] * c1, x[4 * j + i], fmaf(kz[i], sq, -m));
                    s[4 * j + i] = y;
                }
            }
            if (masked)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = (i < 8 ? pos0 : pos1) + 8 * (i >> 2 & 1) + 4 * half + (i & 3), far = row_pos - key;
                    s[i] = (far >= 0) & ((window < 0) | (far <= window) | (key < A.sinks)) ? s[i] : -INFINITY;
                }
            float pd[16], sum, zs;
            uint32_t top;
            auto weigh_as = [&](auto masked_) {
                constexpr bool MASKED = decltype(masked_)::value;
                sum = zs = 0.f;
                top = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x4 vd = *reinterpret_cast<const f32x4 *>(&lds.meta[buf][2][32 * w + 8 * j + 4 * half]), vz = *reinterpret_cast<const f32x4 *>(&lds.meta[buf][3][32 * w + 8 * j + 4 * half]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float y = s[4 * j + i], p = __builtin_amdgcn_exp2f(y);
                        const bool none = MASKED && y == -INFINITY;  // (what is masked may be anything)
                        const float d = none ? 0.f : vd[i], z = none ? 0.f : vz[i];
                        sum += p;
                        zs = fmaf(p, z, zs);
                        pd[4 * j + i] = p * d * norm;
                        top = max(top, __builtin_bit_cast(uint32_t, pd[4 * j + i]));
                    }
                }
            };
            auto weigh = [&] {
                if (masked) weigh_as(std::true_type{});
                else weigh_as(std::false_type{});
            };
            weigh();
            if (__ballot(!set || top > __builtin_bit_cast(uint32_t, P_MOST) || !(sum < P_SUM))) {
                float at = s[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) at = fmaxf(at, s[i]);
                at = over_halves(at, kv4_max{});
                float f = 1.f;
                if (at > -INFINITY && (!set || at > 0.f)) {
                    f = set ? __builtin_amdgcn_exp2f(-at) : 1.f;
                    m += at;
                    set = true;
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] -= at;
                }
                l *= f;
                zsum *= f;
                float most = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x4 vd = *reinterpret_cast<const f32x4 *>(&lds.meta[buf][2][32 * w + 8 * j + 4 * half]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) most = fmaxf(most, __builtin_amdgcn_exp2f(s[4 * j + i]) * vd[i]);  // (a NaN is passed over: masked ones are 0)
                }
                peak = fmaxf(peak * f, over_halves(most, kv4_max{}));
                const float next = norm_over(peak), fo = rescaled(f, next, norm);
                norm = next;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[dt] *= fo;
                weigh();
            }
            l += sum;
            zsum += zs;
            float minus = -1.f;
            asm("" : "+s"(minus));  // (not a subtraction, so that one instruction takes the f16 as it is)
            f16x8 ph[2], pl[2];
#pragma unroll
            for (int i = 0; i < 16; ++i) ph[i >> 3][i & 7] = (_Float16)pd[i];
#pragma unroll
            for (int i = 0; i < 16; ++i) pl[i >> 3][i & 7] = (_Float16)fmaf((float)ph[i >> 3][i & 7], minus, pd[i]);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const f16x8 v = *reinterpret_cast<const f16x8 *>(&lds.v[buf][(((2 * w + t) * DT + dt) * 64 + lane) * 16]);
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph[t], o[dt], 0, 0, 0);
                    o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl[t], o[dt], 0, 0, 0);
                }
        }
    };
    if (begin < end) store(0);
    __syncthreads();
    for (int tile = begin; tile < end; ++tile) {
        const int buf = (tile - begin) & 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) run_pos[i] = next_pos[i];
        if (tile + 1 < end) {
            fetch(tile + 1);
            look(min(tile + 2, end - 1));
        }
        const int far = max(max(run_pos[0], run_pos[1]), max(run_pos[2], run_pos[3])), close = min(min(run_pos[0], run_pos[1]), min(run_pos[2], run_pos[3]));
        if (close <= high_pos) take(far + 15 > low_pos || (windowed && high_pos - close > window), buf);
        if (tile + 1 < end) store(buf ^ 1);
        __syncthreads();
    }

    settle_all();
    l = over_halves(l, kv4_add{});
    zsum = over_halves(zsum, kv4_add{});
    if (!live) return;
    const float back = back_from(norm);
    float *out;
    float by = 1.f;
    if (A.splits > 1) {
        const size_t tile = ((size_t)b * A.c.heads + head) * A.row_tiles + r / 16;
        float *base = A.part + (tile * A.splits + split) * (16 * D + 32);
        out = base + (r & 15) * D;
        if (half == 0) base[16 * D + (r & 15)] = set ? m : l == 0.f ? -INFINITY : 0.f, base[16 * D + 16 + (r & 15)] = l;
    } else {
        out = A.out + ((size_t)(rq.first + r / A.group) * A.q_heads + head * A.group + r % A.group) * A.c.head_dim;
        by = l == 0.f ? 0.f : 1.f / l;
    }
    const int most = A.splits > 1 ? D : A.c.head_dim;
    const bool wide = (most & 3) == 0 && ((uintptr_t)out & 15) == 0;
    auto put = [&](int d, float x0, float x1, float x2, float x3) {
        const float4 y = make_float4(fmaf(x0, back, zsum) * by, fmaf(x1, back, zsum) * by, fmaf(x2, back, zsum) * by, fmaf(x3, back, zsum) * by);
        if (wide) {
            if (d < most) *reinterpret_cast<float4 *>(out + d) = y;
        } else {
            if (d < most) out[d] = y.x;
            if (d + 1 < most) out[d + 1] = y.y;
            if (d + 2 < most) out[d + 2] = y.z;
            if (d + 3 < most) out[d + 3] = y.w;
        }
    };
    // Row rho = a + 8 j + 4 half of a tile is word rho % W of a row of values, and of the word's channels the one that `store` chose.
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        if constexpr (D == 64) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) put(8 * (a + 4 * half) + 4 * dt, o[dt][a], o[dt][4 + a], o[dt][8 + a], o[dt][12 + a]);
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int dt = 0; dt < DT; dt += 2) put(8 * (a + 8 * j + 4 * half) + 2 * dt, o[dt][4 * j + a], o[dt][4 * (j + 2) + a], o[dt + 1][4 * j + a], o[dt + 1][4 * (j + 2) + a]);
        }
    }
}

// The splits of a row into its output, in their order: a wavefront a row, `RT` rows a tile.  The splits' weights first, a lane a
// split, so that the loop over their rows waits for nothing but its loads.
template <int D, int RT, bool SELECTED>
__global__ __launch_bounds__(256) void kv4_join_kernel(kv4_attn A) {
    constexpr size_t NEXT = RT * D + 32;
    const int lane = threadIdx.x & 63;
    const unsigned id = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int row = id % RT;
    unsigned tile = id / RT;
    const size_t first = (size_t)tile * A.splits;
    const int rt = tile % A.row_tiles;
    tile /= A.row_tiles;
    const int head = tile % A.c.heads, unit = tile / A.c.heads;
    kv4_request rq;
    const int b = SELECTED ? kv4_find(A.ba, unit, A.c.shift, rq) : unit;
    if (b < 0 || b >= A.ba.batch) return;
    if (!SELECTED) rq = kv4_request_at(A.ba, b, A.c.shift);
    const int rows = SELECTED ? A.group : min(min(rq.rows, A.max_query), A.ba.tokens - rq.first) * A.group, r = rt * RT + row;
    if (r >= rows || (SELECTED && (unsigned)(unit - rq.first) >= (unsigned)rq.rows)) return;
    const int token = SELECTED ? unit : rq.first + r / A.group;
    const float *part = A.part + first * NEXT;
    float m = -INFINITY;
    for (int s = lane; s < A.splits; s += 64) m = fmaxf(m, part[s * NEXT + RT * D + row]);
    m = over_wave(m, kv4_max{});
    float l = 0.f, o[D / 64];
#pragma unroll
    for (int i = 0; i < D / 64; ++i) o[i] = 0.f;
    for (int s0 = 0; s0 < A.splits; s0 += 64) {
        const int s = s0 + lane, n = min(64, A.splits - s0);
        const float ms = s < A.splits ? part[s * NEXT + RT * D + row] : -INFINITY;
        const float w = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - m);
        float mine = s < A.splits ? w * part[s * NEXT + RT * D + 16 + row] : 0.f;
        mine = over_wave(mine, kv4_add{});
        l += mine;
        const float *rows_at = part + s0 * NEXT + row * D + lane;
        auto add = [&](int j, const float (&x)[D / 64]) {
            const float wj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), j));
#pragma unroll
            for (int i = 0; i < D / 64; ++i) o[i] += wj * x[i];  // (a weight of 0 drops no NaN; a run that saw nothing holds zeros)
        };
        int j = 0;
        for (; j + 8 <= n; j += 8) {  // eight splits' rows on their way at once
            float x[8][D / 64];
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int i = 0; i < D / 64; ++i) x[u][i] = rows_at[(j + u) * NEXT + 64 * i];
#pragma unroll
            for (int u = 0; u < 8; ++u) add(j + u, x[u]);
        }
        for (; j < n; ++j) {
            float x[D / 64];
#pragma unroll
            for (int i = 0; i < D / 64; ++i) x[i] = rows_at[j * NEXT + 64 * i];
            add(j, x);
        }
    }
    const float by = l == 0.f ? 0.f : 1.f / l;
    float *out = A.out + ((size_t)token * A.q_heads + head * A.group + (SELECTED ? r : r % A.group)) * A.c.head_dim;
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
        if (64 * i + lane < A.c.head_dim) out[64 * i + lane] = o[i] * by;
}

// ---- selection ------------------------------------------------------------------------------

struct kv4_pick {
    const float *q;
    size_t q_token, q_head;
    kv4_view c;
    kv4_batch ba;
    int group, top, first, recent;
    int *selected;
};

// Blocks in the order of their scores as whole numbers: a larger key is a larger score.
__device__ __forceinline__ uint32_t score_key(float s) {
    const uint32_t u = __builtin_bit_cast(uint32_t, s + 0.f);  // -0 counts as 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// 16 query rows as the operands of the scores' products (rows of the product are x where positive and x where negative), with the
// values of the units of this lane's four rows of a result.
template <int D>
struct pick_rows {
    i32x4 pos8[D / 64], neg8[D / 64];
    float unit[4];
};
template <int D>
__device__ __forceinline__ void round_rows(const float (&a)[D / 64][16], int g, pick_rows<D> &r) {
    constexpr int NJ = D / 64;
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = max(top, __builtin_bit_cast(uint32_t, a[j][e]) & 0x7fffffffu);  // (of magnitudes the bits are in order, NaN last)
    top = over_halves(over_rows(top, kv4_umax{}), kv4_umax{});
    const bool bad = top >= 0x7f800000u;
    const float most = __builtin_bit_cast(float, top);
    const float by = bad || most < 7.88860905e-31f ? 0.f : 1.0f / most * 127.f;  // 2^-100
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            uint32_t up = 0, down = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int v = bad ? 0 : (int)rintf(a[j][4 * w + e] * by);
                up |= (uint32_t)(max(v, 0) & 255) << (8 * e);
                down |= (uint32_t)(min(v, 0) & 255) << (8 * e);
            }
            r.pos8[j][w] = (int)up;
            r.neg8[j][w] = (int)down;
        }
    // a lane's four rows of the result are rows 4 g + i
#pragma unroll
    for (int i = 0; i < 4; ++i) r.unit[i] = __shfl(bad ? 0.f : most * (1.0f / 127.f), 4 * g + i);
}
// This lane's part of a block's summary.
template <int D>
struct pick_block {
    i32x4 hi[D / 64], lo[D / 64];
    float scale;  // -1 (a mark: no scale is negative) where there is no block
};
template <int D>
__device__ __forceinline__ void load_summary(const kv4_view &c, int phys, int head, int g, pick_block<D> &s) {
    using R = kv4_rec<D>;
    const bool there = (unsigned)phys < (unsigned)c.num_blocks;
    const uint8_t *at = c.sums + ((size_t)(there ? phys : 0) * c.heads + head) * R::SUM;
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
        s.hi[j] = *reinterpret_cast<const i32x4 *>(at + 64 * j + 16 * g);
        s.lo[j] = *reinterpret_cast<const i32x4 *>(at + D + 64 * j + 16 * g);
    }
    s.scale = *reinterpret_cast<const float *>(at + 2 * D);
    if (!there) s.scale = -1.f;
}
// Scores of this lane's four rows: whole numbers and two f32 products.
template <int D>
__device__ __forceinline__ void score_rows(const pick_rows<D> &r, const pick_block<D> &s, float (&score)[4]) {
    i32x4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(r.pos8[j], s.hi[j], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(r.neg8[j], s.lo[j], acc, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) score[i] = ((float)acc[i] * r.unit[i]) * s.scale;
}
// ... of a block that is to be taken by itself: a key that is not finite is not to be missed, no block never taken.
__device__ __forceinline__ float score_of(float score, float scale) { return scale == INFINITY ? INFINITY : scale < 0.f ? -INFINITY : score; }

// Of 256 bins, from the top: the one in which the want-th entry lies, and its number in that bin.  (Four bins a lane.)
__device__ __forceinline__ void bin_of(const uint32_t *bins, uint32_t want, int lane, uint32_t &bin, uint32_t &left) {
    uint32_t h[4], mine = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[i] = bins[255 - 4 * lane - i];
        mine += h[i];
    }
    uint32_t upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t u = __shfl_up(upto, d);
        if (lane >= d) upto += u;
    }
    uint32_t over = upto - mine, at = 0, rest = 0;
    bool here = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (over < want && over + h[i] >= want) here = true, at = 255 - 4 * lane - i, rest = want - over;
        over += h[i];
    }
    const int who = __builtin_ctzll(__ballot(here));
    bin = (uint32_t)__builtin_amdgcn_readlane((int)at, who);
    left = (uint32_t)__builtin_amdgcn_readlane((int)rest, who);
}
// One workgroup: one query token and key head.  Scores of 16 blocks a wavefront at a time -- rows of the product are the
// group's query rows (x where positive, x where negative), columns the blocks (hi, lo), whole numbers throughout, and two
// f32 products a score.  Then the key that exactly as many blocks reach as are wanted: passes of 8 bits over a histogram in LDS,
// from the highest bit in which the keys differ, every wavefront with its own sums over the bins, so a pass is one barrier.  Then
// the blocks over that key, and of those at it the first, in ascending order.  It is a chain of latencies (request, table,
// summaries, passes): several tiles' loads go out together, queries ahead of everything.  8 rows of 8 key heads over 1024 blocks
// 20 us: 64 workgroups of 1024 threads, each bound by what one CU loads (about 20 GB/s).
template <int D, int T>
__global__ __launch_bounds__(T) void kv4_select_kernel(kv4_pick A) {
    constexpr int NJ = D / 64, W = T / 64, U = T == 256 || D == 256 ? 1 : 4;  // U: tiles of 16 blocks whose loads go out together (few wavefronts: all that they have; many: registers count)
    extern __shared__ uint32_t keys[];  // [blocks]
    __shared__ uint32_t hist[4][256], least, most_key;
    __shared__ int above[W], at_key[W];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = lane & 15, g = lane >> 4, tid = threadIdx.x;
    const int token = blockIdx.x / (unsigned)A.c.heads, head = blockIdx.x % (unsigned)A.c.heads, shift = A.c.shift;
    for (int i = tid; i < 1024; i += T) hist[i >> 8][i & 255] = 0;
    if (tid == 0) least = 0xffffffffu, most_key = 0;
    float a[NJ][16];
    const query_rows qr = rows_of(A.q, A.q_token, A.q_head, A.c.head_dim);
    auto load_rows = [&](int r0) {
        const float *x = r0 + row < A.group ? A.q + (size_t)token * A.q_token + (size_t)(head * A.group + r0 + row) * A.q_head : nullptr;
#pragma unroll
        for (int j = 0; j < NJ; ++j) take_channels<16>(qr, x, 64 * j + 16 * g, a[j]);
    };
    if (A.ba.max_blocks > A.top) load_rows(0);  // (or no request has more blocks than are wanted)
    int *out = A.selected + ((size_t)token * A.c.heads + head) * A.top;
    kv4_request rq;
    const int b = kv4_find(A.ba, token, shift, rq);
    if (b < 0) return;
    const int pos = rq.len - rq.rows + (token - rq.first);
    const int blocks = pos < 0 ? 0 : (pos >> shift) + 1;
    if (blocks <= A.top) {
        for (int j = tid; j < A.top; j += T) out[j] = j < blocks ? j : -1;
        return;
    }
    const int *table = A.ba.table + (size_t)b * A.ba.max_blocks;
    const int free_from = A.first, free_to = blocks - A.recent;  // the blocks that are chosen by score
    __syncthreads();
    uint32_t low = 0xffffffffu, high = 0;
    for (int r0 = 0; r0 < A.group; r0 += 16) {
        if (r0) load_rows(r0);
        pick_rows<D> r;
        round_rows<D>(a, g, r);
        for (int j0 = 16 * wave; j0 < blocks; j0 += 16 * W * U) {
            int phys[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int block = j0 + 16 * W * u + row;
                phys[u] = table[min(block, blocks - 1)];
            }
            pick_block<D> s[U];
#pragma unroll
            for (int u = 0; u < U; ++u) load_summary<D>(A.c, phys[u], head, g, s[u]);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int block = j0 + 16 * W * u + row;
                float mine[4], score = -INFINITY;
                score_rows<D>(r, s[u], mine);
#pragma unroll
                for (int i = 0; i < 4; ++i) score = fmaxf(score, r0 + 4 * g + i < A.group ? mine[i] : -INFINITY);
                score = score_of(score, s[u].scale);
                score = max_groups(score);
                uint32_t key = score_key(score);
                if (g == 0 && block < blocks) {
                    if (r0) key = max(key, keys[block]);
                    keys[block] = key;
                    if (r0 + 16 >= A.group && block >= free_from && block < free_to) low = min(low, key), high = max(high, key);
                }
            }
        }
    }
    if (g == 0 && low <= high) {
        atomicMin(&least, low);
        atomicMax(&most_key, high);
    }
    __syncthreads();
    // The key of the last block that is wanted, as its difference from the least, and how many at that key are.
    const uint32_t base = least;
    int want = A.top - A.first - A.recent;
    uint32_t prefix = 0, mask = 0;
    if (want > 0) {
        const uint32_t range = most_key - base;
        int at = range ? max(24 - __builtin_clz(range), 0) : 0;
#pragma unroll 1
        for (int pass = 0; pass < 4; ++pass) {
            uint32_t *bins = hist[pass];
            for (int j = free_from + tid; j < free_to; j += T) {
                const uint32_t key = keys[j] - base;
                if ((key & mask) == prefix) atomicAdd(&bins[key >> at & 255], 1u);
            }
            __syncthreads();
            uint32_t bin, left;
            bin_of(bins, (uint32_t)want, lane, bin, left);
            prefix |= bin << at;
            want = (int)left;
            mask |= 255u << at;
            if (at == 0) break;
            at = max(at - 8, 0);  // (the last pass may look at bits that are settled: they are the same in all that are left)
        }
    }
    // A thread's run of blocks: how many of them are in, or at the key, then where its own go.
    const int wanted = A.top - A.first - A.recent;
    auto kind = [&](int j) { return j < free_from || j >= free_to ? 2 : wanted == 0 ? 0 : keys[j] - base > prefix ? 2 : keys[j] - base == prefix ? 1 : 0; };
    const int per = (blocks + T - 1) / T, from = min(tid * per, blocks), to = min(from + per, blocks);
    int over = 0, equal = 0;
    for (int j = from; j < to; ++j) {
        const int k = kind(j);
        over += k == 2;
        equal += k == 1;
    }
    int over_upto = over, equal_upto = equal;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(over_upto, d), v = __shfl_up(equal_upto, d);
        if (lane >= d) over_upto += u, equal_upto += v;
    }
    if (lane == 63) above[wave] = over_upto, at_key[wave] = equal_upto;
    __syncthreads();
    int o = over_upto - over, q = equal_upto - equal;
    for (int w = 0; w < wave; ++w) o += above[w], q += at_key[w];
    for (int j = from; j < to; ++j) {
        const int k = kind(j);
        if (k == 2 || (k == 1 && q < want)) out[o + min(q, want)] = j;
        o += k == 2;
        q += k == 1;
    }
}

// Several tokens of a prompt share a workgroup where a group's rows leave room among the 16 of a product (SLOTS of them a token, a
// power of two): the summaries are read once for 16 / SLOTS tokens, their keys wait in LDS, and then a wavefront chooses for a
// token by itself, without barriers.  300 rows of 4 x 8 heads over 250 blocks: 16.6 us, with a workgroup a token 38.5; 200 rows
// of 8 x 2 heads of 256 over 500: 18 and 41.
template <int D, int SLOTS>
__global__ __launch_bounds__(256) void kv4_select_prompt_kernel(kv4_pick A) {
    constexpr int NJ = D / 64, TOKENS = 16 / SLOTS;
    extern __shared__ uint32_t keys[];  // [TOKENS][max_blocks]
    __shared__ uint32_t hist[4][256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = lane & 15, g = lane >> 4, shift = A.c.shift;
    const int head = blockIdx.x % (unsigned)A.c.heads, width = A.ba.max_blocks;
    int t = blockIdx.x / (unsigned)A.c.heads * TOKENS;
    const int behind = min(t + TOKENS, A.ba.tokens);
    const query_rows qr = rows_of(A.q, A.q_token, A.q_head, A.c.head_dim);
    while (t < behind) {
        kv4_request rq;
        const int b = kv4_find(A.ba, t, shift, rq);
        if (b < 0) {
            ++t;
            continue;
        }
        const int n = min(behind, rq.first + rq.rows) - t, pos0 = rq.len - rq.rows + (t - rq.first);  // tokens t .. t + n - 1, the first one's position
        const int blocks = pos0 + n - 1 < 0 ? 0 : ((pos0 + n - 1) >> shift) + 1;
        if (blocks > A.top) {
            float a[NJ][16];
            const int token = row / SLOTS, h = row % SLOTS;
            const float *x = token < n && h < A.group ? A.q + (size_t)(t + token) * A.q_token + (size_t)(head * A.group + h) * A.q_head : nullptr;
#pragma unroll
            for (int j = 0; j < NJ; ++j) take_channels<16>(qr, x, 64 * j + 16 * g, a[j]);
            pick_rows<D> r;
            round_rows<D>(a, g, r);
            const int *table = A.ba.table + (size_t)b * A.ba.max_blocks;
            for (int j0 = 16 * wave; j0 < blocks; j0 += 64) {
                const int block = j0 + row;
                pick_block<D> s;
                load_summary<D>(A.c, table[min(block, blocks - 1)], head, g, s);
                float mine[4];
                score_rows<D>(r, s, mine);
#pragma unroll
                for (int i = 0; i < 4; ++i) mine[i] = (4 * g + i) % SLOTS < A.group ? mine[i] : -INFINITY;
                constexpr int EACH = SLOTS < 4 ? SLOTS : 4;  // rows of a token in a lane
#pragma unroll
                for (int i = 0; i < 4; i += EACH) {
                    float score = mine[i];
#pragma unroll
                    for (int e = 1; e < EACH; ++e) score = fmaxf(score, mine[i + e]);
                    if (SLOTS == 8) score = over_rows(score, kv4_max{});
                    if (block < blocks) keys[(4 * g + i) / SLOTS * width + block] = score_key(score_of(score, s.scale));
                }
            }
        }
        __syncthreads();
        for (int token = wave; token < n; token += 4) {
            const int pos = pos0 + token, mine = pos < 0 ? 0 : (pos >> shift) + 1;  // this token's blocks
            int *out = A.selected + ((size_t)(t + token) * A.c.heads + head) * A.top;
            if (mine <= A.top) {
                for (int j = lane; j < A.top; j += 64) out[j] = j < mine ? j : -1;
                continue;
            }
            const uint32_t *key = keys + token * width;
            const int free_from = A.first, free_to = mine - A.recent, wanted = A.top - A.first - A.recent;
            uint32_t low = 0xffffffffu, high = 0, prefix = 0, mask = 0;
            int want = wanted;
            if (wanted > 0) {
                for (int j = free_from + lane; j < free_to; j += 64) low = min(low, key[j]), high = max(high, key[j]);
                low = ~over_wave(~low, kv4_umax{});
                high = over_wave(high, kv4_umax{});
                const uint32_t range = high - low;
                int at = range ? max(24 - __builtin_clz(range), 0) : 0;
#pragma unroll 1
                for (int pass = 0; pass < 4; ++pass) {
                    uint32_t *bins = hist[wave];
#pragma unroll
                    for (int i = 0; i < 4; ++i) bins[64 * i + lane] = 0;
                    wave_fence();
                    for (int j = free_from + lane; j < free_to; j += 64) {
                        const uint32_t v = key[j] - low;
                        if ((v & mask) == prefix) atomicAdd(&bins[v >> at & 255], 1u);
                    }
                    wave_fence();
                    uint32_t bin, left;
                    bin_of(bins, (uint32_t)want, lane, bin, left);
                    wave_fence();
                    prefix |= bin << at;
                    want = (int)left;
                    mask |= 255u << at;
                    if (at == 0) break;
                    at = max(at - 8, 0);  // (the last pass may look at bits that are settled: they are the same in all that are left)
                }
            }
            int o = 0, equal = 0;
            for (int j0 = 0; j0 < mine; j0 += 64) {
                const int j = j0 + lane;
                int kind = 0;
                if (j < mine) kind = j < free_from || j >= free_to ? 2 : wanted == 0 ? 0 : key[j] - low > prefix ? 2 : key[j] - low == prefix ? 1 : 0;
                const uint64_t before = (1ull << lane) - 1, same = __ballot(kind == 1);
                const bool in = kind == 2 || (kind == 1 && equal + __popcll(same & before) < want);
                const uint64_t taken = __ballot(in);
                if (in) out[o + __popcll(taken & before)] = j;
                o += __popcll(taken);
                equal += __popcll(same);
            }
        }
        __syncthreads();
        t += n;
    }
}

template <class F>
pg_status with_width(int D, F f) {
    if (D == 64) return f(std::integral_constant<int, 64>{});
    if (D == 128) return f(std::integral_constant<int, 128>{});
    return f(std::integral_constant<int, 256>{});
}

// Runs that a row tile's keys are divided in: as many as fill the chip with workgroups, none shorter than a tile of 64
// tokens a wavefront.  Not at all where a workgroup alone takes less longer than the joining launch does: one row of two key heads
// of 128 at 512 / 1024 / 1536 / 2048 tokens takes 9.0 / 11.3 / 14.4 / 17.1 us alone and 13.4 to 13.9 divided (heads of 256 at
// 1024: 19.6 and 17.9).  Prompts, with more work a token: 23 x 16 rows at 512 / 1024 tokens 36 / 61 alone, 30 / 33 divided.
size_t pick_splits(const pg_ctx *ctx, size_t tiles, size_t tokens, bool prompts, size_t D) {
    const size_t fill = (size_t)ctx->num_cu * 2;  // what runs at once
    size_t splits = tiles ? fill / tiles : 1;
    if (!prompts && tokens * std::max<size_t>(D, 128) <= 1024 * 128) return 1;
    // One and a half tiles a CU: in two runs each where they are long (43 requests of 8 key heads at 8000 tokens 88 instead of 99 us,
    // of lengths up to that 63 instead of 70; at 2500 33 and 32).
    if (!prompts && splits == 1 && 2 * tiles <= 3 * (size_t)ctx->num_cu && tokens >= 4096) splits = 2;
    const size_t most = (tokens + 255) / 256;
    if (splits > most) splits = most;
    return splits < 1 ? 1 : splits;
}

struct plan {
    size_t rows, row_tiles, tiles, splits, bytes;  // rows a tile (4, 8 or 16)
    size_t wide;                                   // row tiles a workgroup of the prompts' kernels, or 0: the others
};

// What a unit's many rows take on the prompts' kernels and on kv4_rows_kernel, in us, from 38 timed steps (5 to 2048 rows of a group of
// 1 to 16, 1 to 32 requests of 60 to 16384 tokens): rounds of workgroups, each a start and its tokens, and the joining launch with its bytes.
// Eight row tiles in one workgroup take what 5.7 of them take apart, but the workgroup starts later (queries and the first operands
// through LDS), its tiles are not always eight, nor its workgroups always as many as the chip runs: 320 rows of 8 x 8 heads over
// 2000 tokens 101 us and 78 apart, 200 of 8 over 1000 30 and 15; 256 of 16 x 8 over 4000 187 and 215, 624 of 12 x 8 over 60 25 and
// 46, 8192 of 8 over 16384 1130 and 1370.
double join_us(size_t rows, size_t D, size_t splits) { return splits > 1 ? 4 + (double)rows * D * 4 * (2 * splits + 1) / 4.5e6 : 0; }
double rounds_of(size_t workgroups, double run) { return workgroups <= run ? 1 : (double)workgroups / run + 0.15; }
bool prompts_pay(const pg_ctx *ctx, size_t units, size_t row_tiles, size_t tokens, size_t D) {
    const size_t groups = units * ((row_tiles + 7) / 8), tiles = units * row_tiles, rows = tiles * 16;
    const double cus = ctx->num_cu, each = tokens * (double)D / 128;
    const size_t ws = pick_splits(ctx, groups, tokens, true, D), rs = pick_splits(ctx, tiles, tokens, false, D);
    const double whole = rounds_of(groups * ws, D == 256 ? cus : 2 * cus) * (14 + (D == 256 ? 0.0358 : 0.0716) * each / ws) + join_us(rows, D, ws);
    const double apart = rounds_of(tiles * rs, D == 256 ? 2 * cus : 3 * cus) * (6 + (D == 256 ? 0.0118 : 0.0188) * each / rs) + join_us(rows, D, rs);
    return whole < apart;
}
// tokens: of the table; seen: of those that any row sees, where a window says so (fewer runs than were reported without it need no
// more scratch; the kernel is chosen without it, so that it is the same one).
plan plan_for(const pg_ctx *ctx, const pg_paged_kv4 *c, size_t units, size_t unit_rows, size_t tokens, size_t seen, bool prompts) {
    plan p;
    p.rows = unit_rows <= 4 ? 4 : unit_rows <= 8 ? 8 : 16;
    p.row_tiles = (unit_rows + p.rows - 1) / p.rows;
    p.tiles = units * c->heads * p.row_tiles;
    p.wide = prompts && p.row_tiles >= 4 && prompts_pay(ctx, units * c->heads, p.row_tiles, tokens, (size_t)c->D) ? 8 : 0;
    const size_t workgroups = p.wide ? units * c->heads * ((p.row_tiles + p.wide - 1) / p.wide) : p.tiles;
    p.splits = pick_splits(ctx, workgroups, std::min(tokens, seen), p.wide, (size_t)c->D);
    p.bytes = p.splits > 1 ? p.tiles * p.splits * (p.rows * (size_t)c->D + 32) * sizeof(float) : 0;
    return p;
}
plan dense_plan(const pg_ctx *ctx, const pg_paged_kv4 *c, size_t num_q_heads, size_t batch, size_t max_query, size_t max_blocks, size_t seen = SIZE_MAX) {
    return plan_for(ctx, c, batch, max_query * (num_q_heads / c->heads), max_blocks * c->block_size, seen, true);
}
plan selected_plan(const pg_ctx *ctx, const pg_paged_kv4 *c, size_t num_q_heads, size_t tokens, size_t top) {
    return plan_for(ctx, c, tokens, num_q_heads / c->heads, top * c->block_size, SIZE_MAX, false);
}

template <bool SELECTED>
pg_status launch_rows(pg_ctx *ctx, const char *fn, const pg_paged_kv4 *c, kv4_attn &A, const plan &p) {
    if (p.tiles * p.splits >= (1u << 24)) return pg_fail(PG_EUNSUPPORTED, "%s: %zu row tiles in %zu runs are more than a launch takes", fn, p.tiles, p.splits);
    A.splits = (int)p.splits;
    A.row_tiles = (int)p.row_tiles;
    A.by_length = !SELECTED && p.splits == 1 && A.ba.batch > 1 && A.ba.batch <= RANKED && p.tiles > (size_t)ctx->num_cu * 2;
    const dim3 grid((unsigned)(p.tiles * p.splits)), join((unsigned)(p.tiles * p.rows / 4)), block(256);
    return with_width(c->D, [&](auto w) -> pg_status {
        constexpr int D = decltype(w)::value;
        auto go = [&](const char *name, auto plain, auto capped, auto joined) -> pg_status {
            PG_TRY(pg_launch(ctx, name, A.cap > 0.f ? capped : plain, grid, block, 0, A));
            return p.splits == 1 ? PG_OK : pg_launch(ctx, "kv4_join_kernel", joined, join, block, 0, A);
        };
        if constexpr (!SELECTED)
            if (p.wide) {
                const dim3 workgroups((unsigned)(A.ba.batch * c->heads * ((p.row_tiles + p.wide - 1) / p.wide) * p.splits));
                auto prompt = [&](const char *name, auto kernel, size_t lds, unsigned threads) -> pg_status {
                    PG_TRY(pg_allow_dynamic_lds(ctx, reinterpret_cast<const void *>(kernel), lds));
                    return pg_launch(ctx, name, kernel, workgroups, dim3(threads), lds, A);
                };
                if constexpr (D == 256)
                    PG_TRY(prompt("kv4_prompt_kernel", A.cap > 0.f ? kv4_prompt_kernel<true> : kv4_prompt_kernel<false>, sizeof(prompt_lds<D>), 512));
                else
                    PG_TRY(prompt("kv4_prompt32_kernel", A.cap > 0.f ? kv4_prompt32_kernel<D, true> : kv4_prompt32_kernel<D, false>, sizeof(prompt32_lds<D>), 256));
                return p.splits == 1 ? PG_OK : pg_launch(ctx, "kv4_join_kernel", kv4_join_kernel<D, 16, SELECTED>, join, block, 0, A);
            }
        if (p.rows == 4) return go(SELECTED ? "kv4_few_selected_kernel" : "kv4_few_kernel", kv4_few_kernel<D, 4, false, SELECTED>, kv4_few_kernel<D, 4, true, SELECTED>, kv4_join_kernel<D, 4, SELECTED>);
        if (p.rows == 8) return go(SELECTED ? "kv4_few_selected_kernel" : "kv4_few_kernel", kv4_few_kernel<D, 8, false, SELECTED>, kv4_few_kernel<D, 8, true, SELECTED>, kv4_join_kernel<D, 8, SELECTED>);
        return go(SELECTED ? "kv4_rows_selected_kernel" : "kv4_rows_kernel", kv4_rows_kernel<D, false, SELECTED>, kv4_rows_kernel<D, true, SELECTED>, kv4_join_kernel<D, 16, SELECTED>);
    });
}

pg_status check_score(const char *fn, float scale, float logit_cap) {
    PG_CHECK_ARG(isfinite(scale), "%s: scale is not finite", fn);
    PG_CHECK_ARG(logit_cap >= 0.f && isfinite(logit_cap), "%s: logit_cap is negative or not finite", fn);
    return PG_OK;
}

}  // namespace

PG_API pg_status pg_paged_kv4_attention_scratch(pg_ctx *ctx, const pg_paged_kv4 *c, size_t num_q_heads, size_t batch, size_t max_query, size_t max_blocks, size_t *bytes) {
    PG_TRY(pg_use(ctx));
    PG_TRY(pg_kv4_check_step("pg_paged_kv4_attention_scratch", c, num_q_heads, batch, max_query, max_blocks));
    PG_CHECK_ARG(bytes != nullptr, "pg_paged_kv4_attention_scratch: null output");
    *bytes = dense_plan(ctx, c, num_q_heads, batch, max_query, max_blocks).bytes;
    return PG_OK;
}

PG_API pg_status pg_paged_kv4_selected_scratch(pg_ctx *ctx, const pg_paged_kv4 *c, size_t num_q_heads, size_t tokens, size_t top_k, size_t *bytes) {
    PG_TRY(pg_use(ctx));
    PG_TRY(pg_kv4_check_step("pg_paged_kv4_selected_scratch", c, num_q_heads, 0, tokens, 1));
    PG_CHECK_ARG(top_k < (1ull << 31) && top_k * c->block_size <= PG_KV4_MAX_TOKENS, "pg_paged_kv4_selected_scratch: %zu blocks: out of range", top_k);
    PG_CHECK_ARG(bytes != nullptr, "pg_paged_kv4_selected_scratch: null output");
    *bytes = selected_plan(ctx, c, num_q_heads, tokens, top_k).bytes;
    return PG_OK;
}

PG_API pg_status pg_paged_kv4_attention_dev(pg_ctx *ctx, const pg_paged_kv4 *c, const float *q_dev, size_t q_token_stride, size_t q_head_stride, size_t num_q_heads,
                                            const int32_t *query_start_dev, const int32_t *seq_lens_dev, size_t batch, size_t tokens, size_t max_query,
                                            const int32_t *block_table_dev, size_t max_blocks, float scale, int mask_kind, size_t window, size_t sink_tokens, float logit_cap,
                                            void *scratch_dev, size_t scratch_bytes, float *out_dev) {
    static const char *fn = "pg_paged_kv4_attention";
    PG_TRY(pg_use(ctx));
    PG_TRY(pg_kv4_check_step(fn, c, num_q_heads, batch, tokens, max_blocks));
    PG_TRY(check_score(fn, scale, logit_cap));
    PG_CHECK_ARG(mask_kind >= PG_MASK_NONE && mask_kind <= PG_MASK_CAUSAL_SLIDING_WINDOW, "%s: unknown mask kind %d", fn, mask_kind);
    if (tokens == 0 || batch == 0 || max_query == 0) return PG_OK;
    PG_CHECK_ARG(q_dev && query_start_dev && seq_lens_dev && block_table_dev && out_dev, "%s: null pointer", fn);
    PG_CHECK_ARG(q_token_stride < (1ull << 40) && q_head_stride < (1ull << 40), "%s: strides out of range", fn);
    PG_CHECK_ARG(max_query < (1ull << 31), "%s: %zu rows a request: out of range", fn, max_query);
    // (Planned by max_query even where there are fewer rows than that: the scratch was asked for without their number.)
    // What a tile of rows sees behind its window and of the sinks, in whole tiles of keys.
    const size_t seen = mask_kind == PG_MASK_CAUSAL_SLIDING_WINDOW && window < (1u << 30) && sink_tokens < (1u << 30) ? window + max_query + sink_tokens + 128 : SIZE_MAX;
    const plan p = dense_plan(ctx, c, num_q_heads, batch, max_query, max_blocks, seen);
    PG_CHECK_ARG(p.bytes == 0 || (scratch_dev && scratch_bytes >= p.bytes && ((uintptr_t)scratch_dev & 15) == 0),
                 "%s: scratch of %zu bytes, %zu are needed (16-byte aligned)", fn, scratch_bytes, p.bytes);
    PG_TRY(c->use(fn, ctx));
    kv4_attn A = {};
    A.q = q_dev, A.q_token = q_token_stride, A.q_head = q_head_stride;
    A.c = kv4_view_of(c);
    A.ba = {query_start_dev, seq_lens_dev, block_table_dev, (int)batch, (int)tokens, (int)max_blocks};
    A.scale = scale, A.cap = logit_cap, A.mask = mask_kind;
    A.window = (int)std::min<size_t>(window, 0x7fffffffu), A.sinks = (int)std::min<size_t>(sink_tokens, 0x7fffffffu);
    A.group = (int)(num_q_heads / c->heads), A.q_heads = (int)num_q_heads, A.max_query = (int)max_query;
    A.part = static_cast<float *>(scratch_dev), A.out = out_dev;
    return launch_rows<false>(ctx, fn, c, A, p);
}

PG_API pg_status pg_paged_kv4_select_dev(pg_ctx *ctx, const pg_paged_kv4 *c, const float *q_dev, size_t q_token_stride, size_t q_head_stride, size_t num_q_heads,
                                         const int32_t *query_start_dev, const int32_t *seq_lens_dev, size_t batch, size_t tokens, const int32_t *block_table_dev,
                                         size_t max_blocks, size_t top_k, size_t first_blocks, size_t recent_blocks, int32_t *selected_dev) {
    static const char *fn = "pg_paged_kv4_select";
    PG_TRY(pg_use(ctx));
    PG_TRY(pg_kv4_check_step(fn, c, num_q_heads, batch, tokens, max_blocks));
    PG_CHECK_ARG(top_k > 0 && top_k < (1u << 24) && recent_blocks >= 1 && first_blocks <= top_k && recent_blocks <= top_k && first_blocks + recent_blocks <= top_k,
                 "%s: %zu blocks with the first %zu and the last %zu of them (the last at least one)", fn, top_k, first_blocks, recent_blocks);
    if (tokens == 0 || batch == 0) return PG_OK;
    PG_CHECK_ARG(q_dev && query_start_dev && seq_lens_dev && block_table_dev && selected_dev, "%s: null pointer", fn);
    PG_CHECK_ARG(q_token_stride < (1ull << 40) && q_head_stride < (1ull << 40), "%s: strides out of range", fn);
    const size_t lds = max_blocks * sizeof(uint32_t);
    if (lds > (144u << 10)) return pg_fail(PG_EUNSUPPORTED, "%s: tables of %zu blocks (36864 at most: their scores live in on-chip memory)", fn, max_blocks);
    if (tokens * c->heads >= (1u << 22)) return pg_fail(PG_EUNSUPPORTED, "%s: %zu rows of %zu key heads are more than a launch takes", fn, tokens, c->heads);
    PG_TRY(c->use(fn, ctx));
    kv4_pick A = {q_dev, q_token_stride, q_head_stride, kv4_view_of(c), {query_start_dev, seq_lens_dev, block_table_dev, (int)batch, (int)tokens, (int)max_blocks},
                  (int)(num_q_heads / c->heads), (int)top_k, (int)first_blocks, (int)recent_blocks, selected_dev};
    return with_width(c->D, [&](auto w) -> pg_status {
        constexpr int D = decltype(w)::value;
        auto go = [&](auto kernel, unsigned threads) -> pg_status {
            if (lds > (48u << 10)) PG_TRY(pg_allow_dynamic_lds(ctx, reinterpret_cast<const void *>(kernel), lds));
            return pg_launch(ctx, "kv4_select_kernel", kernel, dim3((unsigned)(tokens * c->heads)), dim3(threads), lds, A);
        };
        // Prompts (four rows a request and more, on the whole) of groups that leave room for other tokens, if the chip has enough of them:
        // 16 requests of 4 rows, 8 heads of 4 over 62 blocks 7.4 us against 9.9, of 2 rows 11.6 against 8.5; 4 of 8 rows of 2 heads of 1,
        // which leave ten workgroups, 13.9 against 7.9.
        size_t slots = 1;
        while (slots < (size_t)A.group) slots *= 2;
        const size_t each = 16 / slots, shared_lds = each * lds;
        if (slots <= 8 && max_blocks > top_k && tokens >= 4 * batch && shared_lds <= (40u << 10) && (tokens + each - 1) / each * c->heads >= (size_t)ctx->num_cu / 2) {
            const dim3 grid((unsigned)((tokens + each - 1) / each * c->heads));
            auto prompt = [&](auto kernel) { return pg_launch(ctx, "kv4_select_prompt_kernel", kernel, grid, dim3(256), shared_lds, A); };
            return slots == 1 ? prompt(kv4_select_prompt_kernel<D, 1>) : slots == 2 ? prompt(kv4_select_prompt_kernel<D, 2>) :
                   slots == 4 ? prompt(kv4_select_prompt_kernel<D, 4>) : prompt(kv4_select_prompt_kernel<D, 8>);
        }
        // 1024 threads where a row has many blocks and the chip has room: 64 rows and heads over 500 / 1000 / 2000 blocks 17 / 23 / 32 us
        // against 14 / 29 / 52 of 256 threads; 512 of them over 1000 51 against 38.
        return max_blocks > 640 && tokens * c->heads <= (size_t)ctx->num_cu ? go(kv4_select_kernel<D, 1024>, 1024) : go(kv4_select_kernel<D, 256>, 256);
    });
}

PG_API pg_status pg_paged_kv4_attention_selected_dev(pg_ctx *ctx, const pg_paged_kv4 *c, const float *q_dev, size_t q_token_stride, size_t q_head_stride, size_t num_q_heads,
                                                     const int32_t *query_start_dev, const int32_t *seq_lens_dev, size_t batch, size_t tokens,
                                                     const int32_t *block_table_dev, size_t max_blocks, const int32_t *selected_dev, size_t top_k, float scale,
                                                     float logit_cap, void *scratch_dev, size_t scratch_bytes, float *out_dev) {
    static const char *fn = "pg_paged_kv4_attention_selected";
    PG_TRY(pg_use(ctx));
    PG_TRY(pg_kv4_check_step(fn, c, num_q_heads, batch, tokens, max_blocks));
    PG_TRY(check_score(fn, scale, logit_cap));
    PG_CHECK_ARG(top_k > 0 && top_k < (1ull << 31) && top_k * c->block_size <= PG_KV4_MAX_TOKENS, "%s: %zu blocks: out of range", fn, top_k);
    if (tokens == 0 || batch == 0) return PG_OK;
    PG_CHECK_ARG(q_dev && query_start_dev && seq_lens_dev && block_table_dev && selected_dev && out_dev, "%s: null pointer", fn);
    PG_CHECK_ARG(q_token_stride < (1ull << 40) && q_head_stride < (1ull << 40), "%s: strides out of range", fn);
    const plan p = selected_plan(ctx, c, num_q_heads, tokens, std::min(top_k, max_blocks));  // (no more scratch than was reported without the table)
    PG_CHECK_ARG(p.bytes == 0 || (scratch_dev && scratch_bytes >= p.bytes && ((uintptr_t)scratch_dev & 15) == 0),
                 "%s: scratch of %zu bytes, %zu are needed (16-byte aligned)", fn, scratch_bytes, p.bytes);
    PG_TRY(c->use(fn, ctx));
    kv4_attn A = {};
    A.q = q_dev, A.q_token = q_token_stride, A.q_head = q_head_stride;
    A.c = kv4_view_of(c);
    A.ba = {query_start_dev, seq_lens_dev, block_table_dev, (int)batch, (int)tokens, (int)max_blocks};
    A.selected = selected_dev, A.top = (int)top_k;
    A.scale = scale, A.cap = logit_cap, A.mask = PG_MASK_CAUSAL;
    A.group = (int)(num_q_heads / c->heads), A.q_heads = (int)num_q_heads, A.max_query = 1;
    A.part = static_cast<float *>(scratch_dev), A.out = out_dev;
    return launch_rows<true>(ctx, fn, c, A, p);
}

// ---- host arrays ----------------------------------------------------------------------------

namespace {

// What a step's host arrays say, refused where a kernel would have had to leave something out.
pg_status check_host_step(const char *fn, const pg_paged_kv4 *c, const int32_t *query_start, const int32_t *seq_lens, size_t batch, size_t tokens, const int32_t *block_table,
                          size_t max_blocks) {
    PG_CHECK_ARG(query_start[0] == 0 && query_start[batch] >= 0 && (size_t)query_start[batch] <= tokens, "%s: rows %d to %d of %zu", fn, query_start[0], query_start[batch], tokens);
    for (size_t b = 0; b < batch; ++b) {
        PG_CHECK_ARG(query_start[b + 1] >= query_start[b], "%s: request %zu starts at row %d and ends at %d", fn, b, query_start[b], query_start[b + 1]);
        PG_CHECK_ARG(seq_lens[b] >= 0 && (size_t)seq_lens[b] <= max_blocks * c->block_size, "%s: request %zu has %d tokens, its table room for %zu", fn, b, seq_lens[b],
                     max_blocks * c->block_size);
        PG_CHECK_ARG(query_start[b + 1] - query_start[b] <= seq_lens[b], "%s: request %zu has %d rows and %d tokens", fn, b, query_start[b + 1] - query_start[b], seq_lens[b]);
        const size_t used = ((size_t)seq_lens[b] + c->block_size - 1) / c->block_size;
        for (size_t j = 0; j < used; ++j) {
            const int32_t e = block_table[b * max_blocks + j];
            PG_CHECK_ARG(e >= 0 && (size_t)e < c->num_blocks, "%s: request %zu's block %zu is %d of %zu", fn, b, j, e, c->num_blocks);
        }
    }
    return PG_OK;
}

struct host_step {
    pg_dev_block starts, lens, table;
    pg_status in(pg_ctx *ctx, const int32_t *query_start, const int32_t *seq_lens, size_t batch, const int32_t *block_table, size_t max_blocks) {
        PG_TRY(pg_host_in(ctx, query_start, (batch + 1) * sizeof(int32_t), starts));
        PG_TRY(pg_host_in(ctx, seq_lens, batch * sizeof(int32_t), lens));
        return pg_host_in(ctx, block_table, batch * max_blocks * sizeof(int32_t), table);
    }
};

}  // namespace

PG_API pg_status pg_paged_kv4_summarise(pg_ctx *ctx, pg_paged_kv4 *c, const int32_t *query_start, const int32_t *seq_lens, size_t batch, const int32_t *block_table,
                                        size_t max_blocks) {
    static const char *fn = "pg_paged_kv4_summarise";
    PG_TRY(pg_use(ctx));
    PG_CHECK_ARG(c != nullptr, "%s: null cache", fn);
    PG_TRY(pg_kv4_check_step(fn, c, c->heads, batch, 0, max_blocks));
    if (batch == 0) return PG_OK;
    PG_CHECK_ARG(query_start && seq_lens && block_table, "%s: null pointer", fn);
    PG_TRY(check_host_step(fn, c, query_start, seq_lens, batch, 0x7fffffff, block_table, max_blocks));
    const size_t tokens = (size_t)query_start[batch];
    host_step h;
    PG_TRY(h.in(ctx, query_start, seq_lens, batch, block_table, max_blocks));
    PG_TRY(pg_paged_kv4_summarise_dev(ctx, c, h.starts.as<int32_t>(), h.lens.as<int32_t>(), batch, tokens, h.table.as<int32_t>(), max_blocks));
    PG_HIP(hipStreamSynchronize(ctx->stream));
    return PG_OK;
}

PG_API pg_status pg_paged_kv4_attention(pg_ctx *ctx, const pg_paged_kv4 *c, const float *q, size_t num_q_heads, const int32_t *query_start, const int32_t *seq_lens,
                                        size_t batch, size_t tokens, const int32_t *block_table, size_t max_blocks, float scale, int mask_kind, size_t window,
                                        size_t sink_tokens, float logit_cap, float *out) {
    static const char *fn = "pg_paged_kv4_attention";
    PG_TRY(pg_use(ctx));
    PG_TRY(pg_kv4_check_step(fn, c, num_q_heads, batch, tokens, max_blocks));
    PG_TRY(check_score(fn, scale, logit_cap));
    PG_CHECK_ARG(mask_kind >= PG_MASK_NONE && mask_kind <= PG_MASK_CAUSAL_SLIDING_WINDOW, "%s: unknown mask kind %d", fn, mask_kind);
    if (tokens == 0 || batch == 0) return PG_OK;
    PG_CHECK_ARG(q && query_start && seq_lens && block_table && out, "%s: null pointer", fn);
    PG_TRY(check_host_step(fn, c, query_start, seq_lens, batch, tokens, block_table, max_blocks));
    size_t longest = 0;
    for (size_t b = 0; b < batch; ++b) longest = std::max(longest, (size_t)(query_start[b + 1] - query_start[b]));
    const size_t rows = (size_t)query_start[batch], row = num_q_heads * c->head_dim, bytes = rows * row * sizeof(float);
    if (rows == 0) return PG_OK;
    size_t scratch = 0;
    PG_TRY(pg_paged_kv4_attention_scratch(ctx, c, num_q_heads, batch, longest, max_blocks, &scratch));
    host_step h;
    pg_dev_block dq, dout, ds;
    PG_TRY(h.in(ctx, query_start, seq_lens, batch, block_table, max_blocks));
    PG_TRY(pg_host_in(ctx, q, bytes, dq));
    PG_TRY(dout.alloc(ctx, bytes));
    PG_TRY(ds.alloc(ctx, scratch));
    PG_TRY(pg_paged_kv4_attention_dev(ctx, c, dq.as<float>(), row, c->head_dim, num_q_heads, h.starts.as<int32_t>(), h.lens.as<int32_t>(), batch, rows, longest,
                                      h.table.as<int32_t>(), max_blocks, scale, mask_kind, window, sink_tokens, logit_cap, ds.p, scratch, dout.as<float>()));
    return pg_host_out(ctx, out, dout.p, bytes);
}

PG_API pg_status pg_paged_kv4_select(pg_ctx *ctx, const pg_paged_kv4 *c, const float *q, size_t num_q_heads, const int32_t *query_start, const int32_t *seq_lens, size_t batch,
                                     size_t tokens, const int32_t *block_table, size_t max_blocks, size_t top_k, size_t first_blocks, size_t recent_blocks,
                                     int32_t *selected) {
    static const char *fn = "pg_paged_kv4_select";
    PG_TRY(pg_use(ctx));
    PG_TRY(pg_kv4_check_step(fn, c, num_q_heads, batch, tokens, max_blocks));
    if (tokens == 0 || batch == 0) return PG_OK;
    PG_CHECK_ARG(q && query_start && seq_lens && block_table && selected, "%s: null pointer", fn);
    PG_TRY(check_host_step(fn, c, query_start, seq_lens, batch, tokens, block_table, max_blocks));
    const size_t rows = (size_t)query_start[batch], row = num_q_heads * c->head_dim, bytes = rows * c->heads * top_k * sizeof(int32_t);
    if (rows == 0) return PG_OK;
    host_step h;
    pg_dev_block dq, dsel;
    PG_TRY(h.in(ctx, query_start, seq_lens, batch, block_table, max_blocks));
    PG_TRY(pg_host_in(ctx, q, rows * row * sizeof(float), dq));
    PG_CHECK_ARG(top_k < (1u << 24), "%s: %zu blocks: out of range", fn, top_k);
    PG_TRY(dsel.alloc(ctx, bytes));
    PG_TRY(pg_paged_kv4_select_dev(ctx, c, dq.as<float>(), row, c->head_dim, num_q_heads, h.starts.as<int32_t>(), h.lens.as<int32_t>(), batch, rows, h.table.as<int32_t>(),
                                   max_blocks, top_k, first_blocks, recent_blocks, dsel.as<int32_t>()));
    return pg_host_out(ctx, selected, dsel.p, bytes);
}

PG_API pg_status pg_paged_kv4_attention_selected(pg_ctx *ctx, const pg_paged_kv4 *c, const float *q, size_t num_q_heads, const int32_t *query_start, const int32_t *seq_lens,
                                                 size_t batch, size_t tokens, const int32_t *block_table, size_t max_blocks, const int32_t *selected, size_t top_k,
                                                 float scale, float logit_cap, float *out) {
    static const char *fn = "pg_paged_kv4_attention_selected";
    PG_TRY(pg_use(ctx));
    PG_TRY(pg_kv4_check_step(fn, c, num_q_heads, batch, tokens, max_blocks));
    PG_TRY(check_score(fn, scale, logit_cap));
    PG_CHECK_ARG(top_k > 0 && top_k < (1ull << 31) && top_k * c->block_size <= PG_KV4_MAX_TOKENS, "%s: %zu blocks: out of range", fn, top_k);
    if (tokens == 0 || batch == 0) return PG_OK;
    PG_CHECK_ARG(q && query_start && seq_lens && block_table && selected && out, "%s: null pointer", fn);
    PG_TRY(check_host_step(fn, c, query_start, seq_lens, batch, tokens, block_table, max_blocks));
    const size_t rows = (size_t)query_start[batch], row = num_q_heads * c->head_dim, bytes = rows * row * sizeof(float);
    if (rows == 0) return PG_OK;
    for (size_t b = 0, t = 0; b < batch; ++b)
        for (; t < (size_t)query_start[b + 1]; ++t) {
            const int64_t pos = seq_lens[b] - (query_start[b + 1] - (int64_t)t);
            for (size_t h = 0; h < c->heads; ++h) {
                const int32_t *s = selected + (t * c->heads + h) * top_k;
                for (size_t i = 0; i < top_k; ++i)
                    PG_CHECK_ARG(s[i] == -1 || (s[i] >= 0 && s[i] <= pos / (int64_t)c->block_size && (i == 0 || (s[i - 1] >= 0 && s[i] > s[i - 1]))),
                                 "%s: row %zu, key head %zu: block %d as number %zu (ascending, up to the row's own %lld, -1 behind them)", fn, t, h, s[i], i,
                                 (long long)(pos / (int64_t)c->block_size));
            }
        }
    size_t scratch = 0;
    PG_TRY(pg_paged_kv4_selected_scratch(ctx, c, num_q_heads, rows, top_k, &scratch));
    host_step h;
    pg_dev_block dq, dsel, dout, ds;
    PG_TRY(h.in(ctx, query_start, seq_lens, batch, block_table, max_blocks));
    PG_TRY(pg_host_in(ctx, q, bytes, dq));
    PG_TRY(pg_host_in(ctx, selected, rows * c->heads * top_k * sizeof(int32_t), dsel));
    PG_TRY(dout.alloc(ctx, bytes));
    PG_TRY(ds.alloc(ctx, scratch));
    PG_TRY(pg_paged_kv4_attention_selected_dev(ctx, c, dq.as<float>(), row, c->head_dim, num_q_heads, h.starts.as<int32_t>(), h.lens.as<int32_t>(), batch, rows,
                                               h.table.as<int32_t>(), max_blocks, dsel.as<int32_t>(), top_k, scale, logit_cap, ds.p, scratch, dout.as<float>()));
    return pg_host_out(ctx, out, dout.p, bytes);
}
