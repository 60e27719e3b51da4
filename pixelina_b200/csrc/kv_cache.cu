// kv_cache.cu -- writing, rewinding, reading and evicting the 8-bit
// key/value cache (layout and formulas: kv_cache.cuh).
//
//   k_kv_append    one CTA per (block touched, head): the block's rows from
//                  the fp32 tail and the new rows, its two scales, its codes
//   k_kv_truncate  one CTA per (head, sequence): the block that the new
//                  length ends in, quantized anew without the dropped rows
//   k_kv_read      one CTA per (block, head, sequence): the fp32 values
//   k_kv_select    one CTA per (head, sequence): the kept tokens, in order
//   k_kv_compact   one CTA per (destination block, head, sequence)
//
// All have 2 * D threads per CTA but k_kv_select: for K, thread (token,
// 16 consecutive channels); for V, thread (channel, 16 consecutive tokens),
// the shapes in which a record's bytes lie together.
#include <algorithm>
#include <type_traits>
#include "kv_cache.cuh"

namespace pxq {
namespace {

constexpr float kKvTiny = 3.009265538105056e-36f;  // 2^-118: blocks below it are stored as zeros (1 / d stays finite)

// Largest magnitudes of the CTA's K and V values; not finite: +inf.
__device__ __forceinline__ float kv_mag(float m, float x)
{
    const float a = fabsf(x);
    return a <= FLT_MAX ? fmaxf(m, a) : INFINITY;
}
__device__ __forceinline__ float2 kv_block_max(float mk, float mv, float2* red)
{
#pragma unroll
    for (int off = 16; off; off >>= 1) {
        mk = fmaxf(mk, __shfl_xor_sync(0xffffffffu, mk, off));
        mv = fmaxf(mv, __shfl_xor_sync(0xffffffffu, mv, off));
    }
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(mk, mv);
    __syncthreads();
    for (int w = 0; w < (int)(blockDim.x >> 5); w++) {
        mk = fmaxf(mk, red[w].x);
        mv = fmaxf(mv, red[w].y);
    }
    return make_float2(mk, mv);
}
__device__ __forceinline__ float kv_scale(float a)
{
    if (a == INFINITY) return __int_as_float(0x7fffffff);
    return a < kKvTiny ? 0.f : __fdiv_rn(a, 127.f);
}

// Code byte of x under scale d (inv = 1 / d rounded): the integer nearest to
// x / d, ties to even.  rint(x * inv) is within one of it, and r = x - q d is
// exact (|r| < 2 d on the grid of d's last place), so comparing 2 |r| with d
// settles it.
__device__ __forceinline__ uint32_t kv_code(float x, float d, float inv)
{
    float q = rintf(__fmul_rn(x, inv));
    const float r = __fmaf_rn(-q, d, x), e = 2.f * fabsf(r);
    if (e > d || (e == d && ((int)q & 1))) q += copysignf(1.f, r);
    return (uint32_t)((int)q + 128) & 255u;
}

// Quantize and store a block from registers: xk = 16 channels (16 * kc ..) of
// token kt, xv = 16 tokens (16 * vt ..) of channel vd; rows past the present
// ones are zero.
template <int D>
__device__ __forceinline__ void kv_store_block(const KvView& c, int64_t sh, int b, const float (&xk)[16], const float (&xv)[16],
                                               float2* red)
{
    const int tid = threadIdx.x, kt = tid / (D / 16), kc = tid % (D / 16), vd = tid % D, vt = tid / D;
    float mk = 0.f, mv = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        mk = kv_mag(mk, xk[i]);
        mv = kv_mag(mv, xv[i]);
    }
    const float2 m = kv_block_max(mk, mv, red);
    const float dk = kv_scale(m.x), dv = kv_scale(m.y);
    const float ik = dk > 0.f ? __fdiv_rn(1.f, dk) : 0.f, iv = dv > 0.f ? __fdiv_rn(1.f, dv) : 0.f;
    uint8_t* rec = c.codes + (sh * c.nb + b) * kv_record_bytes(D);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        w[i] = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) w[i] |= (dk > 0.f ? kv_code(xk[4 * i + j], dk, ik) : 128u) << (8 * j);
    }
    if (D % 64 != 0 && kc >= D / 64 * 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<uint32_t*>(rec + kv_k_offset<D>(kt, 16 * kc + 4 * i)) = w[i];
    } else {
        *reinterpret_cast<uint4*>(rec + kv_k_offset<D>(kt, 16 * kc)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        w[i] = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) w[i] |= (dv > 0.f ? kv_code(xv[4 * i + j], dv, iv) : 128u) << (8 * j);
    }
    *reinterpret_cast<uint2*>(rec + kv_v_offset<D>(16 * vt, vd)) = make_uint2(w[0], w[1]);
    *reinterpret_cast<uint2*>(rec + kv_v_offset<D>(16 * vt + 8, vd)) = make_uint2(w[2], w[3]);
    if (tid == 0) c.scales[sh * c.nb + b] = make_float2(dk, dv);
}

// The thread's 16 K channels (token kt) and 16 V tokens (channel vd) of a
// block, as the values it stands for.
template <int D>
__device__ __forceinline__ void kv_values(const KvView& c, int64_t sh, int b, float (&xk)[16], float (&xv)[16])
{
    const int tid = threadIdx.x, kt = tid / (D / 16), kc = tid % (D / 16), vd = tid % D, vt = tid / D;
    const uint8_t* rec = c.codes + (sh * c.nb + b) * kv_record_bytes(D);
    const float2 d = c.scales[sh * c.nb + b];
    uint32_t w[4];
    if (D % 64 != 0 && kc >= D / 64 * 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = *reinterpret_cast<const uint32_t*>(rec + kv_k_offset<D>(kt, 16 * kc + 4 * i));
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(rec + kv_k_offset<D>(kt, 16 * kc));
        w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    }
    const uint2 a = *reinterpret_cast<const uint2*>(rec + kv_v_offset<D>(16 * vt, vd));
    const uint2 e = *reinterpret_cast<const uint2*>(rec + kv_v_offset<D>(16 * vt + 8, vd));
    const uint32_t z[4] = {a.x, a.y, e.x, e.y};
#pragma unroll
    for (int i = 0; i < 16; i++) {
        xk[i] = __fmul_rn((float)((int)((w[i / 4] >> (8 * (i % 4))) & 255u) - 128), d.x);
        xv[i] = __fmul_rn((float)((int)((z[i / 4] >> (8 * (i % 4))) & 255u) - 128), d.y);
    }
}

__device__ __forceinline__ float* kv_tail(const KvView& c, int s, int slot, int h, int kv)
{
    return c.tail + ((((int64_t)s * 2 + slot) * c.H + h) * 2 + kv) * kKvBlock * c.D;
}

__device__ __forceinline__ void ld16(const float* p, float (&x)[16], bool vec)
{
    if (vec) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4 v = *reinterpret_cast<const float4*>(p + 4 * i);
            x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = p[i];
    }
}
__device__ __forceinline__ void st16(float* p, const float (&x)[16], bool vec)
{
    if (vec) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            *reinterpret_cast<float4*>(p + 4 * i) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) p[i] = x[i];
    }
}

// Blocks that an append of n rows to len tokens touches; 0 when they do not fit.
__device__ __forceinline__ int kv_touched(const KvView& c, int len, int n)
{
    if (n <= 0 || (int64_t)len + n > c.cap) return 0;
    return (len % kKvBlock + n - 1) / kKvBlock + 1;
}

template <int D>
__global__ void __launch_bounds__(2 * D)
    k_kv_append(const __grid_constant__ KvView c, const float* k, int64_t ldk, const float* v, int64_t ldv,
                int64_t rows, const int32_t* starts, int veck, uint32_t* status)
{
    __shared__ int sum[kKvMaxSequences + 1];
    __shared__ int warp_sums[32];
    __shared__ float2 red[2 * D / 32];
    const int tid = threadIdx.x, h = blockIdx.y;
    griddep_wait();
    griddep_launch_dependents();
    int bad = 0;
    kv_prefix(c.S, sum, warp_sums, [&](int s) {
        const KvSeq q = kv_seq(c, starts, rows, s);
        bad |= q.n < 0;
        kv_prefetch(c.slot + s);
        return kv_touched(c, q.len, q.n);
    });
    const bool work = (int)blockIdx.x < sum[c.S];
    const int s = work ? kv_find(sum, c.S, (int)blockIdx.x) : 0;
    const KvSeq q = kv_seq(c, starts, rows, s);
    const int slot = c.slot[s];
    bad = __syncthreads_or(bad);  // bounds outside the arrays: nothing is appended
    bool last_reader = false;     // (used at the end: the atomic's latency passes meanwhile)
    if (tid == 0) last_reader = kv_last_reader(c.ticket, gridDim.x * gridDim.y);
    if (!bad && work) {
        const int b0 = q.len / kKvBlock, b = b0 + (int)blockIdx.x - sum[s], last = b0 + sum[s + 1] - sum[s] - 1;
        const int have = b == b0 ? q.len % kKvBlock : 0;                  // rows of the block already there
        const int64_t first = (int64_t)b * kKvBlock - q.len;              // new row index of the block's token 0
        const int end = (int)min((int64_t)kKvBlock, q.n - first);         // present rows
        const int to = (q.len % kKvBlock != 0 && last != b0) ? slot ^ 1 : slot;
        const float* tk = kv_tail(c, s, slot, h, 0);
        const float* tv = kv_tail(c, s, slot, h, 1);
        const int kt = tid / (D / 16), kc = tid % (D / 16), vd = tid % D, vt = tid / D;
        float xk[16], xv[16];
#pragma unroll
        for (int i = 0; i < 16; i++) xk[i] = 0.f;
        if (kt < have) ld16(tk + kt * D + 16 * kc, xk, true);
        else if (kt < end) ld16(k + (q.row0 + first + kt) * ldk + (int64_t)h * D + 16 * kc, xk, veck != 0);
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int t = 16 * vt + i;
            xv[i] = t < have ? tv[t * D + vd] : t < end ? v[(q.row0 + first + t) * ldv + (int64_t)h * D + vd] : 0.f;
        }
        if (b == last) {  // the last block's rows stay at hand in fp32
            float* ok = kv_tail(c, s, to, h, 0);
            float* ov = kv_tail(c, s, to, h, 1);
            if (kt >= have && kt < end) st16(ok + kt * D + 16 * kc, xk, true);
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int t = 16 * vt + i;
                if (t >= have && t < end) ov[t * D + vd] = xv[i];
            }
        }
        kv_store_block<D>(c, (int64_t)s * c.H + h, b, xk, xv, red);
    }
    // every CTA has read the lengths: the last one to do so advances them
    if (!__syncthreads_or(last_reader)) return;
    for (int s = tid; s < c.S; s += blockDim.x) {
        const KvSeq q = kv_seq(c, starts, rows, s);
        if (bad || q.n < 0) {
            atomicCAS(status, 0u, kDevKvStarts);
            continue;
        }
        const int n = kv_touched(c, q.len, q.n);
        if (n) {
            const int last = q.len / kKvBlock + n - 1;
            if (q.len % kKvBlock != 0 && n > 1) c.slot[s] ^= 1;
            c.held[s] = last;
            c.lens[s] = q.len + q.n;
        } else if (q.n > 0) {
            atomicCAS(status, 0u, kDevKvCapacity);
        }
    }
}

template <int D>
__global__ void __launch_bounds__(2 * D) k_kv_truncate(const __grid_constant__ KvView c, const int32_t* lengths)
{
    __shared__ float2 red[2 * D / 32];
    const int tid = threadIdx.x, h = blockIdx.x, s = blockIdx.y;
    griddep_wait();
    griddep_launch_dependents();
    const int len = c.lens[s], to = lengths ? lengths[s] : 0, slot = c.slot[s], holds = c.held[s];
    __syncthreads();
    bool last_reader = false;
    if (tid == 0) last_reader = kv_last_reader(c.ticket, gridDim.x * gridDim.y);
    if (to >= 0 && to < len && to % kKvBlock != 0) {
        const int b = to / kKvBlock, end = to % kKvBlock;
        const int kt = tid / (D / 16), kc = tid % (D / 16), vd = tid % D, vt = tid / D;
        float* tk = kv_tail(c, s, slot, h, 0);
        float* tv = kv_tail(c, s, slot, h, 1);
        const int64_t sh = (int64_t)s * c.H + h;
        float xk[16], xv[16];
        const bool held = holds == b;
        if (held) {
            ld16(tk + kt * D + 16 * kc, xk, true);
#pragma unroll
            for (int i = 0; i < 16; i++) xv[i] = tv[(16 * vt + i) * D + vd];
        } else {
            kv_values<D>(c, sh, b, xk, xv);
        }
#pragma unroll
        for (int i = 0; i < 16; i++) {
            if (kt >= end) xk[i] = 0.f;
            if (16 * vt + i >= end) xv[i] = 0.f;
        }
        if (!held) {
            st16(tk + kt * D + 16 * kc, xk, true);
#pragma unroll
            for (int i = 0; i < 16; i++) tv[(16 * vt + i) * D + vd] = xv[i];
        }
        __syncthreads();  // every code of the block is read
        kv_store_block<D>(c, sh, b, xk, xv, red);
    }
    if (!__syncthreads_or(last_reader)) return;
    for (int i = tid; i < c.S; i += blockDim.x) {
        const int n = c.lens[i], t = lengths ? lengths[i] : 0;
        if (t < 0 || t >= n) continue;
        c.lens[i] = t;
        if (t % kKvBlock != 0) c.held[i] = t / kKvBlock;
        else if (c.held[i] != t / kKvBlock - 1) c.held[i] = -1;
    }
}

template <int D>
__global__ void __launch_bounds__(2 * D) k_kv_read(const __grid_constant__ KvView c, const int32_t* first, int64_t count,
                                                    float* k, float* v, int vec)
{
    const int tid = threadIdx.x, h = blockIdx.y, s = blockIdx.z;
    griddep_wait();
    griddep_launch_dependents();
    const int64_t f = first ? first[s] : 0, len = c.lens[s];
    if (f < 0) return;
    const int64_t b = f / kKvBlock + blockIdx.x;
    const int64_t end = min(f + count, len);  // tokens [f, end) are wanted
    if (b * kKvBlock >= end) return;
    const int kt = tid / (D / 16), kc = tid % (D / 16), vd = tid % D, vt = tid / D;
    float xk[16], xv[16];
    kv_values<D>(c, (int64_t)s * c.H + h, (int)b, xk, xv);
    const int64_t ld = (int64_t)c.H * D, row = s * count + b * kKvBlock - f, t0 = b * kKvBlock;
    if (k && t0 + kt >= f && t0 + kt < end) st16(k + (row + kt) * ld + (int64_t)h * D + 16 * kc, xk, vec != 0);
    if (!v) return;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int t = 16 * vt + i;
        if (t0 + t >= f && t0 + t < end) v[(row + t) * ld + (int64_t)h * D + vd] = xv[i];
    }
}

// Order-preserving integer of a weight; NaN and -inf tie, -0 and +0 tie.
__device__ __forceinline__ uint32_t kv_order(float w)
{
    if (isnan(w)) w = -INFINITY;
    const uint32_t u = __float_as_uint(w + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The kept tokens of one (head, sequence), ascending: the last `recent` ones
// and the keep - recent largest weights of the others.  The border value is
// found by three histogram passes (11, 11 and 10 bits of the ordered
// integer), then one pass in index order writes what lies above it and the
// first ties.  Integer counts only, so the result is exact.
constexpr int SEL_THREADS = 1024, SEL_ITEMS = 4, SEL_BINS = 2048;

__global__ void __launch_bounds__(SEL_THREADS)
    k_kv_select(const __grid_constant__ KvView c, const __grid_constant__ KvView dst, const float* weights, int keep,
                int recent, float* weights_out, int32_t* kept)
{
    __shared__ uint32_t bins[SEL_BINS];
    __shared__ uint32_t warp_sums[32], found[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, h = blockIdx.x, s = blockIdx.y;
    griddep_wait();
    griddep_launch_dependents();
    const int64_t sh = (int64_t)s * c.H + h;
    const int len = c.lens[s], count = min(len, keep), rec = min(recent, count), old = len - rec;
    const float* w = weights + sh * c.cap;
    kept += sh * keep;
    float* wo = weights_out ? weights_out + sh * dst.cap : nullptr;
    if (h == 0 && tid == 0) {
        dst.lens[s] = count;
        dst.slot[s] = 0;
        dst.held[s] = count ? (count - 1) / kKvBlock : -1;
    }
    uint32_t border = 0, ties = 0xffffffffu;  // keep every value above `border` and the first `ties` equal to it
    if (len > keep) {
        uint32_t want = (uint32_t)(count - rec), mask = 0;
        if (want == 0) {
            border = 0xffffffffu;
            ties = 0;
        }
        for (int pass = 0; pass < 3 && want; pass++) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass == 2 ? 1024 : 2048;
            for (int i = tid; i < SEL_BINS; i += SEL_THREADS) bins[i] = 0;
            __syncthreads();
            for (int i = tid; i < old; i += SEL_THREADS) {
                const uint32_t u = kv_order(w[i]);
                if ((u & mask) == border) atomicAdd(&bins[(u >> shift) & (width - 1)], 1u);
            }
            __syncthreads();
            // the bin that holds the want-th largest: counts from the top, two bins per thread
            const int hi = SEL_BINS - 1 - 2 * tid;
            const uint32_t a = bins[hi], b = bins[hi - 1];
            uint32_t v = a + b;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const uint32_t x = __shfl_up_sync(0xffffffffu, v, off);
                if (lane >= off) v += x;
            }
            if (lane == 31) warp_sums[warp] = v;
            __syncthreads();
            for (int i = 0; i < warp; i++) v += warp_sums[i];
            const uint32_t before = v - a - b;
            if (before < want && want <= before + a) {
                found[0] = (uint32_t)hi;
                found[1] = want - before;
            } else if (before + a < want && want <= v) {
                found[0] = (uint32_t)hi - 1;
                found[1] = want - before - a;
            }
            __syncthreads();
            border |= found[0] << shift;
            mask |= (uint32_t)(width - 1) << shift;
            want = found[1];
            __syncthreads();
        }
        if (count > rec) ties = want;
    }
    // one pass in order: kept tokens so far, ties so far
    uint32_t sel = 0, tied = 0;
    for (int base = 0; base < len; base += SEL_THREADS * SEL_ITEMS) {
        uint32_t above[SEL_ITEMS], equal[SEL_ITEMS], mine = 0;  // counts: above in the low half, equal in the high half
        float x[SEL_ITEMS];
#pragma unroll
        for (int i = 0; i < SEL_ITEMS; i++) {
            const int t = base + tid * SEL_ITEMS + i;
            x[i] = t < len ? w[t] : 0.f;
            const uint32_t u = kv_order(x[i]);
            above[i] = t < len && (t >= old || u > border);
            equal[i] = t < old && u == border;
            mine += above[i] | equal[i] << 16;
        }
        uint32_t v = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, v, off);
            if (lane >= off) v += y;
        }
        if (lane == 31) warp_sums[warp] = v;
        __syncthreads();
        uint32_t before = v - mine, all = 0;
        for (int i = 0; i < 32; i++) {
            const uint32_t y = warp_sums[i];
            if (i < warp) before += y;
            all += y;
        }
        uint32_t na = sel + (before & 0xffffu), ne = tied + (before >> 16);
#pragma unroll
        for (int i = 0; i < SEL_ITEMS; i++) {
            const bool take = above[i] || (equal[i] && ne < ties);
            if (take) {
                const uint32_t at = na + min(ne, ties);
                kept[at] = base + tid * SEL_ITEMS + i;
                if (wo) wo[at] = x[i];
            }
            na += above[i];
            ne += equal[i];
        }
        sel += all & 0xffffu;
        tied += all >> 16;
        __syncthreads();
    }
}

template <int D>
__global__ void __launch_bounds__(2 * D) k_kv_compact(const __grid_constant__ KvView c, const __grid_constant__ KvView dst,
                                                      const int32_t* kept, int keep)
{
    __shared__ float2 red[2 * D / 32];
    __shared__ int from[kKvBlock];
    __shared__ float2 scale[kKvBlock];
    const int tid = threadIdx.x, b = blockIdx.x, h = blockIdx.y, s = blockIdx.z;
    griddep_wait();
    griddep_launch_dependents();
    const int count = min(c.lens[s], keep);
    if (b * kKvBlock >= count) return;
    const int64_t sh = (int64_t)s * c.H + h;
    if (tid < kKvBlock) {
        const int i = b * kKvBlock + tid;
        const int t = i < count ? kept[sh * keep + i] : -1;
        from[tid] = t;
        if (t >= 0) scale[tid] = c.scales[sh * c.nb + t / kKvBlock];
    }
    __syncthreads();
    const int kt = tid / (D / 16), kc = tid % (D / 16), vd = tid % D, vt = tid / D;
    const uint8_t* base = c.codes + sh * c.nb * kv_record_bytes(D);
    float xk[16], xv[16];
#pragma unroll
    for (int i = 0; i < 16; i++) xk[i] = 0.f;
    if (from[kt] >= 0) {
        const int t = from[kt];
        const uint8_t* rec = base + (int64_t)(t / kKvBlock) * kv_record_bytes(D);
        uint32_t w[4];
        if (D % 64 != 0 && kc >= D / 64 * 4) {
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = *reinterpret_cast<const uint32_t*>(rec + kv_k_offset<D>(t % kKvBlock, 16 * kc + 4 * i));
        } else {
            const uint4 u = *reinterpret_cast<const uint4*>(rec + kv_k_offset<D>(t % kKvBlock, 16 * kc));
            w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) xk[i] = __fmul_rn((float)((int)((w[i / 4] >> (8 * (i % 4))) & 255u) - 128), scale[kt].x);
    }
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int t = from[16 * vt + i];
        xv[i] = 0.f;
        if (t >= 0) {
            const uint8_t q = base[(int64_t)(t / kKvBlock) * kv_record_bytes(D) + kv_v_offset<D>(t % kKvBlock, vd)];
            xv[i] = __fmul_rn((float)((int)q - 128), scale[16 * vt + i].y);
        }
    }
    if (b == (count - 1) / kKvBlock) {
        st16(kv_tail(dst, s, 0, h, 0) + kt * D + 16 * kc, xk, true);
        float* tv = kv_tail(dst, s, 0, h, 1);
#pragma unroll
        for (int i = 0; i < 16; i++) tv[(16 * vt + i) * D + vd] = xv[i];
    }
    kv_store_block<D>(dst, sh, b, xk, xv, red);
}

template <typename F>
cudaError_t by_dim(int D, F f)
{
    switch (D) {
    case 64: return f(std::integral_constant<int, 64>{});
    case 80: return f(std::integral_constant<int, 80>{});
    case 128: return f(std::integral_constant<int, 128>{});
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace

size_t kv_layout(int64_t S, int64_t H, int64_t D, int64_t cap, uint8_t* base, KvView* v)
{
    const int64_t nb = (cap + kKvBlock - 1) / kKvBlock;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at += (bytes + 255) / 256 * 256;
        return o;
    };
    // the first three are zeroed when the cache is created
    const size_t lens = take(256 + (size_t)S * 12), scales = take((size_t)(S * H * nb) * sizeof(float2)),
                 tail = take((size_t)(S * 2 * H * 2 * kKvBlock * D) * sizeof(float)), codes = take((size_t)(S * H * nb) * 64 * D);
    if (base) {
        v->ticket = reinterpret_cast<uint32_t*>(base + lens);
        v->lens = reinterpret_cast<int32_t*>(base + lens + 256);
        v->slot = v->lens + S;
        v->held = v->slot + S;
        v->scales = reinterpret_cast<float2*>(base + scales);
        v->tail = reinterpret_cast<float*>(base + tail);
        v->codes = base + codes;
        v->S = (int)S;
        v->H = (int)H;
        v->D = (int)D;
        v->cap = (int)cap;
        v->nb = (int)nb;
    }
    return at;
}

cudaError_t launch_kv_append(const KvView& c, const float* k, int64_t ldk, const float* v, int64_t ldv, int64_t rows,
                             const int32_t* starts, uint32_t* status, cudaStream_t s)
{
    // a sequence's n rows touch at most n / 32 + 2 blocks, and at most n
    const int64_t units = std::min(rows, rows / kKvBlock + 2 * (int64_t)c.S);
    const int veck = ((reinterpret_cast<uintptr_t>(k) & 15) == 0 && ldk % 4 == 0) ? 1 : 0;
    return by_dim(c.D, [&](auto d) {
        constexpr int D = decltype(d)::value;
        return launch_pdl(k_kv_append<D>, dim3((unsigned)units, (unsigned)c.H), dim3(2 * D), 0, s, c, k, ldk, v, ldv, rows, starts,
                          veck, status);
    });
}

cudaError_t launch_kv_truncate(const KvView& c, const int32_t* lengths, cudaStream_t s)
{
    return by_dim(c.D, [&](auto d) {
        constexpr int D = decltype(d)::value;
        return launch_pdl(k_kv_truncate<D>, dim3((unsigned)c.H, (unsigned)c.S), dim3(2 * D), 0, s, c, lengths);
    });
}

cudaError_t launch_kv_read(const KvView& c, const int32_t* first, int64_t count, float* k, float* v, cudaStream_t s)
{
    const int64_t blocks = std::min((count + kKvBlock - 2) / kKvBlock + 1, (int64_t)c.nb);
    const int vec = (reinterpret_cast<uintptr_t>(k) & 15) == 0 ? 1 : 0;
    return by_dim(c.D, [&](auto d) {
        constexpr int D = decltype(d)::value;
        return launch_pdl(k_kv_read<D>, dim3((unsigned)blocks, (unsigned)c.H, (unsigned)c.S), dim3(2 * D), 0, s, c, first, count, k, v,
                          vec);
    });
}

cudaError_t launch_kv_evict(const KvView& src, const KvView& dst, const float* weights, int64_t keep, int64_t recent,
                            float* weights_out, int32_t* kept, cudaStream_t s)
{
    cudaError_t e = launch_pdl(k_kv_select, dim3((unsigned)src.H, (unsigned)src.S), dim3(SEL_THREADS), 0, s, src, dst, weights,
                               (int)keep, (int)recent, weights_out, kept);
    if (e != cudaSuccess) return e;
    const int64_t blocks = (std::min(keep, (int64_t)src.cap) + kKvBlock - 1) / kKvBlock;
    return by_dim(src.D, [&](auto d) {
        constexpr int D = decltype(d)::value;
        return launch_pdl(k_kv_compact<D>, dim3((unsigned)blocks, (unsigned)src.H, (unsigned)src.S), dim3(2 * D), 0, s, src, dst, kept,
                          (int)keep);
    });
}

}  // namespace pxq
