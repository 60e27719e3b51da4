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
//
// All are bound by memory when there is much to move and by their chain of
// dependent loads when there is little: appending 65536 rows (4 heads of 128)
// 91 us = 3.7 TB/s (with the truncation before it), truncating and appending
// one row to each of 8 sequences 7.5 us; reading 8 x 8191 tokens 62 us = 5.4
// TB/s; evicting 8 x 32768 tokens to 8191 103 us: the selection, one CTA per
// (head, sequence), about 29 and the packing 78, each timed alone.
#include <algorithm>
#include <type_traits>
#include "kv_cache.cuh"

namespace pxq {
namespace {

constexpr float kKvTiny = 3.009265538105056e-36f;  // 2^-118: blocks below it are stored as zeros (1 / d stays finite)

// max(m, |a|, |b|), NaN if one of them is.
__device__ __forceinline__ float kv_mag(float m, float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
    return r;
}
// Largest magnitudes of the CTA's K and V values.
__device__ __forceinline__ float2 kv_block_max(float mk, float mv, float2* red)
{
#pragma unroll
    for (int off = 16; off; off >>= 1) {
        mk = kv_mag(mk, __shfl_xor_sync(0xffffffffu, mk, off), 0.f);
        mv = kv_mag(mv, __shfl_xor_sync(0xffffffffu, mv, off), 0.f);
    }
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(mk, mv);
    __syncthreads();
    for (int w = 0; w < (int)(blockDim.x >> 5); w++) {
        mk = kv_mag(mk, red[w].x, 0.f);
        mv = kv_mag(mv, red[w].y, 0.f);
    }
    return make_float2(mk, mv);
}
__device__ __forceinline__ float kv_scale(float a)
{
    if (!(a <= FLT_MAX)) return __int_as_float(0x7fffffff);
    return a < kKvTiny ? 0.f : __fdiv_rn(a, 127.f);
}

// 16 code bytes under scale d (inv = 1 / d rounded): the integers nearest to
// x / d, ties to even, plus 128.  x * inv + 1.5 * 2^23 + 128, rounded once,
// has the code byte in its low bits and is within one of the right integer;
// r = x - q d is exact (|r| < 2 d on the grid of d's last place), so 2 |r| < d
// says that it is right.  Where a value of the thread lies so near to a border
// that this fails, all are settled by comparison.
__device__ __forceinline__ void kv_codes(const float (&x)[16], float d, float inv, uint32_t (&w)[4])
{
    constexpr float kMagic = 12582912.f + 128.f;
    if (!(d > 0.f)) {
        w[0] = w[1] = w[2] = w[3] = 0x80808080u;
        return;
    }
    uint32_t c[16];
    const float half = 0.5f * d;
    bool near = false;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const float m = __fmaf_rn(x[i], inv, kMagic);
        c[i] = __float_as_uint(m);
        near |= fabsf(__fmaf_rn(-(m - kMagic), d, x[i])) >= half;
    }
    if (near) {
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float q = __uint_as_float(c[i]) - kMagic;
            const float r = __fmaf_rn(-q, d, x[i]), e = fabsf(r);
            if (e > half || (e == half && (c[i] & 1u))) q += copysignf(1.f, r);
            c[i] = __float_as_uint(q + kMagic);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        w[i] = __byte_perm(__byte_perm(c[4 * i], c[4 * i + 1], 0x0040), __byte_perm(c[4 * i + 2], c[4 * i + 3], 0x0040), 0x5410);
}
// Byte `sel` (0..7) of (lo, hi) as the number it stands for.
__device__ __forceinline__ float kv_number(uint32_t lo, uint32_t hi, uint32_t sel)
{
    return __uint_as_float(__byte_perm(__byte_perm(lo, hi, sel), 0x4b000000u, 0x7440)) - (8388608.f + 128.f);
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
    for (int i = 0; i < 16; i += 2) {
        mk = kv_mag(mk, xk[i], xk[i + 1]);
        mv = kv_mag(mv, xv[i], xv[i + 1]);
    }
    const float2 m = kv_block_max(mk, mv, red);
    const float dk = kv_scale(m.x), dv = kv_scale(m.y);
    const float ik = dk > 0.f ? __fdiv_rn(1.f, dk) : 0.f, iv = dv > 0.f ? __fdiv_rn(1.f, dv) : 0.f;
    uint8_t* rec = c.codes + (sh * c.nb + b) * kv_record_bytes(D);
    uint32_t w[4];
    kv_codes(xk, dk, ik, w);
    if (D % 64 != 0 && kc >= D / 64 * 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<uint32_t*>(rec + kv_k_offset<D>(kt, 16 * kc + 4 * i)) = w[i];
    } else {
        *reinterpret_cast<uint4*>(rec + kv_k_offset<D>(kt, 16 * kc)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    kv_codes(xv, dv, iv, w);
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
        xk[i] = __fmul_rn(kv_number(w[i / 4], 0, i % 4), d.x);
        xv[i] = __fmul_rn(kv_number(z[i / 4], 0, i % 4), d.y);
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
__global__ void __launch_bounds__(2 * D, 4)
    k_kv_append(const __grid_constant__ KvView c, const float* k, int64_t ldk, const float* v, int64_t ldv,
                int64_t rows, const int32_t* starts, int veck, uint32_t* errors)
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
            atomicAdd(errors + kStatusKvStarts, 1u);
            continue;
        }
        const int n = kv_touched(c, q.len, q.n);
        if (n) {
            const int last = q.len / kKvBlock + n - 1;
            if (q.len % kKvBlock != 0 && n > 1) c.slot[s] ^= 1;
            c.held[s] = last;
            c.lens[s] = q.len + q.n;
        } else if (q.n > 0) {
            atomicAdd(errors + kStatusKvCapacity, 1u);
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
// first ties.  Integer counts only, so the result is exact.  The integers stay
// in shared memory from the first pass on, as many as fit.
constexpr int SEL_THREADS = 1024, SEL_BINS = 2048, SEL_CACHE = 50 * 1024;

// Sum of x[0 .. warp - 1] (warp <= 32 values), by every warp for itself.
__device__ __forceinline__ uint32_t sel_before(const uint32_t* x, int warp, int lane)
{
    uint32_t v = lane < warp ? x[lane] : 0u;
    return __reduce_add_sync(0xffffffffu, v);
}

__global__ void __launch_bounds__(SEL_THREADS)
    k_kv_select(const __grid_constant__ KvView c, const __grid_constant__ KvView dst, const float* weights, int keep,
                int recent, float* weights_out, int32_t* kept)
{
    extern __shared__ uint32_t keys[];  // [min(old, SEL_CACHE)]
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
            auto count_in = [&](uint32_t u) {
                if ((u & mask) == border) atomicAdd(&bins[(u >> shift) & (width - 1)], 1u);
            };
            const int cached = min(old, SEL_CACHE);
            if (pass == 0) {
                for (int i0 = tid; i0 < cached; i0 += 8 * SEL_THREADS) {
                    float x[8];
#pragma unroll
                    for (int k = 0; k < 8; k++) x[k] = i0 + k * SEL_THREADS < cached ? w[i0 + k * SEL_THREADS] : 0.f;
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        if (i0 + k * SEL_THREADS < cached) {
                            const uint32_t u = kv_order(x[k]);
                            keys[i0 + k * SEL_THREADS] = u;
                            count_in(u);
                        }
                }
            } else {
#pragma unroll 4
                for (int i = tid; i < cached; i += SEL_THREADS) count_in(keys[i]);
            }
            for (int i = cached + tid; i < old; i += SEL_THREADS) count_in(kv_order(w[i]));
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
            v += sel_before(warp_sums, warp, lane);
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
    // In order: a warp takes a stretch of the tokens, counts what it keeps and its ties, and writes from where the warps
    // before it end.
    const int stretch = (len + SEL_THREADS - 1) / SEL_THREADS * 32;
    const int first = min(len, warp * stretch), last = min(len, first + stretch);
    const uint32_t below = (1u << lane) - 1u;
    const bool keyed = len > keep && count > rec;  // keys[] holds the first tokens' integers
    const int cached = keyed ? min(old, SEL_CACHE) : 0;
    auto look = [&](int t, uint32_t& above, uint32_t& equal) {
        const uint32_t u = t < cached ? keys[t] : t < old ? kv_order(w[t]) : 0u;
        above = __ballot_sync(0xffffffffu, t < last && (t >= old || u > border));
        equal = __ballot_sync(0xffffffffu, t < last && t < old && u == border);
    };
    uint32_t na = 0, ne = 0;
    for (int t0 = first; t0 < last; t0 += 32) {
        uint32_t above, equal;
        look(t0 + lane, above, equal);
        na += __popc(above);
        ne += __popc(equal);
    }
    __syncthreads();
    if (lane == 0) warp_sums[warp] = na, bins[warp] = ne;
    __syncthreads();
    na = sel_before(warp_sums, warp, lane);
    ne = sel_before(bins, warp, lane);
    for (int t0 = first; t0 < last; t0 += 32) {
        uint32_t above, equal;
        look(t0 + lane, above, equal);
        const uint32_t a = na + __popc(above & below), e = ne + __popc(equal & below);
        if ((above >> lane & 1u) || ((equal >> lane & 1u) && e < ties)) {
            const uint32_t at = a + min(e, ties);
            kept[at] = t0 + lane;
            if (wo) wo[at] = w[t0 + lane];
        }
        na += __popc(above);
        ne += __popc(equal);
    }
}

// NB destination blocks per CTA: their tokens' places and scales are looked up
// at once.  All loads of a block are issued before the first is used, and four
// CTAs share an SM: the kernel waits for memory (8 x 32768 tokens to 8191, 4
// heads of 128: 107 us with the selection when this was measured, 155 us at two CTAs per SM).
template <int D, int NB>
__global__ void __launch_bounds__(2 * D, 4) k_kv_compact(const __grid_constant__ KvView c, const __grid_constant__ KvView dst,
                                                      const int32_t* kept, int keep)
{
    __shared__ float2 red[NB][2 * D / 32];
    __shared__ uint32_t from[NB * kKvBlock];
    __shared__ float2 scale[NB * kKvBlock];
    const int tid = threadIdx.x, h = blockIdx.y, s = blockIdx.z, b0 = blockIdx.x * NB;
    griddep_wait();
    griddep_launch_dependents();
    const int count = min(c.lens[s], keep);
    const int64_t sh = (int64_t)s * c.H + h;
    const int total = min(NB * kKvBlock, count - b0 * kKvBlock);  // tokens of these blocks
    if (total <= 0) return;
    if (tid < NB * kKvBlock) {
        const uint32_t t = kept[sh * keep + b0 * kKvBlock + min(tid, total - 1)];  // (absent ones: a token's bytes all the same)
        from[tid] = t;
        scale[tid] = c.scales[sh * c.nb + t / kKvBlock];
    }
    __syncthreads();
    const int kt = tid / (D / 16), kc = tid % (D / 16), vd = tid % D, vt = tid / D;
    const uint8_t* base = c.codes + sh * c.nb * kv_record_bytes(D);
#pragma unroll 1
    for (int u = 0; u < NB && u * kKvBlock < total; u++) {
        const int here = min(kKvBlock, total - u * kKvBlock);
        const uint32_t* ft = from + u * kKvBlock;
        const float2* sc = scale + u * kKvBlock;
        uint2 g[16];  // V: the group of eight tokens that holds the token
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const uint32_t t = ft[16 * vt + i];
            g[i] = *reinterpret_cast<const uint2*>(base + (int64_t)(t / kKvBlock) * kv_record_bytes(D) + kv_v_offset<D>(t % kKvBlock & ~7u, vd));
        }
        uint32_t w[4];
        {
            const uint32_t t = ft[kt];
            const uint8_t* rec = base + (int64_t)(t / kKvBlock) * kv_record_bytes(D);
            if (D % 64 != 0 && kc >= D / 64 * 4) {
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = *reinterpret_cast<const uint32_t*>(rec + kv_k_offset<D>(t % kKvBlock, 16 * kc + 4 * i));
            } else {
                const uint4 v = *reinterpret_cast<const uint4*>(rec + kv_k_offset<D>(t % kKvBlock, 16 * kc));
                w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
            }
        }
        float xk[16], xv[16];
        const float sk = sc[kt].x;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const uint32_t t = ft[16 * vt + i];
            xk[i] = kt < here ? __fmul_rn(kv_number(w[i / 4], 0, i % 4), sk) : 0.f;
            xv[i] = 16 * vt + i < here ? __fmul_rn(kv_number(g[i].x, g[i].y, t & 7), sc[16 * vt + i].y) : 0.f;
        }
        const int b = b0 + u;
        if (b == (count - 1) / kKvBlock) {
            st16(kv_tail(dst, s, 0, h, 0) + kt * D + 16 * kc, xk, true);
            float* tv = kv_tail(dst, s, 0, h, 1);
#pragma unroll
            for (int i = 0; i < 16; i++) tv[(16 * vt + i) * D + vd] = xv[i];
        }
        kv_store_block<D>(dst, sh, b, xk, xv, red[u]);
    }
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
                             const int32_t* starts, uint32_t* errors, cudaStream_t s)
{
    // a sequence's n rows touch at most n / 32 + 2 blocks, and at most n
    const int64_t units = std::min(rows, rows / kKvBlock + 2 * (int64_t)c.S);
    const int veck = ((reinterpret_cast<uintptr_t>(k) & 15) == 0 && ldk % 4 == 0) ? 1 : 0;
    return by_dim(c.D, [&](auto d) {
        constexpr int D = decltype(d)::value;
        return launch_pdl(k_kv_append<D>, dim3((unsigned)units, (unsigned)c.H), dim3(2 * D), 0, s, c, k, ldk, v, ldv, rows, starts,
                          veck, errors);
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
    static std::atomic<uint32_t> done{0};
    cudaError_t e = allow_smem(k_kv_select, SEL_CACHE * 4, done);
    if (e != cudaSuccess) return e;
    const size_t smem = (size_t)std::min<int64_t>(src.cap, SEL_CACHE) * 4;
    e = launch_pdl(k_kv_select, dim3((unsigned)src.H, (unsigned)src.S), dim3(SEL_THREADS), smem, s, src, dst, weights, (int)keep,
                   (int)recent, weights_out, kept);
    if (e != cudaSuccess) return e;
    const int64_t blocks = (std::min(keep, (int64_t)src.cap) + kKvBlock - 1) / kKvBlock;
    return by_dim(src.D, [&](auto d) {
        constexpr int D = decltype(d)::value;
        // four blocks per CTA once there is work for every SM many times over
        const auto kernel = blocks * src.H * src.S >= 8192 ? k_kv_compact<D, 4> : k_kv_compact<D, 1>;
        const int per = kernel == k_kv_compact<D, 4> ? 4 : 1;
        return launch_pdl(kernel, dim3((unsigned)((blocks + per - 1) / per), (unsigned)src.H, (unsigned)src.S), dim3(2 * D), 0, s, src, dst,
                          (const int32_t*)kept, (int)keep);
    });
}

}  // namespace pxq
