// kv_cache.cuh -- layout of the 8-bit key/value cache and the device code
// its kernels share.
//
// A cache holds S sequences x H key/value heads x NB blocks of 32 tokens.
// X being K or V, block b of (s, h) holds codes q and one fp32 scale d each
// for K and V, and stands for the values fl32(q * d):
//     A = max |X| over the block's present tokens and the D channels
//     d = fl32(A / 127), 0 when A < 2^-118, NaN when some |X| is not finite
//     q = the integer nearest to X / d (ties to even), 0 when d is 0 or NaN
// One NaN scale makes every value of its block NaN: a value that is not
// finite is never lost, and rows that may not see the block do not read it.
// Codes are stored as bytes q + 128, so that two of them become fp16 numbers
// with one byte permute (0x64xx = 1024 + byte) and one subtraction of 1152.
//
// A block's record is 64 * D bytes, the K codes then the V codes, each in the
// order in which a warp's mma.m16n8k16 B fragments take them, so that a
// fragment load is 16 consecutive bytes per lane (lane = 4 n + c):
//   K, token t = 8 (n / 2) + 2 nt + n % 2 (nt = 0..3), channels 64 j + 16 c ..
//      + 15 at 16 ((nt J + j) 32 + lane), J = D / 64; D = 80 has channels
//      64 + 4 c .. + 3 at 64 * 32 + 16 lane + 4 nt.
//   V, channel 8 (2 p + f) + n, tokens 8 c .. + 7 at 32 D + 16 (32 p + lane) + 8 f.
// With these orders lane c of a row's four lanes holds the scores of tokens
// 8 c .. 8 c + 7, which is what its A fragments of the value product need.
//
// The rows of a sequence's last block are also kept in fp32 ("tail", two
// slots; slot[s] names the live one), and an append quantizes the whole
// block anew from them: what a block holds depends on its rows alone, not on
// how the appends cut them.
#pragma once
#include <cfloat>
#include "pxq_device.cuh"
#include "pxq_internal.h"

namespace pxq {

__host__ __device__ constexpr int kv_record_bytes(int D) { return 64 * D; }

// Byte of token t (0..31), channel d within a record.
template <int D>
__device__ __forceinline__ int kv_k_offset(int t, int d)
{
    const int n = 2 * (t / 8) + t % 2, nt = (t % 8) / 2;
    if (D % 64 != 0 && d >= D / 64 * 64) return D / 64 * 64 * 32 + (4 * n + (d - D / 64 * 64) / 4) * 16 + nt * 4 + d % 4;
    return ((nt * (D / 64) + d / 64) * 32 + 4 * n + d % 64 / 16) * 16 + d % 16;
}
template <int D>
__device__ __forceinline__ int kv_v_offset(int t, int d)
{
    return 32 * D + (d / 16 * 32 + 4 * (d % 8) + t / 8) * 16 + d % 16 / 8 * 8 + t % 8;
}

// Sequence s of a ragged batch: its cached tokens and its rows
// [row0, row0 + n) of the packed arrays.  n = -1: its bounds are not within
// the arrays.  EARLY: a kernel that has not waited for its predecessors yet
// (whoever wrote the lengths and the starts is over, but L1 may hold older
// ones) takes them from L2.
struct KvSeq {
    int len, n, row0;
};
template <bool EARLY = false>
__device__ __forceinline__ KvSeq kv_seq(const KvView& c, const int32_t* starts, int64_t rows, int s)
{
    KvSeq q;
    q.len = EARLY ? __ldcg(c.lens + s) : c.lens[s];
    if (starts) {
        const int a = EARLY ? __ldcg(starts + s) : starts[s], b = EARLY ? __ldcg(starts + s + 1) : starts[s + 1];
        q.row0 = a;
        q.n = (a < 0 || b < a || b > rows) ? -1 : b - a;
    } else {
        const int n = (int)rows / c.S;
        q.row0 = s * n;
        q.n = n;
    }
    return q;
}

// sum[s] = f(0) + .. + f(s - 1) for s <= S, computed by the whole CTA
// (blockDim.x a multiple of 32, at most 1024); ends with a barrier.  f may be
// evaluated by any number of threads.
template <typename F>
__device__ __forceinline__ void kv_prefix(int S, int* sum, int* warp_sums, F f)
{
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    if (S == 1) {
        const int x = f(0);
        if (tid == 0) sum[0] = 0, sum[1] = x;
        __syncthreads();
        return;
    }
    if (S <= 32) {
        if (warp == 0) {
            const int x = lane < S ? f(lane) : 0;
            int v = x;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, off);
                if (lane >= off) v += u;
            }
            if (lane < S) sum[lane] = v - x;
            if (lane == 31) sum[S] = v;
        }
        __syncthreads();
        return;
    }
    int carry = 0;
    for (int base = 0; base < S; base += blockDim.x) {
        const int s = base + tid;
        const int x = s < S ? f(s) : 0;
        int v = x;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v, off);
            if (lane >= off) v += u;
        }
        if (lane == 31) warp_sums[warp] = v;
        __syncthreads();
        int before = carry, all = 0;
        for (int w = 0; w < warps; w++) {
            const int u = warp_sums[w];
            if (w < warp) before += u;
            all += u;
        }
        if (s < S) sum[s] = before + v - x;
        carry += all;
        __syncthreads();
    }
    if (tid == 0) sum[S] = carry;
    __syncthreads();
}

// The s with sum[s] <= u < sum[s + 1]  (u < sum[S]).
__device__ __forceinline__ int kv_find(const int* sum, int S, int u)
{
    int lo = 0, hi = S;  // sum[lo] <= u < sum[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (sum[mid] <= u) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Count this CTA as one that has read the lengths (called by one thread after
// a barrier behind those reads).  Returns whether it is the last of the grid:
// the one that may write them, as soon as it likes.  Leaves the ticket at zero.
// The reads of every CTA come before the last one's writes: each count is a
// release, and the last CTA alone, after it, acquires (an acquire in every CTA
// empties the L1 caches: 99 us instead of 91 for 65536 rows).
__device__ __forceinline__ bool kv_last_reader(uint32_t* ticket, uint32_t ctas)
{
    uint32_t t;
    asm volatile("atom.release.gpu.global.add.u32 %0, [%1], 1;" : "=r"(t) : "l"(ticket) : "memory");
    if (t != ctas - 1) return false;
    asm volatile("fence.acq_rel.gpu;" ::: "memory");
    *ticket = 0;
    return true;
}
__device__ __forceinline__ void kv_prefetch(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }

__device__ __forceinline__ float kv_log2_inv_sqrt(int D) { return 1.4426950408889634f / sqrtf((float)D); }

__device__ __forceinline__ float kv_ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^e for -126 <= e <= 127
__device__ __forceinline__ float kv_pow2(int e) { return __int_as_float((e + 127) << 23); }
// |x| < 2^this; -126 for 0, 129 for what is not finite
__device__ __forceinline__ int kv_exponent(float x) { return (int)(__float_as_uint(x) >> 23 & 255u) - 126; }

// The unit of a row's value sums.  p dv goes to the tensor core as two fp16
// numbers, whose floor is absolute, so each row has a unit of its own, 2^(E - 15)
// with 2^E at least the row's largest p dv so far among the blocks that it
// sees (p relative to its running max): a block that a row may not see, or to
// which it gives next to no weight, takes no bits from the others.
// E = kv_unit(t), t that p dv's log2, dv rounded up to 2^ev: kept relative to the
// running max, so that large scores leave it its bits, and never below a seen
// block's ev - kUnitSpan, so that dv over the unit stays below 2^127 whatever the p
// (a row that sees blocks whose scales differ by more than 2^128 loses bits of the lesser ones).
constexpr int kNoUnit = -237;  // nothing seen yet; 15 - E stays below 253
constexpr float kUnitSpan = 111.f;
__device__ __forceinline__ int kv_unit(float t) { return max(kNoUnit, __float2int_ru(t)); }
// t behind a block of largest score z (-inf: not seen) and scale exponent ev, the
// running max having gone from `was` to `now` (0 where it is still -inf)
__device__ __forceinline__ float kv_unit_log(float t, float was, float now, float z, float ev)
{
    return fmaxf(t - (now - was), z - now + ev);
}
// ev, dv < 2^ev: -inf for a NaN scale
__device__ __forceinline__ float kv_scale_log(float dv)
{
    const int ev = kv_exponent(dv);
    return ev < 129 ? (float)ev : -INFINITY;
}
// 2^e, |e| <= 252, as two factors, neither of which leaves fp32's range
__device__ __forceinline__ float2 kv_pow2_pair(int e)
{
    const int a = e >> 1;
    return make_float2(kv_pow2(a), kv_pow2(e - a));
}
// what the sums so far are multiplied by as the unit's exponent falls by d (or rises by -d) and the running max's p
// becomes corr
__device__ __forceinline__ float kv_unit_step(float corr, int d)
{
    const float2 f = kv_pow2_pair(max(-252, min(252, d)));
    return corr * f.x * f.y;
}
// 2^(E - 15), what the sums are multiplied by in the end (E >= -126, or nothing is seen)
__device__ __forceinline__ float kv_unit_value(int E)
{
    const int e = max(-149, E - 15);
    return e >= -126 ? kv_pow2(e) : __int_as_float(1 << (e + 149));
}

__device__ __forceinline__ uint32_t kv_pack(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// (a, b) = hi + lo, each a pair of fp16 numbers
__device__ __forceinline__ void kv_split(float a, float b, uint32_t& hi, uint32_t& lo)
{
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    ffma2(a, b, f.x, f.y, -1.f, -1.f);
    lo = kv_pack(a, b);
}

// Tokens that row i of sequence q sees.
__device__ __forceinline__ int kv_limit(const KvAttnCall& a, const KvSeq& q, int i)
{
    return a.causal ? max(0, q.len - q.n + i + 1) : q.len;
}

// Two fp16 numbers from two code bytes (b0, b1 or b2, b3 of w).
__device__ __forceinline__ uint32_t kv_half2(uint32_t w, uint32_t sel)
{
    uint32_t r = __byte_perm(w, 0x64646464u, sel);
    __half2 h = __hsub2(*reinterpret_cast<__half2*>(&r), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t kv_half2_lo(uint32_t w) { return kv_half2(w, 0x4140); }
__device__ __forceinline__ uint32_t kv_half2_hi(uint32_t w) { return kv_half2(w, 0x4342); }

}  // namespace pxq
