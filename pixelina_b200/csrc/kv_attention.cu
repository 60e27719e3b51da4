// kv_attention.cu -- softmax attention over the 8-bit key/value cache
// (kv_cache.cuh), and the weight that each cached token receives.
//
// Query row i of a sequence with n rows and len tokens sees the tokens
// j < L(i) = len (or len - n + i + 1 when causal):
//     z_j = (q . k_j) dk / sqrt(D),  p_j = exp(z_j - max) / sum,  out = sum_j p_j dv v_j
// with k, v the codes and dk, dv their blocks' scales; L <= 0 gives zeros.
// A pair is (query row, head of the kv head's group): pairs p = i * G + g are
// the rows of the matrix products, so every key is read once for the group.
//
// Accuracy: codes are exact in fp16.  q and p dv, brought to below 2^15 by
// powers of two (p dv per pair: kv_unit), are each the sum of two fp16 numbers,
// hi + lo.  That leaves 2^-22 of the value, or 2^-40 of the pair's largest where
// that is more; products and sums are fp32.  So the result is that of an fp32
// computation at two half-precision products per element.
//
//   k_kv_attn     split keys, up to 16 pairs per tile: a CTA takes a part of
//                 a (sequence, head)'s blocks (kv_divide), its warps the
//                 part's blocks in turn, each with a max and a sum of its own;
//                 a lane's fragments are 16 consecutive bytes of a record
//   k_kv_combine  joins the parts of a (sequence, head) that spans CTAs
//   k_kv_weights  the weights, from each pair's max and sum
//
// What bounds k_kv_attn: reading the cache once, 2 len D bytes per (sequence,
// head).  8 x 49000 tokens, 28 heads over 4 of 128: 70.9 us, 5.7 TB/s of 6.5.
// Per block of 32 tokens a warp has 64 products (8 cycles each and SM
// quarter) and, counted in the source, some 470 instructions, about half of
// them turning codes into fp16; the registers leave room for two warps per
// quarter.  With little to read the two kernels' chains of dependent steps
// bound it (lengths, queries, copies, join): 8 x 3000 tokens 13.8 us, 1 x 1000
// 8.7 us.
#include <algorithm>
#include <type_traits>
#include "kv_cache.cuh"

namespace pxq {
namespace {

constexpr int AW = 4;                    // warps per CTA
constexpr int kCtasPerSm = 2;            // one joins its warps or waits for queries while the other streams
constexpr int kMinRun = 4;               // fewest blocks worth a CTA: one per warp

// D += A (16 x 16, row) * B (16 x 8, column), fp16 in, fp32 out
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct AttnParams {
    KvAttnCall a;
    float* part;   // partial results: [pair tile][CTA][2] x {m[PT], l[PT], (O / l)[PT][D]}
    float* lse;    // [rows][heads] log2 of the softmax's denominator with its max, when weights are wanted
    int runs;      // CTAs of the flattened list
};

// Blocks of sequence s: 0 when it has no rows to answer.  An empty cache
// counts one (fully masked) block, so that its rows get their zeros.
template <bool EARLY>
__device__ __forceinline__ int kv_attn_blocks(const KvAttnCall& a, int s)
{
    const KvSeq q = kv_seq<EARLY>(a.c, a.starts, a.rows, s);
    if (q.n <= 0 || q.n > a.max_rows) return 0;
    return max(1, (q.len + kKvBlock - 1) / kKvBlock);
}
// How the CTAs divide the (sequence, head)s' blocks.  Taking up another
// (sequence, head) costs a CTA about as much as kSegmentCost blocks (queries
// to fetch and split, warps to join), so each is cut into equal parts of its
// own, a part per CTA, as many as the CTAs allow: with T blocks, N CTAs and n
// (sequence, head)s, parts of T / (N - n) blocks always fit.  Where that makes
// them longer than an equal share T / N by more than kSegmentCost, CTA i takes
// blocks [i run, (i + 1) run) of the flattened list instead, whatever they
// belong to.
constexpr int kSegmentCost = 10;
struct KvDivision {
    int part;  // most blocks of a part, sum[s]: parts before sequence s; 0: the flattened list
    int run;   // flattened: blocks per CTA, sum[s]: blocks before sequence s
};
template <bool EARLY = false>
__device__ __forceinline__ KvDivision kv_divide(const KvAttnCall& a, int runs, int* sum, int* warp_sums)
{
    const int S = a.c.S, H = a.c.H, n = S * H;
    auto decide = [&](int total) {
        KvDivision d;
        d.run = max(kMinRun, (total + runs - 1) / runs);
        d.part = n < runs ? max(kMinRun, (total + runs - n - 1) / (runs - n)) : 0;
        if (d.part - d.run > kSegmentCost) d.part = 0;
        return d;
    };
    if (S == 1) {
        const int nb = kv_attn_blocks<EARLY>(a, 0);
        const KvDivision d = decide(nb * H);
        if (threadIdx.x == 0) sum[0] = 0, sum[1] = (d.part ? (nb + d.part - 1) / d.part : nb) * H;
        __syncthreads();
        return d;
    }
    kv_prefix(S, sum, warp_sums, [&](int s) { return kv_attn_blocks<EARLY>(a, s) * H; });
    const KvDivision d = decide(sum[S]);
    if (d.part) {
        __syncthreads();  // everyone has read the total
        kv_prefix(S, sum, warp_sums, [&](int s) { return (kv_attn_blocks<EARLY>(a, s) + d.part - 1) / d.part * H; });
    }
    return d;
}

// One warp's A fragments of up to PT pairs' queries: PT = 8 packs hi into
// rows 0-7 and lo into rows 8-15 of one fragment, PT = 16 keeps two.
// coef[r]: log2(e) / sqrt(D) over the pair's power of two.
template <int D, int PT>
struct QFrag {
    uint32_t hi[D / 16][4];
    uint32_t lo[PT == 16 ? D / 16 : 1][4];
    float coef[PT / 8];

    // EARLY: the kernel has not waited for its predecessors yet (who wrote q is over, but L1 may hold older rows)
    template <bool EARLY = false>
    __device__ __forceinline__ void load(const KvAttnCall& a, const KvSeq& q, int h, int tile)
    {
        const int lane = lane_id(), r = lane / 4, c = lane % 4, G = a.G, pairs = q.n * G;
#pragma unroll
        for (int u = 0; u < PT / 8; u++) {
            const int p = tile * PT + r + 8 * u;
            const bool live = p < pairs;
            const float* src = a.q + (int64_t)(q.row0 + (live ? p / G : 0)) * a.ldq + (int64_t)(h * G + (live ? p % G : 0)) * D;
            float m = 0.f;
            float x[D / 16][4];
            auto fetch = [&](auto vec) {
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    const int d = k < D / 64 * 4 ? 64 * (k / 4) + 16 * c + 4 * (k % 4) : D / 64 * 64 + 4 * c;
                    float4 v;
                    if (decltype(vec)::value) v = EARLY ? __ldcg(reinterpret_cast<const float4*>(src + d)) : *reinterpret_cast<const float4*>(src + d);
                    else if (EARLY) v = make_float4(__ldcg(src + d), __ldcg(src + d + 1), __ldcg(src + d + 2), __ldcg(src + d + 3));
                    else v = make_float4(src[d], src[d + 1], src[d + 2], src[d + 3]);
                    x[k][0] = v.x, x[k][1] = v.y, x[k][2] = v.z, x[k][3] = v.w;
                }
            };
            if (!live) {
#pragma unroll
                for (int k = 0; k < D / 16; k++) x[k][0] = x[k][1] = x[k][2] = x[k][3] = 0.f;
            } else if (a.qvec) {
                fetch(std::true_type{});
            } else {
                fetch(std::false_type{});
            }
#pragma unroll
            for (int k = 0; k < D / 16; k++)
                m = fmaxf(m, fmaxf(fmaxf(fabsf(x[k][0]), fabsf(x[k][1])), fmaxf(fabsf(x[k][2]), fabsf(x[k][3]))));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            // |x| 2^e < 2^15; a row of zeros, or one that is not finite, stays as it is
            const int e = m > 0.f && m <= FLT_MAX ? max(-113, min(110, 15 - kv_exponent(m))) : 0;
            const float up = kv_pow2(e);
            coef[u] = kv_log2_inv_sqrt(D) * kv_pow2(-e);
#pragma unroll
            for (int k = 0; k < D / 16; k++) {
                uint32_t h0, l0, h1, l1;
                kv_split(x[k][0] * up, x[k][1] * up, h0, l0);
                kv_split(x[k][2] * up, x[k][3] * up, h1, l1);
                if (PT == 8) {
                    hi[k][0] = h0, hi[k][1] = l0, hi[k][2] = h1, hi[k][3] = l1;
                } else {
                    hi[k][u] = h0, hi[k][2 + u] = h1;
                    lo[k][u] = l0, lo[k][2 + u] = l1;
                }
            }
        }
    }
};

// Scores of a block's 32 tokens: z[u][8] of pair row r + 8 u, tokens 8 c ..
// 8 c + 7, before the scales.  words(i): the lane's 16 bytes i (of D / 16) of
// the block's K codes.
template <int D, int PT, typename F>
__device__ __forceinline__ void block_scores(const QFrag<D, PT>& q, F words, float (&z)[PT / 8][8])
{
    constexpr int J = D / 64;
    float s[4][4];
#pragma unroll
    for (int nt = 0; nt < 4; nt++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[nt][i] = 0.f;
    // the four token groups' sums are independent: their products take turns, so that none waits for the one before it
#pragma unroll
    for (int j = 0; j < J; j++) {
        uint4 w[4];
#pragma unroll
        for (int nt = 0; nt < 4; nt++) w[nt] = words(nt * J + j);
#pragma unroll
        for (int k = 0; k < 4; k++) {
#pragma unroll
            for (int nt = 0; nt < 4; nt++) {
                const uint32_t ww = k == 0 ? w[nt].x : k == 1 ? w[nt].y : k == 2 ? w[nt].z : w[nt].w;
                const uint32_t b0 = kv_half2_lo(ww), b1 = kv_half2_hi(ww);
                mma16816(s[nt], q.hi[4 * j + k], b0, b1);
                if (PT == 16) mma16816(s[nt], q.lo[4 * j + k], b0, b1);
            }
        }
    }
    if (D % 64 != 0) {
        const uint4 w = words(4 * J);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int nt = 0; nt < 4; nt++) {
            const uint32_t b0 = kv_half2_lo(ww[nt]), b1 = kv_half2_hi(ww[nt]);
            mma16816(s[nt], q.hi[4 * J], b0, b1);
            if (PT == 16) mma16816(s[nt], q.lo[PT == 16 ? 4 * J : 0], b0, b1);
        }
    }
#pragma unroll
    for (int nt = 0; nt < 4; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            if (PT == 8) {
                z[0][2 * nt + e] = s[nt][e] + s[nt][2 + e];
            } else {
                z[0][2 * nt + e] = s[nt][e];
                z[PT / 8 - 1][2 * nt + e] = s[nt][2 + e];
            }
        }
}

constexpr int kAttnStages = 2;  // blocks in flight per warp
// The tensor core cuts an accumulator's last bits at every step, always towards
// zero; over the 80 steps that a warp takes for 8 x 65536 tokens that cost
// 2e-6 of the output's norm, twice what fp32 arithmetic loses.  So a warp's
// sums go to shared memory, rounded to nearest, every kFlush blocks.
constexpr int kFlush = 8;
// a warp's sums: m[PT], l[PT], O[PT][D + 8] (rows eight words apart modulo 32: float2 accesses without conflicts)
template <int D, int PT>
constexpr int attn_sum_floats() { return PT * (D + 10); }
template <int D, int PT>
constexpr size_t attn_smem_bytes() { return (size_t)AW * (kAttnStages * kv_record_bytes(D) + attn_sum_floats<D, PT>() * sizeof(float)); }

template <int D, int PT>
__global__ void __launch_bounds__(AW * 32, kCtasPerSm) k_kv_attn(const __grid_constant__ AttnParams P)
{
    constexpr int NST = kAttnStages, REC = kv_record_bytes(D), U = PT / 8, NT = D / 8;
    constexpr int CW = attn_sum_floats<D, PT>(), DS = D + 8;
    extern __shared__ __align__(128) uint8_t dyn[];
    __shared__ int sum[kKvMaxSequences + 1];
    __shared__ int warp_sums[32];
    __shared__ uint64_t bars[AW][NST];
    __shared__ uint32_t abort_flag;
    const KvAttnCall& a = P.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane / 4, c = lane % 4;
    const int tile = blockIdx.y, G = a.G;
    uint8_t* ring = dyn + warp * NST * REC;
    float* comb = reinterpret_cast<float*>(dyn + AW * NST * REC);
    float* mine = comb + warp * CW;
    float2* acc = reinterpret_cast<float2*>(mine + 2 * PT + r * DS + 2 * c);  // this lane's part of its pairs' sums
    if (tid == 0) abort_flag = 0;
    if (lane == 0) {
        for (int i = 0; i < NST; i++) mbar_init(&bars[warp][i], 1);
        fence_mbar_init();
    }
    griddep_wait();
    griddep_launch_dependents();
    const KvDivision dv = kv_divide(a, P.runs, sum, warp_sums);
    const int total = sum[a.c.S], run = dv.part ? 1 : dv.run;  // units: parts, or blocks
    if (blockIdx.x == 0 && blockIdx.y == 0)
        for (int s = tid; s < a.c.S; s += AW * 32) {
            const int n = kv_seq(a.c, a.starts, a.rows, s).n;
            if (n < 0 || n > a.max_rows) atomicAdd(a.status + kStatusKv + kStatusKvStarts, 1u);
        }
    const int w0 = (int)blockIdx.x * run, w1 = min(total, w0 + run);
    uint32_t phase = 0;  // bit i: parity of stage i

    for (int w = w0; w < w1;) {
        const int s = kv_find(sum, a.c.S, w);
        const KvSeq q = kv_seq(a.c, a.starts, a.rows, s);
        const int nb = max(1, (q.len + kKvBlock - 1) / kKvBlock);
        const int room = (sum[s + 1] - sum[s]) / a.c.H;  // units per head
        const int h = (w - sum[s]) / room, seg = sum[s] + h * room;
        int b0, b1;  // this (sequence, head)'s blocks [b0, b1) of nb
        if (dv.part) {
            const int each = (nb + room - 1) / room;
            b0 = min(nb, (w - seg) * each);
            b1 = min(nb, b0 + each);
            w++;
        } else {
            b0 = w - seg;
            b1 = min(nb, w1 - seg);
            w = seg + b1;
        }
        const bool first = dv.part || b0 > 0, whole = b0 == 0 && b1 == nb;  // first: of the CTA's two places for parts
        const int pairs = q.n * G;
        if (tile * PT >= pairs) continue;
        const uint8_t* recs = a.c.codes + ((int64_t)s * a.c.H + h) * a.c.nb * (int64_t)REC;
        const float2* scales = a.c.scales + ((int64_t)s * a.c.H + h) * a.c.nb;

        int issued = b0 + warp;
        auto issue = [&](int st) {
            if (lane == 0 && issued < b1) {
                mbar_expect_tx(&bars[warp][st], REC);
                bulk_load(ring + st * REC, recs + (int64_t)issued * REC, REC, &bars[warp][st]);
            }
            issued += AW;
        };
#pragma unroll
        for (int i = 0; i < NST; i++) issue(i);

        // after a timeout: give the copies still in flight a last, bounded chance to land
        auto drain = [&](int b, int st) {
            for (; b < min(issued, b1); b += AW, st = st + 1 == NST ? 0 : st + 1)
                for (int i = 0; i < 1000 && !mbar_try_wait(&bars[warp][st], (phase >> st) & 1u); i++) {}
        };

        QFrag<D, PT> qf;
        qf.load(a, q, h, tile);
        int lim[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int p = tile * PT + r + 8 * u;
            lim[u] = p < pairs ? kv_limit(a, q, p / G) : 0;
        }
        float m[U], l[U], o[NT][4];
        float t[U];  // o is in units of 2^(E - 15), E = kv_unit(t)
        int E[U];
#pragma unroll
        for (int u = 0; u < U; u++) m[u] = t[u] = -INFINITY, E[u] = kNoUnit, l[u] = 0.f;
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) o[i][j] = 0.f;

        float since[U];  // what the sums flushed so far have to be scaled by
        bool flushed = false;
#pragma unroll
        for (int u = 0; u < U; u++) since[u] = 1.f;
        auto flush = [&](const float (&unit)[U], const float (&back)[U]) {
#pragma unroll
            for (int i = 0; i < NT; i++) {
                float2 x[U];
                x[0] = PT == 8 ? make_float2(o[i][0] + o[i][2], o[i][1] + o[i][3]) : make_float2(o[i][0], o[i][1]);
                x[U - 1] = PT == 8 ? x[0] : make_float2(o[i][2], o[i][3]);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    float2* at = acc + u * 4 * DS + 4 * i;  // (8 rows down: 8 DS floats)
                    if (flushed) {
                        const float2 y = *at;
                        x[u].x = __fmaf_rn(y.x, since[u], x[u].x);
                        x[u].y = __fmaf_rn(y.y, since[u], x[u].y);
                    }
                    x[u].x = x[u].x * unit[u] * back[u], x[u].y = x[u].y * unit[u] * back[u];
                    *at = x[u];
                }
#pragma unroll
                for (int j = 0; j < 4; j++) o[i][j] = 0.f;
            }
#pragma unroll
            for (int u = 0; u < U; u++) since[u] = 1.f;
            flushed = true;
        };

        int st = 0, count = 0;
        float2 next = b0 + warp < b1 ? scales[b0 + warp] : make_float2(0.f, 0.f);
        for (int b = b0 + warp; b < b1; b += AW) {
            const float2 sc = next;
            if (b + AW < b1) next = scales[b + AW];
            if (!mbar_wait(&bars[warp][st], (phase >> st) & 1u, &abort_flag, a.status, kDevTimeoutFull)) {
                drain(b, st);
                break;
            }
            phase ^= 1u << st;
            const uint8_t* rec = ring + st * REC;
            float z[U][8];
            block_scores<D, PT>(qf, [&](int i) { return *reinterpret_cast<const uint4*>(rec + (i * 32 + lane) * 16); }, z);
            // online softmax; lane (r, c) holds tokens 32 b + 8 c .. + 7 of its pairs
            const int t0 = kKvBlock * b + 8 * c;
            uint32_t ph[U][4], pl[U][4];
            const float ev = kv_scale_log(sc.y);
            float corr[U];
            int step[U];  // of the unit's exponent
            bool moved = false;
#pragma unroll
            for (int u = 0; u < U; u++) {
                const float k = qf.coef[u] * sc.x;
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    z[u][i] *= k;
                    if (t0 + i >= lim[u]) z[u][i] = -INFINITY;
                    mx = fmaxf(mx, z[u][i]);
                }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m[u], mx), ms = mn == -INFINITY ? 0.f : mn;
                corr[u] = kv_ex2(m[u] - ms);
                t[u] = fmaxf(kv_unit_log(t[u], m[u], ms, mx, ev), mx > -INFINITY ? ev - kUnitSpan : -INFINITY);
                const int En = kv_unit(t[u]);
                step[u] = E[u] - En;
                const float2 inv = kv_pow2_pair(15 - En);
                const float up = sc.y * inv.x * inv.y;
                moved |= mn != m[u] || step[u] != 0;
                m[u] = mn;
                E[u] = En;
                float add = 0.f, y[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float p = kv_ex2(z[u][i] - ms);
                    add += p;
                    y[i] = t0 + i < lim[u] ? p * up : 0.f;
                }
                l[u] = l[u] * corr[u] + add;
#pragma unroll
                for (int i = 0; i < 4; i++) kv_split(y[2 * i], y[2 * i + 1], ph[u][i], pl[u][i]);
            }
            if (__any_sync(0xffffffffu, moved)) {
                const float c0 = kv_unit_step(corr[0], step[0]), c1 = PT == 8 ? c0 : kv_unit_step(corr[U - 1], step[U - 1]);
                since[0] *= c0;
                if (PT == 16) since[U - 1] *= c1;
#pragma unroll
                for (int i = 0; i < NT; i++) o[i][0] *= c0, o[i][1] *= c0, o[i][2] *= c1, o[i][3] *= c1;
            }
            uint32_t ah[2][4], al[2][4];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                if (PT == 8) {
                    ah[k][0] = ph[0][2 * k], ah[k][1] = pl[0][2 * k], ah[k][2] = ph[0][2 * k + 1], ah[k][3] = pl[0][2 * k + 1];
                } else {
                    ah[k][0] = ph[0][2 * k], ah[k][1] = ph[U - 1][2 * k], ah[k][2] = ph[0][2 * k + 1], ah[k][3] = ph[U - 1][2 * k + 1];
                    al[k][0] = pl[0][2 * k], al[k][1] = pl[U - 1][2 * k], al[k][2] = pl[0][2 * k + 1], al[k][3] = pl[U - 1][2 * k + 1];
                }
            }
#pragma unroll
            for (int np = 0; np < D / 16; np++) {
                const uint4 vw = *reinterpret_cast<const uint4*>(rec + 32 * D + (np * 32 + lane) * 16);
                const uint32_t ww[4] = {vw.x, vw.y, vw.z, vw.w};
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int f = 0; f < 2; f++) {
                        const uint32_t v0 = kv_half2_lo(ww[2 * f + k]), v1 = kv_half2_hi(ww[2 * f + k]);
                        mma16816(o[2 * np + f], ah[k], v0, v1);
                        if (PT == 16) mma16816(o[2 * np + f], al[k], v0, v1);
                    }
            }
            if (++count % kFlush == 0) {
                float one[U];
#pragma unroll
                for (int u = 0; u < U; u++) one[u] = 1.f;
                flush(one, one);
            }
            __syncwarp();
            issue(st);
            if (++st == NST) st = 0;
        }
        // Join the warps.  (Every copy of the segment has been consumed, and each stage's phase bit is kept, so the next
        // segment starts from stage 0 again.)
#pragma unroll
        for (int u = 0; u < U; u++) {
            l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
            l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
            if (c == 0) {
                mine[r + 8 * u] = m[u];
                mine[PT + r + 8 * u] = l[u];
            }
        }
        // divided by their own sums already: the values' units could not hold the sums of the largest ones
        float unit[U], back[U];
#pragma unroll
        for (int u = 0; u < U; u++) unit[u] = l[u] == 0.f ? 0.f : __fdiv_rn(1.f, l[u]), back[u] = kv_unit_value(E[u]);
        flush(unit, back);
        __syncthreads();
        // every thread the same: each warp's weight for each of its pairs, then four channels at a time
        float* part = P.part + (((int64_t)tile * P.runs + blockIdx.x) * 2 + (first ? 0 : 1)) * PT * (D + 2);
        constexpr int TPP = AW * 32 / PT;  // threads per pair
        const int pr = tid / TPP, gp = tile * PT + pr;
        float f[AW], M = -INFINITY, L = 0.f;
#pragma unroll
        for (int i = 0; i < AW; i++) M = fmaxf(M, f[i] = comb[i * CW + pr]);
        const float Ms = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int i = 0; i < AW; i++) {
            f[i] = kv_ex2(f[i] - Ms) * comb[i * CW + PT + pr];
            L += f[i];
        }
        if (gp < pairs) {
            const bool none = M == -INFINITY && L == 0.f;  // no token seen; the max is asked too, so that a NaN sum stays NaN
            const int64_t row = q.row0 + gp / G;
            const int head = h * G + gp % G;
            float* dst = whole ? a.out + row * a.ldo + (int64_t)head * D : part + 2 * PT + pr * D;
            const float scale = none ? 0.f : __fdiv_rn(1.f, L);
            if (tid % TPP == 0) {
                if (!whole) part[pr] = M, part[PT + pr] = L;
                else if (P.lse) P.lse[row * a.heads + head] = none ? INFINITY : M + log2f(L);
            }
            for (int d = 4 * (tid % TPP); d < D; d += 4 * TPP) {
                float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int i = 0; i < AW; i++) {
                    const float4 v = *reinterpret_cast<const float4*>(comb + i * CW + 2 * PT + pr * DS + d);
                    const float g = f[i] * scale;  // (at most 1: no sum outgrows the values)
                    y.x += v.x * g, y.y += v.y * g, y.z += v.z * g, y.w += v.w * g;
                }
                if (!whole || a.ovec) *reinterpret_cast<float4*>(dst + d) = y;
                else dst[d] = y.x, dst[d + 1] = y.y, dst[d + 2] = y.z, dst[d + 3] = y.w;
            }
        }
        __syncthreads();
        if (abort_flag) return;
    }
}

// Parts of a (sequence, head) that spans CTAs: a pair's max and sum over the
// parts by every warp that works on it, then the parts' outputs, four channels
// per lane.  SHARE: one CTA per (pair, head, sequence), its warps taking the
// parts in turn and added up in order -- few (sequence, head)s, many parts
// each.  Else one CTA per (head, sequence) and a warp per pair.
constexpr int CW_WARPS = 8;
template <int D, int PT, bool SHARE>
__global__ void __launch_bounds__(CW_WARPS * 32) k_kv_combine(const __grid_constant__ AttnParams P)
{
    __shared__ int sum[kKvMaxSequences + 1];
    __shared__ int warp_sums[32];
    __shared__ __align__(16) float total[SHARE ? CW_WARPS : 1][D];
    const KvAttnCall& a = P.a;
    // The kernel before lets this one start once its own wait for its predecessors is over, so what those wrote (the
    // lengths, the starts) may be read already; its own results may not.
    const KvDivision dv = kv_divide<true>(a, P.runs, sum, warp_sums);
    const int s = blockIdx.z, h = blockIdx.y, G = a.G;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const KvSeq q = kv_seq<true>(a.c, a.starts, a.rows, s);
    const int room = (sum[s + 1] - sum[s]) / a.c.H;  // units per head
    const int seg = sum[s] + h * room, run = dv.part ? 1 : dv.run;
    const int c0 = seg / run, n = room ? (seg + room - 1) / run - c0 + 1 : 0;
    griddep_wait();
    griddep_launch_dependents();
    if (n <= 1) return;  // nothing to answer, or written by the CTA that had all of it
    for (int gp = SHARE ? (int)blockIdx.x : warp; gp < q.n * G; gp += SHARE ? (int)gridDim.x : CW_WARPS) {
        const int tile = gp / PT, p = gp % PT;
        auto part = [&](int i) {
            return P.part + (((int64_t)tile * P.runs + c0 + i) * 2 + (!dv.part && i == 0 ? 1 : 0)) * PT * (D + 2);
        };
        float M = -INFINITY, L = 0.f;
        for (int i = lane; i < n; i += 32) M = fmaxf(M, part(i)[p]);
#pragma unroll
        for (int off = 16; off; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
        const float Ms = M == -INFINITY ? 0.f : M;
        for (int i = lane; i < n; i += 32) L += part(i)[PT + p] * kv_ex2(part(i)[p] - Ms);
#pragma unroll
        for (int off = 16; off; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
        const bool none = M == -INFINITY && L == 0.f;
        const float scale = none ? 0.f : __fdiv_rn(1.f, L);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        const int64_t row = q.row0 + gp / G;
        const int head = h * G + gp % G;
        float* dst = a.out + row * a.ldo + (int64_t)head * D;
        if (lane < D / 4) {
#pragma unroll 4
            for (int i = SHARE ? warp : 0; i < n; i += SHARE ? CW_WARPS : 1) {
                const float f = kv_ex2(part(i)[p] - Ms) * part(i)[PT + p] * scale;
                const float4 x = *reinterpret_cast<const float4*>(part(i) + 2 * PT + p * D + 4 * lane);
                o.x += x.x * f, o.y += x.y * f, o.z += x.z * f, o.w += x.w * f;
            }
        }
        if (SHARE) {
            if (lane < D / 4) *reinterpret_cast<float4*>(&total[warp][4 * lane]) = o;
            __syncthreads();
            for (int d = tid; d < D; d += CW_WARPS * 32) {
                float x = 0.f;
#pragma unroll
                for (int i = 0; i < CW_WARPS; i++) x += total[SHARE ? i : 0][d];
                dst[d] = x;
            }
            __syncthreads();
        } else if (lane < D / 4) {
            dst[4 * lane] = o.x, dst[4 * lane + 1] = o.y, dst[4 * lane + 2] = o.z, dst[4 * lane + 3] = o.w;
        }
        if (P.lse && lane == 0 && (!SHARE || warp == 0)) P.lse[row * a.heads + head] = none ? INFINITY : M + log2f(L);
    }
}

// weights_out = weights + the p of every pair that sees the token (at most T
// tiles of PT pairs).  A warp takes blocks of 32 tokens in turn; a lane adds up
// its rows' p for its 8 tokens, then the eight lanes that share them add up by
// butterfly.
template <int D, int PT, int T>
__global__ void __launch_bounds__(AW * 32, PT == 8 ? 3 : 2) k_kv_weights(const __grid_constant__ AttnParams P)
{
    constexpr int U = PT / 8;
    constexpr bool AHEAD = T == 1;  // (two tiles' queries leave no registers for a second block)
    const KvAttnCall& a = P.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane / 4, c = lane % 4;
    const int s = blockIdx.z, h = blockIdx.y, G = a.G;
    // (the call's own earlier kernels wait for what came before it and write neither the lengths nor the queries)
    const KvSeq q = kv_seq<true>(a.c, a.starts, a.rows, s);
    const int nb = (q.len + kKvBlock - 1) / kKvBlock, pairs = q.n > 0 && q.n <= a.max_rows ? q.n * G : 0;
    const int64_t sh = (int64_t)s * a.c.H + h;
    int b = blockIdx.x * AW + warp;
    QFrag<D, PT> qf[T];
    if (pairs && b < nb) {
#pragma unroll
        for (int tile = 0; tile < T; tile++) qf[tile].template load<true>(a, q, h, tile);
    }
    griddep_wait();
    griddep_launch_dependents();
    if (b >= nb) return;
    if (!pairs) {  // nothing received
        for (; b < nb; b += gridDim.x * AW) {
            const int t = kKvBlock * b + lane;
            const int64_t at = sh * a.c.cap + t;
            if (t < q.len) a.weights_out[at] = a.weights ? a.weights[at] : 0.f;
        }
        return;
    }
    int lim[T][U];
    float lse[T][U];
#pragma unroll
    for (int tile = 0; tile < T; tile++)
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int p = tile * PT + r + 8 * u;
            lim[tile][u] = p < pairs ? kv_limit(a, q, p / G) : 0;
            lse[tile][u] = p < pairs ? P.lse[(int64_t)(q.row0 + p / G) * a.heads + h * G + p % G] : 0.f;
        }
    // the next block's codes are fetched while this one's products run (8 x 30000 tokens, 28 heads over 4 of 128, the
    // attention included: 82 us; fetched when they are needed: 99)
    uint4 next[D / 16];
    float dnext = 0.f;
    auto fetch = [&](int block) {
        const uint4* rec = reinterpret_cast<const uint4*>(a.c.codes + (sh * a.c.nb + block) * kv_record_bytes(D)) + lane;
#pragma unroll
        for (int i = 0; i < D / 16; i++) next[i] = rec[32 * i];
        dnext = a.c.scales[sh * a.c.nb + block].x;
    };
    if (AHEAD) fetch(b);
    for (; b < nb; b += gridDim.x * AW) {
        uint4 rec[D / 16];
        if (!AHEAD) fetch(b);
#pragma unroll
        for (int i = 0; i < D / 16; i++) rec[i] = next[i];
        const float dk = dnext;
        if (AHEAD && b + (int)gridDim.x * AW < nb) fetch(b + gridDim.x * AW);
        const int t0 = kKvBlock * b + 8 * c, t = t0 + r;
        const int64_t at = sh * a.c.cap + t;
        const float before = a.weights && t < q.len ? a.weights[at] : 0.f;
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = 0.f;
#pragma unroll
        for (int tile = 0; tile < T; tile++) {
            float z[U][8];
            block_scores<D, PT>(qf[tile], [&](int i) { return rec[i]; }, z);
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int u = 0; u < U; u++)
                    w[i] += t0 + i < lim[tile][u] ? kv_ex2(__fmul_rn(z[u][i], qf[tile].coef[u] * dk) - lse[tile][u]) : 0.f;
        }
        // each step adds two rows and halves the tokens that a lane holds: lane (r, c) ends up with token 8 c + r
#pragma unroll
        for (int half = 4; half; half >>= 1)
#pragma unroll
            for (int i = 0; i < half; i++) {
                const bool up = r & half;
                const float give = up ? w[i] : w[i + half], keep = up ? w[i + half] : w[i];
                w[i] = keep + __shfl_xor_sync(0xffffffffu, give, 4 * half);
            }
        if (t < q.len) a.weights_out[at] = before + w[0];
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

constexpr int64_t kSideBySide = 2048;  // blocks

struct AttnPlan {
    bool prompt;
    int pt, tiles, runs;
    size_t part_bytes, lse_bytes;
};

AttnPlan plan_kv(const KvAttnCall& a, int num_sms)
{
    AttnPlan p{};
    const int64_t pairs = a.max_rows * a.G;
    p.pt = pairs <= 8 ? 8 : 16;
    p.tiles = (int)((pairs + p.pt - 1) / p.pt);
    // 17 to 32 pairs also run here, as two tiles side by side, over short caches: k_kv_prompt takes about 8 us more to begin
    // and end, but less per block (28 heads over 4, 4 rows).  One sequence: 13.7 us against 21.9 us over 512 blocks, 21.3
    // against 30.4 over 2048, 29.2 against 39.1 over 4096.  Eight: 23.6 against 17.7 over 1024, 36.6 against 31.4 over 4096;
    // four over 2048: 31.7 against 23.4.  (From four sequences on the join goes by one CTA per (head, sequence), which costs
    // more than the bound here allows for.)  The lengths being unknown here, the capacity stands for them.
    const int64_t blocks = (int64_t)a.c.S * a.c.H * a.c.nb;
    p.prompt = pairs > 16 && (pairs > 32 || blocks > kSideBySide);  // (two tiles is what k_kv_weights takes)
    p.runs = std::max(1, kCtasPerSm * num_sms / p.tiles);
    if (p.prompt) p.part_bytes = (kv_prompt_part_bytes(a, num_sms) + 255) / 256 * 256;
    else p.part_bytes = ((size_t)p.tiles * p.runs * 2 * p.pt * (a.c.D + 2) * sizeof(float) + 255) / 256 * 256;
    p.lse_bytes = a.weights_out ? (size_t)a.rows * a.heads * sizeof(float) : 0;
    return p;
}

template <int D, int PT>
cudaError_t launch_split(const AttnParams& P, const AttnPlan& p, cudaStream_t s)
{
    constexpr size_t smem = attn_smem_bytes<D, PT>();
    static std::atomic<uint32_t> done{0};
    cudaError_t e = allow_smem(k_kv_attn<D, PT>, (int)smem, done);
    if (e != cudaSuccess) return e;
    e = launch_pdl(k_kv_attn<D, PT>, dim3((unsigned)p.runs, (unsigned)p.tiles), dim3(AW * 32), smem, s, P);
    if (e != cudaSuccess) return e;
    const int64_t pairs = P.a.max_rows * P.a.G, n = (int64_t)P.a.c.H * P.a.c.S;
    const bool share = n * pairs <= 2 * p.runs;
    return launch_pdl(share ? k_kv_combine<D, PT, true> : k_kv_combine<D, PT, false>,
                      dim3((unsigned)(share ? pairs : 1), (unsigned)P.a.c.H, (unsigned)P.a.c.S), dim3(CW_WARPS * 32), 0, s, P);
}

}  // namespace

size_t kv_attention_scratch_bytes(const KvAttnCall& a, int num_sms)
{
    const AttnPlan p = plan_kv(a, num_sms);
    return p.part_bytes + p.lse_bytes;
}

cudaError_t launch_kv_attention(const KvAttnCall& a, void* scratch, int num_sms, cudaStream_t s, int* launches)
{
    const AttnPlan p = plan_kv(a, num_sms);
    AttnParams P{};
    P.a = a;
    P.part = static_cast<float*>(scratch);
    P.lse = p.lse_bytes ? reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + p.part_bytes) : nullptr;
    P.runs = p.runs;
    if (p.prompt) {
        return launch_kv_prompt(a, P.part, P.lse, num_sms, s, launches);
    }
    *launches = a.weights_out ? 3 : 2;
    return by_dim(a.c.D, [&](auto d) {
        constexpr int D = decltype(d)::value;
        cudaError_t e = p.pt == 8 ? launch_split<D, 8>(P, p, s) : launch_split<D, 16>(P, p, s);
        if (e != cudaSuccess || !a.weights_out) return e;
        // about four CTAs per SM, so that a warp's queries serve several blocks
        const int64_t n = (int64_t)a.c.H * a.c.S, most = ((int64_t)a.c.nb + AW - 1) / AW;
        const int64_t x = std::max<int64_t>(1, std::min(most, (4 * (int64_t)num_sms + n - 1) / n));
        return launch_pdl(p.pt == 8 ? k_kv_weights<D, 8, 1> : p.tiles == 1 ? k_kv_weights<D, 16, 1> : k_kv_weights<D, 16, 2>, dim3((unsigned)x, (unsigned)a.c.H, (unsigned)a.c.S),
                          dim3(AW * 32), 0, s, P);
    });
}

}  // namespace pxq
