// kv_prompt.cu -- attention of many query rows over the 8-bit key/value cache
// on the 5th-generation tensor cores (formulas and accuracy: kv_attention.cu).
//
// A CTA takes 128 pairs (query row, head of the group) of one (sequence, kv
// head) over a range of the keys, in tiles i of 128 tokens = 4 cache blocks:
//     S_i = Qlo K^T + Qhi K^T          (fp32 in TMEM; Q hi and lo in TMEM, K the codes as fp16 in smem)
//     P_i = exp2(S_i coef dk - m)      (hi and lo fp16, over S_i's own columns)
//     O_i = (Plo dv) V + (Phi dv) V    (fp32 in TMEM; V the codes as fp16 in smem)
// The scales of K enter the exponent, those of V the probabilities, so the
// operands stay exact codes.  Warp roles (640 threads):
//   0-3, 4-7  softmax of the even / odd key tiles, thread = row; the running max
//             goes from one to the other through smem
//   8-11      sums of the O_i, in registers, thread = row; the output
//   12-15     codes (bulk copies, two tiles ahead) -> fp16 in 128-byte-swizzled
//             smem, two buffers each for K and V
//   16        MMA issue, in the order QK(i+1) PV(i) QK(i+2) PV(i+1): while one
//             tile's softmax runs, the tensor core has the other parity's work;
//             PV(i) starts when the first half of P_i is there
// S_{i+2} may overwrite P_i because the products of one thread are executed
// in the order in which it issues them.
//
// With W the kernel finds the weight that each token received instead: the
// rows' maxima and sums being known (lse), p = exp2(S coef dk - lse) is summed
// over the tile's 128 pairs, first over a warp's rows (lane j ends up with
// column j), then over the four warps; k_kv_weight_sum adds the tiles up in
// their order.  No atomics: the result does not depend on the order of
// execution.
//
// The tensor core cuts the accumulator's last bits at every K = 16 step, always
// towards zero, and over a long sum that adds up: with one accumulator for a
// whole prompt of 4096 tokens (256 steps on average) the output was off by
// 5.6e-6 of its norm, five times what fp32 arithmetic loses.  So O_i starts at
// zero for every tile, and the rows' sums over tiles are kept in registers,
// rounded to nearest.
//
// What bounds it: with hi and lo, four half-precision products per element.  A
// 4096-token prompt of 28 heads over 4 (D = 128, causal) takes 248 us, in which
// the tensor cores are issued 248 GFLOP (tiles on the diagonal whole): 1.00
// PFLOP/s, where a plain bf16 product sustains 1.38.  No unit is full (of 2048
// rows' cycles: tensor pipe 38 %, instruction issue 45 %, XU 21 %): a tile goes
// through a chain, scores, maximum, probabilities, PV, which two softmax warps
// per SM quarter do not hide, and a CTA takes some 8 us to begin and end.  The
// power cap (985 W) takes the clock to 1.81 GHz of 1.965.
// 148 x 128 rows take 40.6 us over 2048 keys and 137.9 over 8192: 2.03 us per
// tile of 128 keys.  By clock64, before each row had its own unit (2 % since): about
// 3400 cycles a tile for 2048 of products; softmax 2900, PV 1900 to 3100 after
// it, QK 1600 to 1900.
// The roles' loops are kept short: unrolled over a tile they did not fit the
// instruction caches together, and warps waited for instructions (123 -> 93 us
// for 148 x 128 rows over 4096 keys, together with the sums' warpgroup and the
// bulk copies of the codes).
#include <algorithm>
#include <type_traits>
#include "kv_cache.cuh"

namespace pxq {
namespace {

constexpr int kThreads = 640;
constexpr int kTileRows = 128;   // pairs per CTA
constexpr int kTileKeys = 128;
// registers per thread by role: 128 x (2 x 104 + 168 + 72 + 32) = 640 x 96, what the launch has
constexpr uint32_t kRegsSoftmax = 104, kRegsSum = 168, kRegsConvert = 72, kRegsMma = 32;

template <int D>
struct PromptSmem {
    static constexpr int K_PANEL = kTileKeys * 128;           // 128 tokens x 64 channels
    static constexpr int K_TILE = (D + 63) / 64 * K_PANEL;
    static constexpr int V_PANEL = D * 128;                   // D channels x 64 tokens
    static constexpr int V_TILE = 2 * V_PANEL;
    static constexpr int V = 2 * K_TILE;                      // after two K tiles
    static constexpr int RAW_TILE = 4 * kv_record_bytes(D);   // the codes of a key tile
    static constexpr int RAW = V + 2 * V_TILE;
    static constexpr int BYTES = RAW + 2 * RAW_TILE + 1024;   // + alignment
};
// TMEM columns; a CTA takes all 512, so they are addresses too
constexpr uint32_t kColS = 0, kColO = 256, kColQ = 384;

__device__ __forceinline__ uint64_t desc128(uint32_t saddr) { return smem_desc(saddr, 16, 1024, 2); }

// D[tmem] (+)= A[tmem] * B[smem]^T, kind::f16
__device__ __forceinline__ void mma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint32_t (&r)[4])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
                 : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Up to here a score's product and its distance from the max may be one fused
// step.  Above, the max being a rounded product, the unrounded one can exceed it by
// so much that p would leave fp16's range: those tiles take the rounded products,
// like those with masks.
constexpr float kFusedScores = 1048576.f;

struct PromptParams {
    KvAttnCall a;
    float* part;  // splits > 1: [split][tile][head]: planes m[128], l[128], (O / l)[128][D]
    float* lse;
    int tiles, splits;
    // weights (W): pair tiles [tile0, tile0 + tiles) of the batch; sums over a tile's pairs go to wpart [tile][head][wkeys]
    int tile0;
    float* wpart;
    int64_t wkeys;
};

template <bool EARLY = false>
__device__ __forceinline__ int prompt_tiles(const KvAttnCall& a, int s)
{
    const KvSeq q = kv_seq<EARLY>(a.c, a.starts, a.rows, s);
    if (q.n <= 0 || q.n > a.max_rows) return 0;
    return (q.n * a.G + kTileRows - 1) / kTileRows;  // (the host checks that rows x G fits)
}

// The part of a (sequence, head)'s keys that a split of one CTA takes:
// key tiles [t0, t1) of those that the tile's last row sees.
__device__ __forceinline__ void prompt_keys(const KvAttnCall& a, const KvSeq& q, int tile, int split, int splits, int& t0, int& t1)
{
    const int G = a.G, pairs = q.n * G;
    const int last = min(pairs, (tile + 1) * kTileRows) - 1;
    const int lim = kv_limit(a, q, last / G);
    const int n = (lim + kTileKeys - 1) / kTileKeys, per = splits == 1 ? n : (n + splits - 1) / splits;
    t0 = min(n, split * per);
    t1 = min(n, t0 + per);
}

template <int D, bool W>
__global__ void __launch_bounds__(kThreads, 1) k_kv_prompt(const __grid_constant__ PromptParams P)
{
    using M = PromptSmem<D>;
    constexpr uint32_t IDESC_S = idesc_f16_f32(128, kTileKeys), IDESC_O = idesc_f16_f32(128, D);
    constexpr int J = D / 64, REC = kv_record_bytes(D);
    extern __shared__ uint8_t dyn[];
    __shared__ int sum[kKvMaxSequences + 1];
    __shared__ int warp_sums[32];
    __shared__ uint64_t bar_k_full[2], bar_k_empty[2], bar_v_full[2], bar_v_empty[2], bar_raw[2], bar_raw_empty[2], bar_s[2], bar_m[2], bar_w[2], bar_p[2][2], bar_o_full[2],
        bar_o_empty, bar_rows, bar_q, bar_fin;
    __shared__ float row_max[2][kTileRows], row_sum[2][kTileRows], row_gain[4][kTileRows];  // by tile's parity; gain by tile % 4
    __shared__ float row_log[2][kTileRows];  // the rows' units (kv_unit), by tile's parity
    __shared__ float col_sum[W ? 2 : 1][2][4][kTileKeys];  // by tile's parity, alternating
    __shared__ uint32_t tmem_slot, abort_flag;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn) + 1023) & ~(uintptr_t)1023);

    const KvAttnCall& a = P.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int h = blockIdx.x % a.c.H, gt = (W ? P.tile0 : 0) + P.tiles - 1 - blockIdx.x / a.c.H, split = blockIdx.y, G = a.G;
    if (tid == 0) {
        abort_flag = 0;
        for (int i = 0; i < 2; i++) {
            mbar_init(&bar_k_full[i], 128);
            mbar_init(&bar_k_empty[i], 1);
            mbar_init(&bar_v_full[i], 128);
            mbar_init(&bar_v_empty[i], 1);
            mbar_init(&bar_raw[i], 4);
            mbar_init(&bar_raw_empty[i], 128);
            mbar_init(&bar_w[i], 128);
            mbar_init(&bar_s[i], 1);
            mbar_init(&bar_m[i], 128);
            mbar_init(&bar_p[i][0], 128);
            mbar_init(&bar_p[i][1], 128);
            mbar_init(&bar_o_full[i], 1);
        }
        mbar_init(&bar_o_empty, 128);
        mbar_init(&bar_rows, 128);
        mbar_init(&bar_q, 256);
        mbar_init(&bar_fin, 1);
        fence_mbar_init();
    }
    if (warp == 16) {
        tmem_alloc(&tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    griddep_wait();
    griddep_launch_dependents();
    kv_prefix(a.c.S, sum, warp_sums, [&](int s) {
        const KvSeq q = kv_seq(a.c, a.starts, a.rows, s);
        if (!W && blockIdx.x == 0 && blockIdx.y == 0 && (q.n < 0 || q.n > a.max_rows)) atomicAdd(a.status + kStatusKv + kStatusKvStarts, 1u);
        return prompt_tiles(a, s);
    });
    tc_fence_after();
    if (tmem_slot != 0 && tid == 0) {  // (the whole of TMEM begins at 0)
        abort_flag = 1;
        atomicCAS(a.status, 0u, (uint32_t)kDevBadTmem);
    }
    uint32_t* status = a.status;
    int n = 0, t0 = 0, tile = 0;
    KvSeq q{};
    int64_t sh = 0;
    if (gt < sum[a.c.S]) {
        const int s = kv_find(sum, a.c.S, gt);
        tile = gt - sum[s];
        q = kv_seq(a.c, a.starts, a.rows, s);
        int t1;
        prompt_keys(a, q, tile, split, P.splits, t0, t1);
        n = t1 - t0;  // key tiles
        sh = (int64_t)s * a.c.H + h;
    }
    const int pairs = q.n * G, tile0 = tile * kTileRows;
    float* part = P.part + (((int64_t)split * P.tiles + gt) * a.c.H + h) * kTileRows * (D + 2);  // (splits > 1)
    const uint8_t* recs = a.c.codes + sh * a.c.nb * (int64_t)REC;
    const float2* scales = a.c.scales + sh * a.c.nb;
    // codes of key tile i: converter warp cw copies one of its blocks; past the cache's end: its last block (masked)
    auto copy_codes = [&](int i, int cw) {
        mbar_expect_tx(&bar_raw[i & 1], REC);
        bulk_load(smem + M::RAW + (i & 1) * M::RAW_TILE + cw * REC,
                  recs + (int64_t)min((t0 + i) * (kTileKeys / kKvBlock) + cw, a.c.nb - 1) * REC, REC, &bar_raw[i & 1]);
    };
    if (warp >= 12 && warp < 16 && lane == 0)
        for (int i = 0; i < min(n, 2); i++) copy_codes(i, warp - 12);
    const int X = warp / 4, row = tid & 127, p = tile0 + row;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    // rows of q at first, and of the result at last, stand where the second K tile and V are in between
    float* const mine = reinterpret_cast<float*>(smem + M::K_TILE) + row * (D + 4);
    static_assert(kTileRows * (D + 4) * 4 <= M::RAW - M::K_TILE, "rows fit");

    if (warp < 8) {
        regs_inc<kRegsSoftmax>();
        // the row's query: one bulk copy (or, unaligned, plain loads), then scaled to below 2^15, split, stored in TMEM;
        // the two warpgroups take half of the channels each
        const bool bulk = a.qvec != 0;
        float4 x[D / 8];
        {
            const float* src = a.q + (int64_t)(q.row0 + p / G) * a.ldq + (int64_t)(h * G + p % G) * D;
            if (bulk) {
                if (X == 0) {
                    if (p < pairs) {
                        mbar_expect_tx(&bar_rows, D * 4);
                        bulk_load(mine, src, D * 4, &bar_rows);
                    } else {
                        mbar_arrive(&bar_rows);
                    }
                }
                mbar_wait(&bar_rows, 0, &abort_flag, status, kDevTimeoutFull);
            }
            src += X * (D / 2);
#pragma unroll
            for (int i = 0; i < D / 8; i++) {
                if (p >= pairs) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                else if (bulk) x[i] = *reinterpret_cast<const float4*>(mine + X * (D / 2) + 4 * i);
                else x[i] = make_float4(src[4 * i], src[4 * i + 1], src[4 * i + 2], src[4 * i + 3]);
            }
        }
        float coef;
        {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < D / 8; i++) top = max3(max3(top, fabsf(x[i].x), fabsf(x[i].y)), fabsf(x[i].z), fabsf(x[i].w));
            row_sum[X][row] = top;
            named_bar_sync(3, 256);
            top = fmaxf(top, row_sum[X ^ 1][row]);
            const int e = top > 0.f && top <= FLT_MAX ? max(-113, min(110, 15 - kv_exponent(top))) : 0;
            const float up = kv_pow2(e);
            coef = kv_log2_inv_sqrt(D) * kv_pow2(-e);
#pragma unroll
            for (int i = 0; i < D / 8; i += 2) {
                uint32_t hi[4], lo[4];
                kv_split(x[i].x * up, x[i].y * up, hi[0], lo[0]);
                kv_split(x[i].z * up, x[i].w * up, hi[1], lo[1]);
                kv_split(x[i + 1].x * up, x[i + 1].y * up, hi[2], lo[2]);
                kv_split(x[i + 1].z * up, x[i + 1].w * up, hi[3], lo[3]);
                tmem_st4(lanes + kColQ + X * (D / 4) + 2 * i, hi);
                tmem_st4(lanes + kColQ + D / 2 + X * (D / 4) + 2 * i, lo);
            }
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&bar_q);
        const int lim = p < pairs ? kv_limit(a, q, p / G) : 0;
        const uint32_t ts = lanes + kColS + X * 128;
        // lane j < 4: the scales of key tile i's block j; blocks past the end hold anything
        auto fetch = [&](int i) {
            const int b = (t0 + i) * (kTileKeys / kKvBlock) + lane;
            return lane < 4 && i < n && b * kKvBlock < q.len ? scales[b] : make_float2(0.f, 0.f);
        };
        float2 next = fetch(X);
        if constexpr (W) {
            float* const dst = P.wpart + ((int64_t)(gt - P.tile0) * a.c.H + h) * P.wkeys;
            const float lse = p < pairs ? P.lse[(int64_t)(q.row0 + p / G) * a.heads + h * G + p % G] : INFINITY;
            for (int i = X; i < n; i += 2) {
                const int key0 = (t0 + i) * kTileKeys;
                const float2 sc = next;
                next = fetch(i + 2);
                if (!mbar_wait(&bar_s[X], (i >> 1) & 1, &abort_flag, status, kDevTimeoutTmemFull)) break;
                tc_fence_after();
                const bool full = __all_sync(0xffffffffu, key0 + kTileKeys <= lim);
                float* const cols = col_sum[X][(i >> 1) & 1][warp & 3];
                auto add_up = [&](auto careful) {
#pragma unroll 1
                    for (int j = 0; j < 4; j++) {
                        uint32_t r[32];
                        float w[32];
                        tmem_ld32(ts + 32 * j, r);
                        const float k = coef * __shfl_sync(0xffffffffu, sc.x, j);
                        tmem_ld_wait_dep(r);
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            float p0 = -lse, p1 = -lse;
                            if (decltype(careful)::value) {
                                p0 += __fmul_rn(__uint_as_float(r[c]), k);
                                p1 += __fmul_rn(__uint_as_float(r[c + 1]), k);
                            } else {
                                ffma2(p0, p1, __uint_as_float(r[c]), __uint_as_float(r[c + 1]), k, k);
                            }
                            w[c] = kv_ex2(p0);
                            w[c + 1] = kv_ex2(p1);
                            if (decltype(careful)::value) {
                                const int t = key0 + 32 * j + c;
                                if (t >= lim) w[c] = 0.f;
                                if (t + 1 >= lim) w[c + 1] = 0.f;
                            }
                        }
                        // each step adds two rows and halves the columns that a lane holds
#pragma unroll
                        for (int half = 16; half; half >>= 1)
#pragma unroll
                            for (int c = 0; c < half; c++) {
                                const bool up = lane & half;
                                const float give = up ? w[c] : w[c + half];
                                const float keep = up ? w[c + half] : w[c];
                                w[c] = keep + __shfl_xor_sync(0xffffffffu, give, half);
                            }
                        cols[32 * j + lane] = w[0];
                    }
                };
                if (full && __all_sync(0xffffffffu, fabsf(lse) < kFusedScores)) add_up(std::false_type{});
                else add_up(std::true_type{});
                tc_fence_before();
                mbar_arrive(&bar_p[X][0]);
                mbar_arrive(&bar_w[X]);
                if (!mbar_wait(&bar_w[X], (i >> 1) & 1, &abort_flag, status, kDevTimeoutScaleFull)) break;
                const float(&c4)[4][kTileKeys] = col_sum[X][(i >> 1) & 1];
                dst[key0 + row] = (c4[0][row] + c4[1][row]) + (c4[2][row] + c4[3][row]);
            }
        } else {
        float m = -INFINITY, l = 0.f;  // over this parity's tiles, m with the other's before it
        float t = -INFINITY;           // P_i holds p dv / 2^(kv_unit(t) - 15)
        for (int i = X; i < n; i += 2) {
            const int key0 = (t0 + i) * kTileKeys;
            const float2 sc = next;
            next = fetch(i + 2);
            const float evs = kv_scale_log(sc.y);
            if (!mbar_wait(&bar_s[X], (i >> 1) & 1, &abort_flag, status, kDevTimeoutTmemFull)) break;
            tc_fence_after();
            const bool full = __all_sync(0xffffffffu, key0 + kTileKeys <= lim);
            float mt = -INFINITY, tt = -INFINITY, et = -INFINITY;  // the tile's max, its t relative to that, its largest ev
            // TMEM loads run one chunk of 16 tokens ahead of their use
            auto maxima = [&](auto masked) {
                uint32_t r[2][16];
                tmem_ld16(ts, r[0]);
#pragma unroll 1
                for (int j = 0; j < 4; j++) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        tmem_ld_wait_dep(r[u]);
                        tmem_ld16(ts + (32 * j + 16 * u + 16) % kTileKeys, r[u ^ 1]);
#pragma unroll
                        for (int c = 0; c < 16; c += 2) {
                            float x0 = __uint_as_float(r[u][c]), x1 = __uint_as_float(r[u][c + 1]);
                            if (decltype(masked)::value) {
                                const int key = key0 + 32 * j + 16 * u + c;
                                if (key >= lim) x0 = -INFINITY;
                                if (key + 1 >= lim) x1 = -INFINITY;
                            }
                            mx = max3(mx, x0, x1);
                        }
                    }
                    const float k = coef * __shfl_sync(0xffffffffu, sc.x, j);
                    const float ev = __shfl_sync(0xffffffffu, evs, j);
                    if (!decltype(masked)::value || mx != -INFINITY) {
                        const float z = mx * k, mb = fmaxf(mt, z);
                        tt = kv_unit_log(tt, mt, mb, z, ev);
                        et = fmaxf(et, ev);
                        mt = mb;
                    }
                }
                tmem_ld_wait_dep(r[0]);
            };
            if (full) maxima(std::false_type{});
            else maxima(std::true_type{});
            // the max and the unit of the tiles before, from the other parity
            float mp = -INFINITY, tp = -INFINITY;
            if (i > 0) {
                if (!mbar_wait(&bar_m[X ^ 1], ((i - 1) >> 1) & 1, &abort_flag, status, kDevTimeoutScaleFull)) break;
                mp = row_max[X ^ 1][row];
                tp = row_log[X ^ 1][row];
            }
            const float mn = fmaxf(mp, mt), ms = mn == -INFINITY ? 0.f : mn;
            t = fmaxf(fmaxf(tp - (ms - mp), tt - (ms - mt)), et - kUnitSpan);
            row_max[X][row] = mn;
            row_log[X][row] = t;
            mbar_arrive(&bar_m[X]);
            const int E = kv_unit(t);
            row_gain[i & 3][row] = kv_unit_step(kv_ex2(mp - ms), kv_unit(tp) - E);
            const float2 inv = kv_pow2_pair(15 - E);
            l *= kv_ex2(m - ms);
            m = mn;
            float add0 = 0.f, add1 = 0.f;
            auto weigh = [&](auto careful) {
                uint32_t r[2][16];
                tmem_ld16(ts, r[0]);
#pragma unroll 1
                for (int j = 0; j < 4; j++) {
                    const float k = coef * __shfl_sync(0xffffffffu, sc.x, j), y = __shfl_sync(0xffffffffu, sc.y, j) * inv.x * inv.y;
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        uint32_t hi[8], lo[8];
                        tmem_ld_wait_dep(r[u]);
                        tmem_ld16(ts + (32 * j + 16 * u + 16) % kTileKeys, r[u ^ 1]);
#pragma unroll
                        for (int c = 0; c < 8; c++) {
                            float p0 = -ms, p1 = -ms, y0, y1;
                            if (decltype(careful)::value) {
                                p0 += __fmul_rn(__uint_as_float(r[u][2 * c]), k);
                                p1 += __fmul_rn(__uint_as_float(r[u][2 * c + 1]), k);
                            } else {
                                ffma2(p0, p1, __uint_as_float(r[u][2 * c]), __uint_as_float(r[u][2 * c + 1]), k, k);
                            }
                            p0 = kv_ex2(p0);
                            p1 = kv_ex2(p1);
                            fmul2(y0, y1, p0, p1, y, y);
                            if (decltype(careful)::value) {
                                const int key = key0 + 32 * j + 16 * u + 2 * c;
                                if (key >= lim) p0 = y0 = 0.f;
                                if (key + 1 >= lim) p1 = y1 = 0.f;
                            }
                            ffma2(add0, add1, p0, p1, 1.f, 1.f);
                            kv_split(y0, y1, hi[c], lo[c]);
                        }
                        tmem_st8(ts + 32 * j + 16 * u, hi);
                        tmem_st8(ts + 32 * j + 16 * u + 8, lo);
                    }
                    if (j & 1) {
                        tmem_st_wait();
                        tc_fence_before();
                        mbar_arrive(&bar_p[X][j >> 1]);
                    }
                }
                tmem_ld_wait_dep(r[0]);
            };
            if (full && __all_sync(0xffffffffu, fabsf(ms) < kFusedScores)) weigh(std::false_type{});
            else weigh(std::true_type{});
            l += add0 + add1;
        }
        row_max[X][row] = m;  // (read by nobody but the sums' warps any more)
        row_sum[X][row] = l;
        row_log[X][row] = t;
        named_bar_sync(1, 384);
        }
    } else if (warp < 12) {
        regs_inc<kRegsSum>();
        if constexpr (!W) {
        const uint32_t to = lanes + kColO;
        float o[D];
        bool ok = true;
#pragma unroll
        for (int d = 0; d < D; d++) o[d] = 0.f;
        for (int i = 0; i < n; i++) {
            if (!mbar_wait(&bar_o_full[i & 1], (i >> 1) & 1, &abort_flag, status, kDevTimeoutTmemFull)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const float g = row_gain[i & 3][row];
            uint32_t r[2][16];
            tmem_ld16(to, r[0]);
#pragma unroll
            for (int d = 0; d < D; d += 16) {
                tmem_ld_wait_dep(r[d / 16 & 1]);
                if (d + 16 < D) tmem_ld16(to + d + 16, r[(d / 16 + 1) & 1]);
#pragma unroll
                for (int c = 0; c < 16; c += 2) {
                    float x = __uint_as_float(r[d / 16 & 1][c]), y = __uint_as_float(r[d / 16 & 1][c + 1]);
                    ffma2(x, y, o[d + c], o[d + c + 1], g, g);
                    o[d + c] = x;
                    o[d + c + 1] = y;
                }
            }
            tc_fence_before();
            mbar_arrive(&bar_o_empty);
        }
        named_bar_sync(1, 384);
        if (ok) {
            const float m0 = row_max[0][row], m1 = row_max[1][row], mn = fmaxf(m0, m1), ms = mn == -INFINITY ? 0.f : mn;
            const float l = row_sum[0][row] * kv_ex2(m0 - ms) + row_sum[1][row] * kv_ex2(m1 - ms);
            const bool none = mn == -INFINITY && l == 0.f;  // on the max too: a NaN sum stays NaN
            if (P.splits > 1 && p < pairs) {
                part[row] = mn;
                part[kTileRows + row] = l;
            } else if (P.lse && p < pairs) {
                P.lse[(int64_t)(q.row0 + p / G) * a.heads + h * G + p % G] = none ? INFINITY : mn + log2f(l);
            }
            const float scale = none || l == 0.f ? 0.f : __fdiv_rn(1.f, l);
            const float back = kv_unit_value(kv_unit(row_log[(n - 1) & 1][row]));
            // every product is done: the row goes through smem, out by one bulk copy (or, unaligned, plain stores)
            float* dst = P.splits > 1 ? part + 2 * kTileRows + (int64_t)row * D : a.out + (int64_t)(q.row0 + p / G) * a.ldo + (int64_t)(h * G + p % G) * D;
            if (P.splits > 1 || a.ovec) {
#pragma unroll
                for (int d = 0; d < D; d += 4)
                    *reinterpret_cast<float4*>(mine + d) = make_float4(o[d] * scale * back, o[d + 1] * scale * back, o[d + 2] * scale * back,
                                                                       o[d + 3] * scale * back);
                fence_proxy_async_smem();
                if (p < pairs) bulk_store(dst, mine, D * 4);
                bulk_commit();
                bulk_wait_read_all();
            } else if (p < pairs) {
#pragma unroll
                for (int d = 0; d < D; d++) dst[d] = o[d] * scale * back;
            }
        }
        }
    } else if (warp < 16) {
        regs_dec<kRegsConvert>();
        const int cw = warp - 12, qn = lane / 4, qc = lane % 4;
        // K: the warp's own block.  V: lanes of even and odd qn take the two blocks of the warp's half tile, so that eight
        // lanes' 16-byte stores fall in different banks.
        const int bv = cw / 2 * 2 + ((qn ^ cw) & 1);
        const uint32_t sb = smem_u32(smem);
        auto ld128 = [](uint32_t at) {
            uint4 v;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
            return v;
        };
        auto st128 = [](uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
        };
        int issued = min(n, 2), i = 0;
        for (; i < n; i++) {
            const int B = i & 1;
            const uint32_t ph = ((i >> 1) - 1) & 1, raw = sb + M::RAW + B * M::RAW_TILE + lane * 16;
            if (!mbar_wait(&bar_raw[B], (i >> 1) & 1, &abort_flag, status, kDevTimeoutFull)) break;
            if (i > 1 && !mbar_wait(&bar_k_empty[B], ph, &abort_flag, status, kDevTimeoutEmpty)) break;
            {
                const uint32_t rk = raw + cw * REC, t = 8 * (qn / 2) + qn % 2;  // token of its block: t + 2 nt
                const uint32_t kb = sb + B * M::K_TILE + (32 * cw + t) * 128;
                // four loads at a time: one load's latency covers 80 instructions
#pragma unroll
                for (uint32_t n0 = 0; n0 < 4; n0 += 4 / J) {
                    uint4 w[4];
#pragma unroll
                    for (int u = 0; u < 4; u++) w[u] = ld128(rk + (n0 * J + u) * 512);
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const uint32_t nt = n0 + u / J, x = (t + 2 * nt) & 7, at = kb + u % J * M::K_PANEL + nt * 256;
                        st128(at + ((2 * qc ^ x) << 4), kv_half2_lo(w[u].x), kv_half2_hi(w[u].x), kv_half2_lo(w[u].y), kv_half2_hi(w[u].y));
                        st128(at + (((2 * qc + 1) ^ x) << 4), kv_half2_lo(w[u].z), kv_half2_hi(w[u].z), kv_half2_lo(w[u].w), kv_half2_hi(w[u].w));
                    }
                }
                if (D % 64) {
                    const uint4 r = ld128(rk + 4 * J * 512);
                    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                    for (uint32_t nt = 0; nt < 4; nt++) {
                        const uint32_t x = (t + 2 * nt) & 7;
                        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(kb + J * M::K_PANEL + nt * 256 + ((qc / 2 ^ x) << 4) + qc % 2 * 8),
                                     "r"(kv_half2_lo(w[nt])), "r"(kv_half2_hi(w[nt]))
                                     : "memory");
                    }
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(&bar_k_full[B]);
            if (i == 0 && !mbar_wait(&bar_q, 0, &abort_flag, status, kDevTimeoutEmpty)) break;  // the queries have left V's place and K's second
            if (!W && i > 1 && !mbar_wait(&bar_v_empty[B], ph, &abort_flag, status, kDevTimeoutEmpty)) break;
            if constexpr (!W) {
                const uint32_t rv = raw + bv * REC + 32 * D;
                const uint32_t vb = sb + M::V + B * M::V_TILE + cw / 2 * M::V_PANEL + qn * 128 + (((4 * (bv & 1) + qc) ^ qn) << 4);
                constexpr int VG = D / 16 % 4 == 0 ? 4 : 5;
                static_assert(D / 16 % VG == 0, "whole groups");
#pragma unroll
                for (uint32_t n0 = 0; n0 < D / 16; n0 += VG) {  // channels 16 np + qn, + 8
                    uint4 w[VG];
#pragma unroll
                    for (int u = 0; u < VG; u++) w[u] = ld128(rv + (n0 + u) * 512);
#pragma unroll
                    for (int u = 0; u < VG; u++) {
                        st128(vb + (n0 + u) * 2048, kv_half2_lo(w[u].x), kv_half2_hi(w[u].x), kv_half2_lo(w[u].y), kv_half2_hi(w[u].y));
                        st128(vb + (n0 + u) * 2048 + 1024, kv_half2_lo(w[u].z), kv_half2_hi(w[u].z), kv_half2_lo(w[u].w), kv_half2_hi(w[u].w));
                    }
                }
            }
            if (!W) {
                fence_proxy_async_smem();
                mbar_arrive(&bar_v_full[B]);
            }
            mbar_arrive(&bar_raw_empty[B]);
            if (i + 2 < n) {
                if (lane == 0) {  // all four warps have read the tile's codes
                    if (!mbar_wait(&bar_raw_empty[B], (i >> 1) & 1, &abort_flag, status, kDevTimeoutEmpty)) break;
                    copy_codes(i + 2, cw);
                }
                issued = i + 3;
            }
        }
        // after a timeout: give the copies still in flight a last, bounded chance to land
        for (; i < issued; i++)
            for (int k = 0; k < 1000 && !mbar_try_wait(&bar_raw[i & 1], (i >> 1) & 1); k++) {}
    } else {
        regs_dec<kRegsMma>();
        if (warp == 16 && n > 0) {
            // The warp stays together and one lane issues: operands are then known to be the same for all lanes and
            // live in uniform registers.
            const bool one = elect_one();
            const uint64_t dk = desc128(smem_u32(smem)), dv = desc128(smem_u32(smem + M::V));  // + byte offset / 16
            auto qk = [&](int i, auto parity) {
                constexpr int B = decltype(parity)::value;
                if (!mbar_wait(&bar_k_full[B], (i >> 1) & 1, &abort_flag, status, kDevTimeoutFull)) return false;
                tc_fence_after();
                if (one) {
#pragma unroll
                    for (int lo = 1; lo >= 0; lo--)
#pragma unroll
                        for (int k = 0; k < D / 16; k++)
                            mma_f16_ta(kColS + B * 128, kColQ + lo * (D / 2) + k * 8,
                                       dk + (B * M::K_TILE + k / 4 * M::K_PANEL + k % 4 * 32) / 16, IDESC_S, !lo || k);
                    mma_commit(&bar_s[B]);
                    mma_commit(&bar_k_empty[B]);
                }
                __syncwarp();
                return true;
            };
            auto pv = [&](int i, auto parity) {
                constexpr int B = decltype(parity)::value;
                if constexpr (W)  // the softmax warps are done with S_i
                    return mbar_wait(&bar_p[B][0], (i >> 1) & 1, &abort_flag, status, kDevTimeoutTmemEmpty);
                if (!mbar_wait(&bar_v_full[B], (i >> 1) & 1, &abort_flag, status, kDevTimeoutFull)) return false;
                if (i > 0 && !mbar_wait(&bar_o_empty, (i - 1) & 1, &abort_flag, status, kDevTimeoutTmemEmpty)) return false;
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    if (!mbar_wait(&bar_p[B][half], (i >> 1) & 1, &abort_flag, status, kDevTimeoutTmemEmpty)) return false;
                    tc_fence_after();
                    if (one) {
#pragma unroll
                        for (int lo = 1; lo >= 0; lo--)
#pragma unroll
                            for (int k = 0; k < kTileKeys / 32; k++)
                                mma_f16_ta(kColO, kColS + B * 128 + half * 64 + k * 16 + lo * 8,
                                           dv + (B * M::V_TILE + half * M::V_PANEL) / 16 + k * 2, IDESC_O, half || !lo || k);
                        if (half) {
                            mma_commit(&bar_o_full[B]);
                            mma_commit(&bar_v_empty[B]);
                        }
                    }
                    __syncwarp();
                }
                return true;
            };
            using Even = std::integral_constant<int, 0>;
            using Odd = std::integral_constant<int, 1>;
            bool ok = mbar_wait(&bar_q, 0, &abort_flag, status, kDevTimeoutFull) && qk(0, Even{});
#pragma unroll 1
            for (int i = 0; ok && i < n; i += 2)
                ok = (i + 1 >= n || qk(i + 1, Odd{})) && pv(i, Even{}) && (i + 2 >= n || qk(i + 2, Even{})) && (i + 1 >= n || pv(i + 1, Odd{}));
            // nothing of this CTA may still run when its TMEM is freed
            if (one) mma_commit(&bar_fin);
            for (int i = 0; i < 2000 && !mbar_try_wait(&bar_fin, 0); i++) {}
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 16) tmem_dealloc(tmem_slot, 512);
}

// Joins the key splits: one warp per pair of a (tile, head).
template <int D>
__global__ void __launch_bounds__(256) k_kv_join(const __grid_constant__ PromptParams P)
{
    __shared__ int sum[kKvMaxSequences + 1];
    __shared__ int warp_sums[32];
    const KvAttnCall& a = P.a;
    // (what came before the kernel that wrote the parts is over: that one waited for it before it let this one start)
    kv_prefix(a.c.S, sum, warp_sums, [&](int s) { return prompt_tiles<true>(a, s); });
    const int gt = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31, G = a.G;
    int used = 0, p = 0, pr = 0;
    KvSeq q{};
    if (gt < sum[a.c.S]) {
        const int s = kv_find(sum, a.c.S, gt), tile = gt - sum[s];
        q = kv_seq<true>(a.c, a.starts, a.rows, s);
        pr = blockIdx.z * 8 + (threadIdx.x >> 5);
        p = tile * kTileRows + pr;
        if (p < q.n * G) {
            int t0, t1;
            prompt_keys(a, q, tile, 0, P.splits, t0, t1);
            const int per = max(1, t1 - t0);
            prompt_keys(a, q, tile, 0, 1, t0, t1);
            used = max(1, (t1 + per - 1) / per);  // splits that had keys (none: the first says so)
        }
    }
    griddep_wait();
    griddep_launch_dependents();
    if (!used) return;
    const int64_t step = (int64_t)P.tiles * a.c.H * kTileRows * (D + 2);
    const float* part = P.part + ((int64_t)gt * a.c.H + h) * kTileRows * (D + 2);
    float m = -INFINITY, l = 0.f;
    for (int i = lane; i < used; i += 32) m = fmaxf(m, part[i * step + pr]);
#pragma unroll
    for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    const float ms = m == -INFINITY ? 0.f : m;
    for (int i = lane; i < used; i += 32) l += part[i * step + kTileRows + pr] * kv_ex2(part[i * step + pr] - ms);
#pragma unroll
    for (int off = 16; off; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    const bool none = m == -INFINITY && l == 0.f;
    const float f = none ? 0.f : __fdiv_rn(1.f, l);
    const int64_t row = q.row0 + p / G;
    const int head = h * G + p % G;
    if (lane < D / 4) {
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int i = 0; i < used; i++) {
            const float w = kv_ex2(part[i * step + pr] - ms) * part[i * step + kTileRows + pr] * f;  // (at most 1)
            const float4 x = *reinterpret_cast<const float4*>(part + i * step + 2 * kTileRows + (int64_t)pr * D + 4 * lane);
            o.x += x.x * w, o.y += x.y * w, o.z += x.z * w, o.w += x.w * w;
        }
        float* dst = a.out + row * a.ldo + (int64_t)head * D + 4 * lane;
        dst[0] = o.x, dst[1] = o.y, dst[2] = o.z, dst[3] = o.w;
    }
    if (P.lse && lane == 0) P.lse[row * a.heads + head] = none ? INFINITY : m + log2f(l);
}

// weights_out = base + the sums of the batch's tiles, in their order
__global__ void __launch_bounds__(128) k_kv_weight_sum(const __grid_constant__ PromptParams P, const float* base)
{
    __shared__ int sum[kKvMaxSequences + 1];
    __shared__ int warp_sums[32];
    const KvAttnCall& a = P.a;
    griddep_wait();
    griddep_launch_dependents();
    kv_prefix(a.c.S, sum, warp_sums, [&](int s) { return prompt_tiles(a, s); });
    const int s = blockIdx.z, h = blockIdx.y;
    const int64_t key = (int64_t)blockIdx.x * 128 + threadIdx.x;
    const KvSeq q = kv_seq(a.c, a.starts, a.rows, s);
    if (key >= q.len) return;
    const int g0 = max(sum[s], P.tile0), g1 = min(sum[s + 1], P.tile0 + P.tiles);
    float w = 0.f;
#pragma unroll 4
    for (int g = g0; g < g1; g++) {
        const int last = min(q.n * a.G, (g - sum[s] + 1) * kTileRows) - 1;
        if (key < kv_limit(a, q, last / a.G)) w += P.wpart[((int64_t)(g - P.tile0) * a.c.H + h) * P.wkeys + key];
    }
    const int64_t at = ((int64_t)s * a.c.H + h) * a.c.cap + key;
    a.weights_out[at] = (base ? base[at] : 0.f) + w;
}

struct PromptPlan {
    int tiles, splits;
    int64_t wkeys, wtiles;  // weights: keys per partial row, pair tiles per pass
    size_t part_bytes;      // (the weights' sums take the place of the split parts)
};

PromptPlan plan_prompt(const KvAttnCall& a, int num_sms)
{
    PromptPlan p{};
    const int64_t G = a.G;
    // a sequence's n rows make at most n G / 128 + 1 tiles
    const int64_t most = std::min<int64_t>(a.c.S * ((a.max_rows * G + kTileRows - 1) / kTileRows), a.rows * G / kTileRows + a.c.S);
    p.tiles = (int)most;
    const int64_t key_tiles = (a.c.cap + kTileKeys - 1) / kTileKeys;
    p.splits = (int)std::max<int64_t>(1, std::min(key_tiles, num_sms / (most * a.c.H)));
    p.part_bytes = p.splits > 1 ? (size_t)p.splits * p.tiles * a.c.H * kTileRows * (a.c.D + 2) * sizeof(float) : 0;
    if (a.weights_out) {
        // as many tiles at a time as 256 MB of partial sums hold
        p.wkeys = key_tiles * kTileKeys;
        const int64_t per = p.wkeys * a.c.H * (int64_t)sizeof(float);
        p.wtiles = std::max<int64_t>(1, std::min<int64_t>(p.tiles, ((int64_t)256 << 20) / per));
        p.part_bytes = std::max(p.part_bytes, (size_t)(p.wtiles * per));
    }
    return p;
}

template <int D>
cudaError_t launch_weights(PromptParams P, const PromptPlan& p, int num_sms, cudaStream_t s, int* launches)
{
    constexpr int smem = PromptSmem<D>::BYTES;
    static std::atomic<uint32_t> done{0};
    cudaError_t e = allow_smem(k_kv_prompt<D, true>, smem, done);
    P.wpart = P.part;
    P.wkeys = p.wkeys;
    for (int64_t t = 0; t < p.tiles && e == cudaSuccess; t += p.wtiles) {
        P.tile0 = (int)t;
        P.tiles = (int)std::min(p.wtiles, p.tiles - t);
        P.splits = (int)std::max<int64_t>(1, std::min<int64_t>(p.wkeys / kTileKeys, num_sms / ((int64_t)P.tiles * P.a.c.H)));
        e = launch_pdl(k_kv_prompt<D, true>, dim3((unsigned)(P.tiles * P.a.c.H), (unsigned)P.splits), dim3(kThreads), smem, s, P);
        if (e != cudaSuccess) break;
        e = launch_pdl(k_kv_weight_sum, dim3((unsigned)((P.a.c.cap + 127) / 128), (unsigned)P.a.c.H, (unsigned)P.a.c.S), dim3(128), 0, s, P,
                       t ? (const float*)P.a.weights_out : P.a.weights);
        *launches += 2;
    }
    return e;
}

template <int D>
cudaError_t launch_d(const PromptParams& P, cudaStream_t s)
{
    constexpr int smem = PromptSmem<D>::BYTES;
    static std::atomic<uint32_t> done{0};
    cudaError_t e = allow_smem(k_kv_prompt<D, false>, smem, done);
    if (e != cudaSuccess) return e;
    e = launch_pdl(k_kv_prompt<D, false>, dim3((unsigned)(P.tiles * P.a.c.H), (unsigned)P.splits), dim3(kThreads), smem, s, P);
    if (e != cudaSuccess || P.splits == 1) return e;
    const int64_t pairs = std::min<int64_t>(kTileRows, P.a.max_rows * P.a.G);
    return launch_pdl(k_kv_join<D>, dim3((unsigned)P.tiles, (unsigned)P.a.c.H, (unsigned)((pairs + 7) / 8)), dim3(256), 0, s, P);
}

}  // namespace

size_t kv_prompt_part_bytes(const KvAttnCall& a, int num_sms) { return plan_prompt(a, num_sms).part_bytes; }

cudaError_t launch_kv_prompt(const KvAttnCall& a, float* part, float* lse, int num_sms, cudaStream_t s, int* launches)
{
    const PromptPlan p = plan_prompt(a, num_sms);
    PromptParams P{};
    P.a = a;
    P.part = part;
    P.lse = lse;
    P.tiles = p.tiles;
    P.splits = p.splits;
    *launches = p.splits > 1 ? 2 : 1;
    auto run = [&](auto d) {
        constexpr int D = decltype(d)::value;
        const cudaError_t e = launch_d<D>(P, s);
        return e != cudaSuccess || !a.weights_out ? e : launch_weights<D>(P, p, num_sms, s, launches);
    };
    switch (a.c.D) {
    case 64: return run(std::integral_constant<int, 64>{});
    case 80: return run(std::integral_constant<int, 80>{});
    case 128: return run(std::integral_constant<int, 128>{});
    default: return cudaErrorInvalidValue;
    }
}

}  // namespace pxq
