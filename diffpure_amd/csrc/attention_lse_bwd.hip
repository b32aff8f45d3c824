// Backward pass of attention_lse.hip.  The probabilities are recomputed from the log-sum-exp, tile by tile:
//     P = exp(scale q k^T - lse)     delta_i = sum_d dout_id out_id     dP = dout v^T     dS = P (dP - delta)
//     dV = P^T dout                  dQ = scale dS K                    dK = scale dS^T Q        (key heads: summed over the heads that share them)
// Rows without a key have P = 0 (a log-sum-exp of +inf); a row whose log-sum-exp is NaN has NaN gradients.
// Two kernels, no atomics (results do not depend on the order of workgroups): dQ keeps queries and streams keys (and writes delta and the
// log2-domain log-sum-exp, +inf where a row has no gradient, for the other), dK / dV keeps keys and streams the queries of every head of its group.
//
// Measured on MI355X (whole calls, warm; kernels by the profiler's clock, mean and least of 100):
//   32 x 1024 tokens, 8 heads of 64, fp16    290 us; dQ 132 and 122: matrix instructions keep a SIMD busy for 39 % of it, vector instructions for 47 %; dK and dV 166 and
//                                            153: 33 % and 34 %, the rest is waiting (a barrier per tile, three waves per SIMD)
//   8191 tokens causal, 16 / 4 heads of 128, bf16    1120 us; dQ 391 and 380, dK and dV 743 and 713, joining two ranges 14: bound by the matrix instructions of 8 products
//   128 x 256 tokens, one head of 256, fp16    79 us; dQ 31, dK and dV 49, of which 30 are kept operands and results
//   1 x 256 tokens, 16 heads of 64, fp32    20 us; 11 each: two launches of four stages, latency
//
// fp16: the probabilities are formed as 2^6 P (an addend of the exponent) and taken out of the sums again at the end.  dS is rounded to fp16 as
// operand of its product, and P (dP - delta) of a long row is easily 1e-3 of dout: without the factor it meets fp16's subnormals (below 6e-5) six
// bits earlier.  Large cotangents (a scaled loss) bring 2^6 dS, or dS itself, beyond 65504.  Such an element is infinite, and so, or NaN, is every sum that it
// enters: a wave that finds one says so, and a last launch (attn_lse_again) forms those columns anew, with 2^-6, 2^-18 and 2^-30 dS (|dS| < 2^39) until they are
// finite - or lost because the input is.  It costs 4 us where nothing was lost; with every column lost 32 x 1024 x 8 heads of 64 take 770 us instead of 290, with all of
// dout NaN 1270.  In tiles of the first two launches a test for it costs more (dQ of the same: 122 us, 128 with a running maximum of |dS|, 140 with a second loop in
// the same kernel, whose registers the first then lacks).
#include "attention_lse.h"

namespace {
using namespace al;

template <int DT, int DP, int RS> struct Dq {
    using St = Stream<DP * Tr<DT>::ES, Tr<DT>::ES, RS * Tr<DT>::ROWS, 4>;
    struct Shared { char stage[2 * St::STAGE]; };
};
// A column that an infinite dS entered: ALL of its channels are infinite or NaN (the operand that it multiplies is something in each).  One channel alone is an operand's:
// a key of an infinite channel and weight 0, say, whose other channels stand.  Of the sums, and of an fp16 (or, wide, fp32) row of D elements:
template <int DT, int ND> __device__ __forceinline__ bool lost_sums(const typename Tr<DT>::Acc (&acc)[ND]) {
    bool all = true;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int r = 0; r < Tr<DT>::NR; ++r) all = all && !(fabsf(acc[dt][r]) < INFINITY);
    return col_reduce<Tr<DT>::TILE>(all ? 1.f : 0.f, [](float a, float b) { return fminf(a, b); }) > 0.f;
}
template <int DT> __device__ __forceinline__ bool lost_row(const char* x, int D, int g, int wide) {
    bool all = true;
    for (int d = g; d < D; d += Tr<DT>::G)
        all = all && (wide ? (reinterpret_cast<const unsigned*>(x)[d] & 0x7f800000) == 0x7f800000 : (reinterpret_cast<const unsigned short*>(x)[d] & 0x7c00) == 0x7c00);
    return col_reduce<Tr<DT>::TILE>(all ? 1.f : 0.f, [](float a, float b) { return fminf(a, b); }) > 0.f;
}

// dQ.  Workgroups, stages and RS as in the forward kernel.  AGAIN: the queries among the workgroup's that were lost.
template <int DT, int DP, int RS, bool AGAIN>
__device__ __forceinline__ void dq_block(const Args& p, int bid0, typename Dq<DT, DP, RS>::Shared& sh) {
    using T = Tr<DT>;
    constexpr int NW = 4, BM = RS * T::ROWS, RB = DP * T::ES, KS = DP / T::KSTEP, ND = DP / T::TILE, NKK = T::ROWS / T::KROWS, COLS = NW / RS * T::TILE;
    using St = typename Dq<DT, DP, RS>::St;
    char* smem = sh.stage;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rw = wave % RS, cl = lane & (T::TILE - 1), g = lane / T::TILE;
    const int split = bid0 % p.splits, bid = bid0 / p.splits;
    const int cols0 = p.packed ? p.Hq / p.Hkv * p.Tq : p.Tq, nblk = (cols0 + COLS - 1) / COLS;
    const int z = bid / nblk, blk = block_of(p, bid - z * nblk, nblk, true);
    if (z >= p.B * (p.packed ? p.Hkv : p.Hq)) return;
    const Kept kept(p, z);
    const int b = kept.b;
    const int n = clamp_len(p.q_lens, b, p.Tq), m = clamp_len(p.kv_lens, b, p.Tk), off = m - n;
    const int c0 = blk * COLS, col = c0 + wave / RS * T::TILE + cl;
    const int row_slots = p.D * T::ES / 16;
    const float c = p.scale * LOG2E;
    const long long half = (long long)p.B * p.Hq * p.Tqp;

    typename T::Frag qf[KS], df[KS];
    int head, tok;
    kept.col(p, col < kept.cols ? col : kept.cols - 1, head, tok);
    bool lost = false;
    if constexpr (AGAIN) {
        lost = lost_row<DT>(p.w0.p + b * p.w0.b + head * p.w0.h + tok * p.w0.t, p.D, g, p.wide);
        if (!__syncthreads_or(lost)) return;
    }
    const int krow = tok < n ? tok : (n > 0 ? n - 1 : 0);
    ld_kept<DT, KS>(qf, p.q.p + b * p.q.b + head * p.q.h + krow * p.q.t, row_slots, g);
    ld_kept<DT, KS>(df, p.dout.p + b * p.dout.b + head * p.dout.h + krow * p.dout.t, row_slots, g);
    float delta = 0.f;
    {
        typename T::Frag of[KS];
        ld_kept<DT, KS>(of, p.o.p + b * p.o.b + head * p.o.h + krow * p.o.t, row_slots, g);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int j = 0; j < 16 / T::ES; ++j) delta = fmaf((float)df[ks][j], (float)of[ks][j], delta);
    }
    delta = col_sum<T::TILE>(delta);
    const long long zh = (long long)b * p.Hq + head;
    const float lse = p.lse[zh * p.Tq + krow];
    const bool some = keys_seen(tok, n, m, p.causal) > 0;       // (not by lse: a NaN must reach the gradients)
    float l2 = some ? lse * LOG2E - (float)T::PSHIFT : INFINITY;
    if (!some) delta = 0.f;
    if (!AGAIN && g == 0 && rw == 0 && split == 0 && col < kept.cols) {
        p.rows[zh * p.Tqp + tok] = l2;
        p.rows[half + zh * p.Tqp + tok] = -delta;
    }
    if (!AGAIN && blk == nblk - 1 && split == 0) {          // the rows that round Tq up: no such query
        const int pad = p.Tqp - p.Tq, heads = p.packed ? p.Hq / p.Hkv : 1;
        for (int i = threadIdx.x; i < pad * heads; i += 256) {
            const long long at = ((long long)b * p.Hq + kept.h0 + i / pad) * p.Tqp + p.Tq + i % pad;
            p.rows[at] = INFINITY;
            p.rows[half + at] = 0.f;
        }
    }
    Score<DT> nd;                                 // dP starts from -delta
    nd.fill(-delta);
    typename T::Acc dq[ND];
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) dq[dt] = typename T::Acc{};

    const int t0 = p.packed ? 0 : c0, t1 = p.packed ? p.Tq : c0 + COLS;
    int begin = split * p.split_rows, end = t0 < n ? m : 0, open;
    if (p.causal) end = min(end, min(t1, n) + off);
    end = min(end, begin + p.split_rows);
    open = p.causal ? min(end, t0 + off + 1) : end;
    open = begin + max(open - begin, 0) / BM * BM;
    St st;
    st.init(p.k.p + b * p.k.b + kept.hk * p.k.h, p.k.t, p.v.p + b * p.v.b + kept.hk * p.v.h, p.v.t, row_slots, wave, lane);
    if (!AGAIN && begin < end) st.issue(smem, begin, m, 0, 0);
    int cur = 0, low = 0;                         // 2^(PSHIFT - low) dS is carried
    auto body = [&](int r0, auto masked) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (r0 + BM < end) st.issue(smem + (cur ^ 1) * St::STAGE, r0 + BM, m, 0, 0);
        const char *Ks = smem + cur * St::STAGE + rw * T::ROWS * RB, *Vs = Ks + St::TILE_BYTES;
        cur ^= 1;
        Score<DT> s{}, ds = nd;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            mma_rows<DT, RB>(Ks, lane, ks, qf[ks], s);
            mma_rows<DT, RB>(Vs, lane, ks, df[ks], ds);
        }
#pragma unroll
        for (int r = 0; r < s.N; ++r) s.set(r, __builtin_amdgcn_exp2f(fmaf(s.get(r), c, -l2)));
        if constexpr (masked.value) {
            const int seen = min(end, p.causal ? tok + off + 1 : end) - r0 - rw * T::ROWS - 4 * g;
#pragma unroll
            for (int r = 0; r < s.N; ++r) s.set(r, reg_row<DT>(r) < seen ? s.get(r) : 0.f);
        }
#pragma unroll
        for (int r = 0; r < s.N; ++r) ds.set(r, ds.get(r) * s.get(r));
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) {
            const typename T::Frag f = ds.pack(kk);
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) dq[dt] = T::mma(ld_tr<DT, RB>(Ks, lane, kk, dt), f, dq[dt]);
        }
        settle();
    };
    auto sweep = [&]() {
        int r0 = begin;
        for (; r0 < open; r0 += BM) body(r0, no{});
        for (; r0 < end; r0 += BM) body(r0, yes{});
    };
    if constexpr (AGAIN) {
        bool still = lost;
        do {
            if (still) {
                l2 += 12.f;
                low += 12;
            }
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) dq[dt] = typename T::Acc{};
            if (begin < end) st.issue(smem + cur * St::STAGE, begin, m, 0, 0);
            sweep();
            still = lost_sums<DT, ND>(dq);
        } while (__syncthreads_or(still && low < 36));
        lost = lost && !still;                    // (what stays lost is the input's: it stands as it is)
    } else {
        sweep();
        if constexpr (T::PSHIFT > 0) {
            const bool any = __any(!(fabsf(dq[0][0]) < INFINITY));
            if (lane == 0) p.lost_q[(((long long)z * nblk + blk) * p.splits + split) * NW + wave] = any;
        }
    }

    if constexpr (RS > 1) __syncthreads();
    const bool out = col < kept.cols;
    const long long kr = (long long)z * kept.cols + col + (long long)split * (p.packed ? p.Hkv : p.Hq) * p.B * kept.cols;
    char* row = const_cast<char*>(p.w0.p) + b * p.w0.b + head * p.w0.h + tok * p.w0.t;
    const float own = p.sample_scale ? p.sample_scale[b] * p.scale : p.scale;
    const float mul = some ? (AGAIN ? ldexpf(own, low - T::PSHIFT) : own / (float)(1 << T::PSHIFT)) : 0.f;
    if constexpr (AGAIN) {
        join_units<DT, ND, 1>(dq, mul, smem, wave, 0, lane, [&](int u, f32x4 v) {
            const int d = Units<DT, ND>::d(u, g);
            if (out && lost && d < p.D) st4<DT>(row, d, v, p.wide);
        });
    } else if (RS == 1 && p.splits == 1 && !p.wide) {
        __syncthreads();
        const int first = c0 + wave * T::TILE;
        store_cols<DT, ND, RB>(dq, mul, smem + wave * T::TILE * RB, lane, row_slots, [&](int i) -> char* {
            int h, t;
            kept.col(p, min(first + i, kept.cols - 1), h, t);
            return first + i < kept.cols ? const_cast<char*>(p.w0.p) + b * p.w0.b + h * p.w0.h + t * p.w0.t : nullptr;
        });
    } else join_units<DT, ND, RS>(dq, mul, smem, wave, rw, lane, [&](int u, f32x4 v) {
        const int d = Units<DT, ND>::d(u, g);
        if (!out || d >= p.D) return;
        if (p.splits > 1) *reinterpret_cast<f32x4*>(p.part0 + kr * p.D + d) = v;
        else st4<DT>(row, d, v, p.wide);
    });
}

template <int DT, int DP, int RS>
__global__ __launch_bounds__(256) AL_WAVES(DT == 0 && DP > 128 ? 1 : DT && DP == 64 && RS == 1 ? 3 : 2) void attn_lse_dq_kernel(Args p) {
    __shared__ __attribute__((aligned(1024))) typename Dq<DT, DP, RS>::Shared sh;
    dq_block<DT, DP, RS, false>(p, logical_block(p.xcd_map), sh);
}

// dK and dV: keys are kept, the queries of every head of the group stream by, one head after the other.  WHAT: 1 dK, 2 dV, 3 both.  AGAIN: the dK among the workgroup's
// that were lost; they take their exponents' addends lowered, the same for all, and a key's dK is that of the first pass in which it is finite.
template <int DT, int DP, int RS> struct Dkv {
    static constexpr int NW = 4, BM = RS * Tr<DT>::ROWS, RB = DP * Tr<DT>::ES, STATS = 2 * BM < 64 ? 64 : 2 * BM;
    using St = Stream<RB, Tr<DT>::ES, BM, NW>;
    struct Shared {
        char stage[2 * St::STAGE];
        float rows[2][STATS];             // stage: BM log-sum-exps, then BM -delta of the streamed queries (copied by whole waves)
    };
};
template <int DT, int DP, int RS, int WHAT, bool AGAIN>
__device__ __forceinline__ void dkv_block(const Args& p, int bid0, typename Dkv<DT, DP, RS>::Shared& sh) {
    using T = Tr<DT>;
    using K = Dkv<DT, DP, RS>;
    using St = typename K::St;
    constexpr int NW = K::NW, BM = K::BM, RB = K::RB, KS = DP / T::KSTEP, ND = DP / T::TILE, NKK = T::ROWS / T::KROWS, COLS = NW / RS * T::TILE;
    constexpr bool DK = WHAT & 1, DV = WHAT & 2;
    static_assert(128 % BM == 0 && K::STATS <= 256, "the statistics exist for a multiple of 128 rows");
    char* smem = sh.stage;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rw = wave % RS, cl = lane & (T::TILE - 1), g = lane / T::TILE;
    const int split = bid0 % p.splits, bid = bid0 / p.splits;
    const int nblk = (p.Tk + COLS - 1) / COLS, group = p.Hq / p.Hkv;
    const int z = bid / nblk, blk = block_of(p, bid - z * nblk, nblk, false);
    if (z >= p.B * p.Hkv) return;
    const int b = z / p.Hkv, hk = z - b * p.Hkv;
    const int n = clamp_len(p.q_lens, b, p.Tq), m = clamp_len(p.kv_lens, b, p.Tk), off = m - n;
    const int c0 = blk * COLS, col = c0 + wave / RS * T::TILE + cl;
    const int row_slots = p.D * T::ES / 16;
    const float c = p.scale * LOG2E;

    bool lost = false;
    if constexpr (AGAIN) {
        lost = lost_row<DT>(p.w1.p + b * p.w1.b + hk * p.w1.h + (col < p.Tk ? col : p.Tk - 1) * p.w1.t, p.D, g, p.wide);
        if (!__syncthreads_or(lost)) return;
    }
    typename T::Frag kf[KS], vf[DK ? KS : 1];
    typename T::Acc dk[DK ? ND : 1], dv[DV ? ND : 1];
    const int krow = col < m ? col : (m > 0 ? m - 1 : 0);
    ld_kept<DT, KS>(kf, p.k.p + b * p.k.b + hk * p.k.h + krow * p.k.t, row_slots, g);
    if constexpr (DK) ld_kept<DT, KS>(vf, p.v.p + b * p.v.b + hk * p.v.h + krow * p.v.t, row_slots, g);
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) {
        if constexpr (DK) dk[dt] = typename T::Acc{};
        if constexpr (DV) dv[dt] = typename T::Acc{};
    }

    // Streamed rows of each head: [begin, open) through the causal mask, [open, end) see every column.  A split launch cuts a block's own rows into equal
    // ranges: with the longest blocks first, two ranges each, the long and the short ones that meet on a CU add up alike.
    int begin = 0, end = c0 < m ? n : 0, open = 0;
    if (p.causal) begin = max(0, (c0 - off) / BM * BM);                // the first query that sees a key of this workgroup (rounded down)
    if (p.splits > 1) {
        const int range = ((max(end - begin, 0) + p.splits - 1) / p.splits + BM - 1) / BM * BM;
        begin += split * range;
        end = min(end, begin + range);
    }
    if (p.causal) open = begin + (max(min(end, c0 + COLS - 1 - off) - begin, 0) + BM - 1) / BM * BM;
    else open = begin;
    St st;
    st.init(p.q.p + b * p.q.b + hk * group * p.q.h, p.q.t, p.dout.p + b * p.dout.b + hk * group * p.dout.h, p.dout.t, row_slots, wave, lane);
    const int stat = tid & (2 * BM - 1);
    const float* mine = p.rows + ((long long)b * p.Hq + hk * group) * p.Tqp + (stat < BM ? stat : (long long)p.B * p.Hq * p.Tqp + stat - BM);
    auto issue = [&](int stage, int head, int r0) {
        st.issue(smem + stage * St::STAGE, r0, n, head * p.q.h, head * p.dout.h);
        if (wave * 64 < K::STATS) AL_GLDS(mine + (long long)head * p.Tqp + r0, reinterpret_cast<char*>(sh.rows[stage]) + wave * 256, 4);
    };
    // Rows are taken from the last one down: a causal mask lets the blocks of a head begin at different rows but end at the same one, and the blocks that run
    // at a time share what they stream (in L2) only while they stand at the same row.
    const int last = begin + (end - begin - 1) / BM * BM;
    int cur = 0, low = 0;                         // 2^(PSHIFT - low) dS is carried
    auto body = [&](int head, int r0, auto masked) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if constexpr (AGAIN) {
            if (tid < BM) sh.rows[cur][tid] += (float)low;
            __syncthreads();
        }
        const bool wrap = r0 == begin;
        if (!wrap || head + 1 < group) issue(cur ^ 1, wrap ? head + 1 : head, wrap ? last : r0 - BM);
        const char *Qs = smem + cur * St::STAGE + rw * T::ROWS * RB, *Ds = Qs + St::TILE_BYTES;
        const float* rs = sh.rows[cur] + rw * T::ROWS + 4 * g;
        cur ^= 1;
        Score<DT> l2, s{}, ds{};
#pragma unroll
        for (int r = 0; r < s.N; r += 4) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(rs + reg_row<DT>(r));
            f32x4 y = {};
            if constexpr (DK) y = *reinterpret_cast<const f32x4*>(rs + BM + reg_row<DT>(r));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                l2.set(r + j, x[j]);
                ds.set(r + j, y[j]);
            }
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            mma_rows<DT, RB>(Qs, lane, ks, kf[ks], s);
            if constexpr (DK) mma_rows<DT, RB>(Ds, lane, ks, vf[ks], ds);
        }
#pragma unroll
        for (int r = 0; r < s.N; ++r) s.set(r, __builtin_amdgcn_exp2f(fmaf(s.get(r), c, -l2.get(r))));
        if constexpr (masked.value) {
            const int first = col - off - r0 - rw * T::ROWS - 4 * g;       // first row of the tile that sees this key
#pragma unroll
            for (int r = 0; r < s.N; ++r) s.set(r, reg_row<DT>(r) >= first ? s.get(r) : 0.f);
        }
        if constexpr (DK) {
#pragma unroll
            for (int r = 0; r < s.N; ++r) ds.set(r, ds.get(r) * s.get(r));
        }
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) {
            typename T::Frag pf, sf;
            if constexpr (DV) pf = s.pack(kk);
            if constexpr (DK) sf = ds.pack(kk);
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) {
                if constexpr (DV) dv[dt] = T::mma(ld_tr<DT, RB>(Ds, lane, kk, dt), pf, dv[dt]);
                if constexpr (DK) dk[dt] = T::mma(ld_tr<DT, RB>(Qs, lane, kk, dt), sf, dk[dt]);
            }
        }
        settle();
    };
    auto sweep = [&]() {
        for (int head = 0; head < group; ++head) {
            int r0 = last;
            for (; r0 >= open; r0 -= BM) body(head, r0, no{});
            for (; r0 >= begin; r0 -= BM) body(head, r0, yes{});
        }
    };
    if constexpr (AGAIN) {
        if (begin >= end) return;
        char* row = const_cast<char*>(p.w1.p) + b * p.w1.b + hk * p.w1.h + (col < p.Tk ? col : p.Tk - 1) * p.w1.t;
        do {
            low += 12;
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) dk[dt] = typename T::Acc{};
            issue(cur, 0, last);
            sweep();
            const bool found = lost && !lost_sums<DT, ND>(dk);
            join_units<DT, ND, 1>(dk, col < m ? ldexpf(p.sample_scale ? p.sample_scale[b] * p.scale : p.scale, low - T::PSHIFT) : 0.f, smem, wave, 0, lane, [&](int u, f32x4 v) {
                const int d = Units<DT, ND>::d(u, g);
                if (found && col < p.Tk && d < p.D) st4<DT>(row, d, v, p.wide);
            });
            lost = lost && !found;
        } while (__syncthreads_or(lost && low < 36));
        return;
    }
    if (begin < end) {
        issue(0, 0, last);
        sweep();
    }
    if constexpr (T::PSHIFT > 0 && DK) {
        const bool any = __any(!(fabsf(dk[0][0]) < INFINITY));
        if (lane == 0) p.lost_k[(long long)bid0 * NW + wave] = any;
    }

    const bool out = col < p.Tk;
    const float pm = col < m ? (p.sample_scale ? p.sample_scale[b] : 1.f) / (float)(1 << T::PSHIFT) : 0.f;
    const long long kr = ((long long)split * p.B * p.Hkv + z) * p.Tk + col;
    auto put = [&](const typename T::Acc(&acc)[ND], float mul, const Ten& w, float* part) {
        __syncthreads();
        if (RS == 1 && p.splits == 1 && !p.wide) {
            const int first = c0 + wave * T::TILE;
            store_cols<DT, ND, RB>(acc, mul, smem + wave * T::TILE * RB, lane, row_slots, [&](int i) -> char* {
                return first + i < p.Tk ? const_cast<char*>(w.p) + b * w.b + hk * w.h + (first + i) * w.t : nullptr;
            });
        } else join_units<DT, ND, RS>(acc, mul, smem, wave, rw, lane, [&](int u, f32x4 v) {
            const int d = Units<DT, ND>::d(u, g);
            if (!out || d >= p.D) return;
            if (p.splits > 1) *reinterpret_cast<f32x4*>(part + kr * p.D + d) = v;
            else st4<DT>(const_cast<char*>(w.p) + b * w.b + hk * w.h + col * w.t, d, v, p.wide);
        });
    };
    if constexpr (DK) put(dk, p.scale * pm, p.w0, p.part0);
    if constexpr (DV) put(dv, pm, p.w1, p.part1);
}

template <int DT, int DP, int RS>
__global__ __launch_bounds__(256) AL_WAVES(DT == 0 && DP > 128 ? 1 : DT && DP == 64 && RS == 1 ? 3 : 2) void attn_lse_dkv_kernel(Args p) {
    __shared__ __attribute__((aligned(1024))) typename Dkv<DT, DP, RS>::Shared sh;
    const int bid = logical_block(p.xcd_map);
    if constexpr (two_roles(DP)) {
        if (bid & 1) dkv_block<DT, DP, RS, 2, false>(p, bid >> 1, sh);
        else dkv_block<DT, DP, RS, 1, false>(p, bid >> 1, sh);
    } else dkv_block<DT, DP, RS, 3, false>(p, bid, sh);
}

// fp16: what the launches before lost.  Nothing is shared with another workgroup, and nothing cut into ranges.  Two workgroups per CU take q_per blocks of queries and
// k_per of keys each, and leave if nothing was lost in the key heads that these belong to.
template <int DT, int DP>
__global__ __launch_bounds__(256) AL_WAVES(2) void attn_lse_again_kernel(Args p, int q_blocks, int q_per, int k_blocks, int k_per) {
    __shared__ __attribute__((aligned(1024))) union {
        typename Dq<DT, DP, 1>::Shared q;
        typename Dkv<DT, DP, 1>::Shared k;
    } sh;
    constexpr int COLS = 4 * Tr<DT>::TILE;
    const int q0 = min((int)blockIdx.x * q_per, q_blocks), q1 = min(q0 + q_per, q_blocks), k0 = min((int)blockIdx.x * k_per, k_blocks), k1 = min(k0 + k_per, k_blocks);
    const int qn = (p.Tq + COLS - 1) / COLS * (p.Hq / p.Hkv), kn = (p.Tk + COLS - 1) / COLS;       // blocks of a key head
    int any = 0;
    auto look = [&](const int* lost, int n, int z0, int z1) {
        for (long long i = (long long)z0 * n + threadIdx.x; i < (z1 + 1LL) * n; i += 256) any |= lost[i];
    };
    if (q0 < q1) look(p.lost_q, p.lost_qn, q0 / qn, (q1 - 1) / qn);
    if (k0 < k1) look(p.lost_k, p.lost_kn, k0 / kn, (k1 - 1) / kn);
    if (!__syncthreads_or(any)) return;
    for (int i = q0; i < q1; ++i) dq_block<DT, DP, 1, true>(p, i, sh.q);
    __syncthreads();
    for (int i = k0; i < k1; ++i) dkv_block<DT, DP, 1, 1, true>(p, i, sh.k);
}

// sums of the ranges of a split launch, in their order: part [split][rows][D] -> rows of a [B, T, H, D] tensor.  Packed as the kept queries are, or plain
// (z = b * H + h, token).
template <int DT>
__global__ __launch_bounds__(256) void attn_lse_sum_kernel(Args p, int keys) {
    const int per = p.D / 4;
    const bool packed = !keys && p.packed;
    const int heads = keys || packed ? p.Hkv : p.Hq, cols = keys ? p.Tk : (packed ? p.Hq / p.Hkv * p.Tq : p.Tq);
    const long long rows = (long long)p.B * heads * cols, id = (long long)blockIdx.x * 256 + threadIdx.x, kr = id / per;
    const int d = (int)(id - kr * per) * 4;
    if (kr >= rows) return;
    const int z = (int)(kr / cols), col = (int)(kr - (long long)z * cols), b = z / heads;
    int h = z - b * heads, t = col;
    if (packed) {
        h = h * (p.Hq / p.Hkv) + col / p.Tq;
        t = col % p.Tq;
    }
    for (int i = 0; i < (keys ? 2 : 1); ++i) {
        const float* part = (i ? p.part1 : p.part0) + kr * p.D + d;
        f32x4 v = *reinterpret_cast<const f32x4*>(part);
        for (int s = 1; s < p.splits; ++s) v += *reinterpret_cast<const f32x4*>(part + s * rows * p.D);
        const Ten& w = i ? p.w1 : p.w0;
        st4<DT>(const_cast<char*>(w.p) + b * w.b + h * w.h + t * w.t, d, v, p.wide);
    }
}

// waves of the launches that form dQ and dK
long long q_waves(const QPlan& pq) { return pq.blocks * pq.splits * 4; }
long long k_waves(const Cover& pk, int DP) { return pk.blocks * pk.splits * 4 / (two_roles(DP) ? 2 : 1); }

// what lies in the workspace before the partial results: 16-byte multiples.  (The key launch's plan goes by `causal`; the workspace holds either.)
long long stats_floats(int dtype, int B, int Tq, int Tk, int Hq, int Hkv, int DP, const QPlan& pq) {
    const long long rows = 2LL * B * Hq * ((Tq + 127LL) / 128 * 128);
    if (dtype != 1) return rows;
    const long long k0 = k_waves(k_plan(dtype, B, Tq, Tk, Hq, Hkv, DP, 0), DP), k1 = k_waves(k_plan(dtype, B, Tq, Tk, Hq, Hkv, DP, 1), DP);
    return rows + q_waves(pq) + (k0 > k1 ? k0 : k1);
}

template <int DTYPE, int DP>
void launch_bwd(const Args& a, const Ten& dq, const Ten& dk, const Ten& dv, hipStream_t s) {
    constexpr int DT = shape_of(DTYPE, DP), FEW = DP > 128 ? 2 : 4;
    const dim3 wg(256);
    Args x = a;
    x.w0 = dq;
    const QPlan pq = q_plan(DTYPE, a.B, a.Tq, a.Tk, a.Hq, a.Hkv, DP);
    x.packed = pq.packed;
    x.splits = pq.splits;
    x.split_rows = pq.split_rows;
    x.stripes = stripes_of((long long)a.B * (pq.packed ? a.Hkv : a.Hq));
    const dim3 gq((unsigned)(pq.blocks * pq.splits));
    if (pq.rs == 1) hipLaunchKernelGGL((attn_lse_dq_kernel<DT, DP, 1>), gq, wg, 0, s, x);
    else hipLaunchKernelGGL((attn_lse_dq_kernel<DT, DP, FEW>), gq, wg, 0, s, x);
    if (pq.splits > 1) {
        const long long items = (long long)a.B * a.Hq * a.Tq * (a.D / 4);
        hipLaunchKernelGGL(attn_lse_sum_kernel<DTYPE>, dim3((unsigned)((items + 255) / 256)), wg, 0, s, x, 0);
    }
    x.w0 = dk;
    x.w1 = dv;
    x.packed = 0;
    const Cover pk = k_plan(DTYPE, a.B, a.Tq, a.Tk, a.Hq, a.Hkv, DP, a.causal);
    x.stripes = stripes_of((long long)a.B * a.Hkv);
    x.splits = pk.splits;
    x.part1 = x.part0 + (long long)pk.splits * a.B * a.Hkv * a.Tk * a.D;
    const dim3 gk((unsigned)(pk.blocks * pk.splits));
    x.lost_k = a.lost_q + q_waves(pq);
    if (pk.rs == 1) hipLaunchKernelGGL((attn_lse_dkv_kernel<DT, DP, 1>), gk, wg, 0, s, x);
    else hipLaunchKernelGGL((attn_lse_dkv_kernel<DT, DP, FEW>), gk, wg, 0, s, x);
    if (pk.splits > 1) {
        const long long items = (long long)a.B * a.Hkv * a.Tk * (a.D / 4);
        hipLaunchKernelGGL(attn_lse_sum_kernel<DTYPE>, dim3((unsigned)((items + 255) / 256)), wg, 0, s, x, 1);
    }
    if constexpr (Tr<DT>::PSHIFT > 0) {
        constexpr int COLS = 4 * Tr<DT>::TILE;
        const int qb = a.B * a.Hq * ((a.Tq + COLS - 1) / COLS), kb = a.B * a.Hkv * ((a.Tk + COLS - 1) / COLS);
        x.w0 = dq;
        x.w1 = dk;
        x.splits = 1;
        x.split_rows = a.split_rows;
        x.stripes = 1;
        x.lost_qn = (int)(q_waves(pq) / ((long long)a.B * a.Hkv));
        x.lost_kn = (int)(k_waves(pk, DP) / ((long long)a.B * a.Hkv));
        const int most = qb > kb ? qb : kb, wgs = most < 512 ? most : 512;
        hipLaunchKernelGGL((attn_lse_again_kernel<DT, DP>), dim3((unsigned)wgs), wg, 0, s, x, qb, (qb + wgs - 1) / wgs, kb, (kb + wgs - 1) / wgs);
    }
}
template <int DTYPE>
void launch_bwd(const Args& a, const Ten& dq, const Ten& dk, const Ten& dv, hipStream_t s) {
    if (a.D <= 32) launch_bwd<DTYPE, 32>(a, dq, dk, dv, s);
    else if (a.D <= 64) launch_bwd<DTYPE, 64>(a, dq, dk, dv, s);
    else if (a.D <= 96) launch_bwd<DTYPE, 96>(a, dq, dk, dv, s);
    else if (a.D <= 128) launch_bwd<DTYPE, 128>(a, dq, dk, dv, s);
    else launch_bwd<DTYPE, 256>(a, dq, dk, dv, s);
}

}  // namespace

extern "C" long long dp_attention_lse_bwd_workspace(int dtype, int B, int Tq, int Tk, int Hq, int Hkv, int D) {
    if (dtype < 0 || dtype > 2 || B <= 0 || Tq <= 0 || Tk <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || D <= 0 || D > 256) return 0;
    const int DP = al::padded_dim(D);
    const al::QPlan pq = al::q_plan(dtype, B, Tq, Tk, Hq, Hkv, DP);
    const al::Cover pk = al::k_plan(dtype, B, Tq, Tk, Hq, Hkv, DP, 1), pk0 = al::k_plan(dtype, B, Tq, Tk, Hq, Hkv, DP, 0);
    const long long rows = stats_floats(dtype, B, Tq, Tk, Hq, Hkv, DP, pq);
    const long long q = pq.splits > 1 ? (long long)pq.splits * B * Hq * Tq * D : 0;
    const int ks = pk.splits > pk0.splits ? pk.splits : pk0.splits;
    const long long k = ks > 1 ? 2LL * ks * B * Hkv * Tk * D : 0;
    return (rows + (q > k ? q : k)) * 4;                // the partial sums of dQ are read before those of dK and dV are written
}

namespace {
int attn_lse_bwd(const char* fn, bool wide, const float* sample_scale, const void* dout, const void* q, const void* k, const void* v, const void* out, const float* lse, const long long* strides,
                 int dtype, int B, int Tq, int Tk, int Hq, int Hkv, int D, const int* q_lens, const int* kv_lens, float scale, int causal, void* dq, void* dk, void* dv,
                 void* work, long long work_bytes, void* stream) {
    al::Args a{};
    if (int rc = dp_attn_lse_common(fn, q, k, v, strides, dtype, B, Tq, Tk, Hq, Hkv, D, q_lens, kv_lens, scale, causal, &a)) return rc;
    const int es = dtype == 0 ? 4 : 2, ges = wide ? 4 : es;
    al::Ten tq, tk, tv;
    DP_REQUIRE(lse, "%s: lse missing", fn);
    if (!dp_attn_lse_tensor(fn, "out", out, strides + 9, es, B, Tq, Hq, false, &a.o) || !dp_attn_lse_tensor(fn, "dout", dout, strides + 12, es, B, Tq, Hq, false, &a.dout) ||
        !dp_attn_lse_tensor(fn, "dq", dq, strides + 15, ges, B, Tq, Hq, true, &tq) || !dp_attn_lse_tensor(fn, "dk", dk, strides + 18, ges, B, Tk, Hkv, true, &tk) ||
        !dp_attn_lse_tensor(fn, "dv", dv, strides + 21, ges, B, Tk, Hkv, true, &tv))
        return 1;
    const long long need = dp_attention_lse_bwd_workspace(dtype, B, Tq, Tk, Hq, Hkv, D);
    DP_REQUIRE(work && dp_aligned16(work) && work_bytes >= need, "%s: workspace of %lld bytes needed (got %lld)", fn, need, work_bytes);
    const long long row = (long long)D * es, grow = (long long)D * ges;
    const dp::Region written[] = {dp_attn_lse_region("dq", tq, B, Tq, Hq, grow), dp_attn_lse_region("dk", tk, B, Tk, Hkv, grow), dp_attn_lse_region("dv", tv, B, Tk, Hkv, grow),
                                  dp::flat("work", work, need)},
                     read[] = {dp_attn_lse_region("q", a.q, B, Tq, Hq, row), dp_attn_lse_region("k", a.k, B, Tk, Hkv, row), dp_attn_lse_region("v", a.v, B, Tk, Hkv, row),
                               dp_attn_lse_region("out", a.o, B, Tq, Hq, row), dp_attn_lse_region("dout", a.dout, B, Tq, Hq, row), dp::flat("lse", lse, 4LL * B * Hq * Tq),
                               dp::flat("q_lens", q_lens, 4LL * B), dp::flat("kv_lens", kv_lens, 4LL * B), dp::flat("sample_scale", sample_scale, 4LL * B)};
    if (dp::check_apart(fn, written, 4, read, 9)) return 1;
    a.wide = wide && dtype != 0;
    a.sample_scale = sample_scale;
    a.lse = const_cast<float*>(lse);
    a.rows = static_cast<float*>(work);
    a.lost_q = reinterpret_cast<int*>(a.rows + 2LL * B * Hq * a.Tqp);
    const int DP = al::padded_dim(D);
    a.part0 = a.rows + stats_floats(dtype, B, Tq, Tk, Hq, Hkv, DP, al::q_plan(dtype, B, Tq, Tk, Hq, Hkv, DP));
    hipStream_t s = (hipStream_t)stream;
    if (dtype == 0) launch_bwd<0>(a, tq, tk, tv, s);
    else if (dtype == 1) launch_bwd<1>(a, tq, tk, tv, s);
    else launch_bwd<2>(a, tq, tk, tv, s);
    DP_LAUNCH_CHECK("attn_lse_bwd");
    return 0;
}
}  // namespace

extern "C" int dp_attention_lse_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out, const float* lse, const long long* strides,
                                    int dtype, int B, int Tq, int Tk, int Hq, int Hkv, int D, const int* q_lens, const int* kv_lens, float scale, int causal,
                                    void* dq, void* dk, void* dv, void* work, long long work_bytes, void* stream) {
    return attn_lse_bwd("dp_attention_lse_bwd", false, nullptr, dout, q, k, v, out, lse, strides, dtype, B, Tq, Tk, Hq, Hkv, D, q_lens, kv_lens, scale, causal, dq, dk, dv, work,
                        work_bytes, stream);
}
extern "C" int dp_attention_lse_bwd_f32(const void* dout, const void* q, const void* k, const void* v, const void* out, const float* lse, const long long* strides,
                                        int dtype, int B, int Tq, int Tk, int Hq, int Hkv, int D, const int* q_lens, const int* kv_lens, float scale, int causal,
                                        float* dq, float* dk, float* dv, const float* sample_scale, void* work, long long work_bytes, void* stream) {
    return attn_lse_bwd("dp_attention_lse_bwd_f32", true, sample_scale, dout, q, k, v, out, lse, strides, dtype, B, Tq, Tk, Hq, Hkv, D, q_lens, kv_lens, scale, causal, dq, dk, dv, work,
                        work_bytes, stream);
}
