// Backward pass of attention_lse.hip.  The probabilities are recomputed from the log-sum-exp, tile by tile:
//     P = exp(scale q k^T - lse)     delta_i = sum_d dout_id out_id     dP = dout v^T     dS = P (dP - delta)
//     dV = P^T dout                  dQ = scale dS K                    dK = scale dS^T Q        (key heads: summed over the heads that share them)
// Two kernels, no atomics (results do not depend on the order of workgroups): dQ keeps queries and streams keys (and writes delta and the
// log2-domain log-sum-exp, +inf where a row has no gradient, for the other), dK / dV keeps keys and streams the queries of every head of its group.
//
// fp16: the probabilities are formed as 2^6 P (an addend of the exponent) and taken out of the sums again at the end.  dS is rounded to fp16 as
// operand of its product, and P (dP - delta) of a long row is easily 1e-3 of dout: without the factor it meets fp16's subnormals (below 6e-5) six
// bits earlier.  |dS| <= P (1 - P) max|dP_i - dP_j|, so 2^6 dS overflows only where the spread of dout v^T along a row passes 4094.
#include "attention_lse.h"

namespace {
using namespace al;

// dQ.  Workgroups, stages and RS as in the forward kernel.
template <int DT, int DP, int CW, int RS, int RT>
__global__ __launch_bounds__(256) AL_WAVES(DT && DP == 64 && RS == 1 ? 3 : DP <= 128 ? 2 : 1) void attn_lse_dq_kernel(Args p) {
    using T = Tr<DT>;
    constexpr int NW = 4, BM = RS * RT * T::TILE, RB = DP * T::ES, KS = DP / 16, ND = DP / T::TILE, NKK = T::TILE / 16, COLS = NW / RS * CW * T::TILE;
    using St = Stream<RB, T::ES, BM, NW>;
    __shared__ __attribute__((aligned(1024))) char smem[2 * St::STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rw = wave % RS, cl = lane & (T::TILE - 1), g = lane / T::TILE;
    const int bid0 = logical_block(p.xcd_map), split = bid0 % p.splits, bid = bid0 / p.splits;
    const int cols0 = p.packed ? p.Hq / p.Hkv * p.Tq : p.Tq, nblk = (cols0 + COLS - 1) / COLS;
    const int z = bid / nblk, blk = block_of(p, bid - z * nblk, nblk, true);
    if (z >= p.B * (p.packed ? p.Hkv : p.Hq)) return;
    const Kept kept(p, z);
    const int b = kept.b;
    const int n = clamp_len(p.q_lens, b, p.Tq), m = clamp_len(p.kv_lens, b, p.Tk), off = m - n;
    const int c0 = blk * COLS, wc0 = c0 + wave / RS * CW * T::TILE;
    const int row_slots = p.D * T::ES / 16;
    const float c = p.scale * LOG2E;
    const long long half = (long long)p.B * p.Hq * p.Tqp;

    typename T::Frag qf[CW][KS], df[CW][KS];
    typename T::Acc dq[CW][ND], nd[CW];
    float l2[CW];
    int head[CW], tok[CW];
#pragma unroll
    for (int cw = 0; cw < CW; ++cw) {
        const int col = wc0 + cw * T::TILE + cl;
        kept.col(p, col < kept.cols ? col : kept.cols - 1, head[cw], tok[cw]);
        const int row = tok[cw] < n ? tok[cw] : (n > 0 ? n - 1 : 0);
        ld_kept<DT, KS>(qf[cw], p.q.p + b * p.q.b + head[cw] * p.q.h + row * p.q.t, row_slots, g);
        ld_kept<DT, KS>(df[cw], p.dout.p + b * p.dout.b + head[cw] * p.dout.h + row * p.dout.t, row_slots, g);
        float delta = 0.f;
        {
            typename T::Frag of[KS];
            ld_kept<DT, KS>(of, p.o.p + b * p.o.b + head[cw] * p.o.h + row * p.o.t, row_slots, g);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int j = 0; j < 16 / T::ES; ++j) delta = fmaf((float)df[cw][ks][j], (float)of[ks][j], delta);
        }
        delta = col_sum<T::TILE>(delta);
        const long long at = (long long)b * p.Hq + head[cw];
        const float lse = p.lse[at * p.Tq + row];
        const bool some = tok[cw] < n && lse > -INFINITY;
        l2[cw] = some ? lse * LOG2E - (float)T::PSHIFT : INFINITY;
        if (!some) delta = 0.f;
        if (g == 0 && rw == 0 && split == 0 && col < kept.cols) {
            p.rows[at * p.Tqp + tok[cw]] = l2[cw];
            p.rows[half + at * p.Tqp + tok[cw]] = -delta;
        }
#pragma unroll
        for (int r = 0; r < T::NR; ++r) nd[cw][r] = -delta;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) dq[cw][dt] = typename T::Acc{};
    }
    if (blk == nblk - 1 && split == 0) {          // the rows that round Tq up: no such query
        const int pad = p.Tqp - p.Tq, heads = p.packed ? p.Hq / p.Hkv : 1;
        for (int i = threadIdx.x; i < pad * heads; i += 256) {
            const long long at = ((long long)b * p.Hq + kept.h0 + i / pad) * p.Tqp + p.Tq + i % pad;
            p.rows[at] = INFINITY;
            p.rows[half + at] = 0.f;
        }
    }

    const int t0 = p.packed ? 0 : c0, t1 = p.packed ? p.Tq : c0 + COLS;
    int begin = split * p.split_rows, end = t0 < n ? m : 0, open;
    if (p.causal) end = min(end, min(t1, n) + off);
    end = min(end, begin + p.split_rows);
    open = p.causal ? min(end, t0 + off + 1) : end;
    open = begin + max(open - begin, 0) / BM * BM;
    St st;
    st.init(p.k.p + b * p.k.b + kept.hk * p.k.h, p.k.t, p.v.p + b * p.v.b + kept.hk * p.v.h, p.v.t, row_slots, wave, lane);
    if (begin < end) st.issue(smem, begin, m, 0, 0);
    int cur = 0;
    auto body = [&](int r0, auto masked) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (r0 + BM < end) st.issue(smem + (cur ^ 1) * St::STAGE, r0 + BM, m, 0, 0);
        const char* stage = smem + cur * St::STAGE;
        cur ^= 1;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int rr = (rw * RT + rt) * T::TILE;
            const char *Ks = stage + rr * RB, *Vs = Ks + St::TILE_BYTES;
            typename T::Acc s[CW], ds[CW];
#pragma unroll
            for (int cw = 0; cw < CW; ++cw) {
                s[cw] = typename T::Acc{};
                ds[cw] = nd[cw];
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const typename T::Frag ak = ld_row<DT, RB>(Ks, lane, ks), av = ld_row<DT, RB>(Vs, lane, ks);
#pragma unroll
                for (int cw = 0; cw < CW; ++cw) {
                    s[cw] = T::mma(ak, qf[cw][ks], s[cw]);
                    ds[cw] = T::mma(av, df[cw][ks], ds[cw]);
                }
            }
#pragma unroll
            for (int cw = 0; cw < CW; ++cw)
#pragma unroll
                for (int r = 0; r < T::NR; ++r) s[cw][r] = __builtin_amdgcn_exp2f(fmaf(s[cw][r], c, -l2[cw]));
            if constexpr (masked.value) {
#pragma unroll
                for (int cw = 0; cw < CW; ++cw) {
                    const int seen = min(end, p.causal ? tok[cw] + off + 1 : end) - r0 - rr - 4 * g;
#pragma unroll
                    for (int r = 0; r < T::NR; ++r) s[cw][r] = reg_row<DT>(r) < seen ? s[cw][r] : 0.f;
                }
            }
#pragma unroll
            for (int cw = 0; cw < CW; ++cw)
#pragma unroll
                for (int r = 0; r < T::NR; ++r) ds[cw][r] *= s[cw][r];
#pragma unroll
            for (int kk = 0; kk < NKK; ++kk) {
                typename T::Frag f[CW];
#pragma unroll
                for (int cw = 0; cw < CW; ++cw) f[cw] = pack<DT>(ds[cw], kk);
#pragma unroll
                for (int dt = 0; dt < ND; ++dt) {
                    const typename T::Frag a = ld_tr<DT, RB>(Ks, lane, kk, dt);
#pragma unroll
                    for (int cw = 0; cw < CW; ++cw) dq[cw][dt] = T::mma(a, f[cw], dq[cw][dt]);
                }
            }
        }
        settle();
    };
    int r0 = begin;
    for (; r0 < open; r0 += BM) body(r0, no{});
    for (; r0 < end; r0 += BM) body(r0, yes{});

    const float mul = p.scale / (float)(1 << T::PSHIFT);
#pragma unroll
    for (int cw = 0; cw < CW; ++cw) {
        if constexpr (RS > 1) __syncthreads();
        const int col = wc0 + cw * T::TILE + cl;
        const bool out = col < kept.cols, some = tok[cw] < n;
        const long long kr = (long long)z * kept.cols + col + (long long)split * (p.packed ? p.Hkv : p.Hq) * p.B * kept.cols;
        char* row = const_cast<char*>(p.w0.p) + b * p.w0.b + head[cw] * p.w0.h + tok[cw] * p.w0.t;
        join_units<DT, ND, RS>(dq[cw], mul, smem, wave, rw, lane, [&](int u, f32x4 v) {
            const int d = Units<DT, ND>::d(u, g);
            if (!out || d >= p.D) return;
            if (!some) v = f32x4{};
            if (p.splits > 1) *reinterpret_cast<f32x4*>(p.part0 + kr * p.D + d) = v;
            else st4<DT>(row, d, v);
        });
    }
}

// dK and dV: keys are kept, the queries of every head of the group stream by, one head after the other.  WHAT: 1 dK, 2 dV, 3 both.
template <int DT, int DP, int CW, int RS, int RT> struct Dkv {
    static constexpr int NW = 4, BM = RS * RT * Tr<DT>::TILE, RB = DP * Tr<DT>::ES;
    using St = Stream<RB, Tr<DT>::ES, BM, NW>;
    struct Shared {
        char stage[2 * St::STAGE];
        float rows[2][2][BM];             // stage: log-sum-exp, -delta of the streamed queries
    };
};
template <int DT, int DP, int CW, int RS, int RT, int WHAT>
__device__ __forceinline__ void dkv_block(const Args& p, int bid0, typename Dkv<DT, DP, CW, RS, RT>::Shared& sh) {
    using T = Tr<DT>;
    using K = Dkv<DT, DP, CW, RS, RT>;
    using St = typename K::St;
    constexpr int NW = K::NW, BM = K::BM, RB = K::RB, KS = DP / 16, ND = DP / T::TILE, NKK = T::TILE / 16, COLS = NW / RS * CW * T::TILE;
    constexpr bool DK = WHAT & 1, DV = WHAT & 2;
    static_assert(BM % 32 == 0 && BM <= 128, "whole waves copy the rows' statistics, of which a multiple of 128 exist");
    char* smem = sh.stage;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rw = wave % RS, cl = lane & (T::TILE - 1), g = lane / T::TILE;
    const int split = bid0 % p.splits, bid = bid0 / p.splits;
    const int nblk = (p.Tk + COLS - 1) / COLS, group = p.Hq / p.Hkv;
    const int z = bid / nblk, blk = block_of(p, bid - z * nblk, nblk, false);
    if (z >= p.B * p.Hkv) return;
    const int b = z / p.Hkv, hk = z - b * p.Hkv;
    const int n = clamp_len(p.q_lens, b, p.Tq), m = clamp_len(p.kv_lens, b, p.Tk), off = m - n;
    const int c0 = blk * COLS, wc0 = c0 + wave / RS * CW * T::TILE;
    const int row_slots = p.D * T::ES / 16;
    const float c = p.scale * LOG2E;

    typename T::Frag kf[CW][KS], vf[CW][DK ? KS : 1];
    typename T::Acc dk[CW][DK ? ND : 1], dv[CW][DV ? ND : 1];
#pragma unroll
    for (int cw = 0; cw < CW; ++cw) {
        const int col = wc0 + cw * T::TILE + cl, row = col < m ? col : (m > 0 ? m - 1 : 0);
        ld_kept<DT, KS>(kf[cw], p.k.p + b * p.k.b + hk * p.k.h + row * p.k.t, row_slots, g);
        if constexpr (DK) ld_kept<DT, KS>(vf[cw], p.v.p + b * p.v.b + hk * p.v.h + row * p.v.t, row_slots, g);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
            if constexpr (DK) dk[cw][dt] = typename T::Acc{};
            if constexpr (DV) dv[cw][dt] = typename T::Acc{};
        }
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
    // lane t < 2 BM of the workgroup copies one value of a tile: log-sum-exp (t < BM) or -delta of query t % BM
    const float* mine = p.rows + ((long long)b * p.Hq + hk * group) * p.Tqp + (tid < BM ? tid : (long long)p.B * p.Hq * p.Tqp + tid - BM);
    auto issue = [&](int stage, int head, int r0) {
        st.issue(smem + stage * St::STAGE, r0, n, head * p.q.h, head * p.dout.h);
        if (wave * 64 < 2 * BM) AL_GLDS(mine + (long long)head * p.Tqp + r0, reinterpret_cast<char*>(&sh.rows[stage][0][0]) + wave * 256, 4);
    };
    // Rows are taken from the last one down: a causal mask lets the blocks of a head begin at different rows but end at the same one, and the blocks that run
    // at a time share what they stream (in L2) only while they stand at the same row.
    const int last = begin + (end - begin - 1) / BM * BM;
    int cur = 0;
    auto body = [&](int head, int r0, auto masked) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        const bool wrap = r0 == begin;
        if (!wrap || head + 1 < group) issue(cur ^ 1, wrap ? head + 1 : head, wrap ? last : r0 - BM);
        const char* stage = smem + cur * St::STAGE;
        const float(*rs)[BM] = sh.rows[cur];
        cur ^= 1;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int rr = (rw * RT + rt) * T::TILE;
            const char *Qs = stage + rr * RB, *Ds = Qs + St::TILE_BYTES;
            typename T::Acc l2, nd;
#pragma unroll
            for (int r = 0; r < T::NR; r += 4) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(&rs[0][rr + r * T::G + 4 * g]);
                f32x4 y = {};
                if constexpr (DK) y = *reinterpret_cast<const f32x4*>(&rs[1][rr + r * T::G + 4 * g]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    l2[r + j] = x[j];
                    nd[r + j] = y[j];
                }
            }
            typename T::Acc s[CW], ds[CW];
#pragma unroll
            for (int cw = 0; cw < CW; ++cw) {
                s[cw] = typename T::Acc{};
                ds[cw] = nd;
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const typename T::Frag aq = ld_row<DT, RB>(Qs, lane, ks);
#pragma unroll
                for (int cw = 0; cw < CW; ++cw) s[cw] = T::mma(aq, kf[cw][ks], s[cw]);
                if constexpr (DK) {
                    const typename T::Frag ad = ld_row<DT, RB>(Ds, lane, ks);
#pragma unroll
                    for (int cw = 0; cw < CW; ++cw) ds[cw] = T::mma(ad, vf[cw][ks], ds[cw]);
                }
            }
#pragma unroll
            for (int cw = 0; cw < CW; ++cw)
#pragma unroll
                for (int r = 0; r < T::NR; ++r) s[cw][r] = __builtin_amdgcn_exp2f(fmaf(s[cw][r], c, -l2[r]));
            if constexpr (masked.value) {
#pragma unroll
                for (int cw = 0; cw < CW; ++cw) {
                    const int first = wc0 + cw * T::TILE + cl - off - r0 - rr - 4 * g;       // first row of the tile that sees this key
#pragma unroll
                    for (int r = 0; r < T::NR; ++r) s[cw][r] = reg_row<DT>(r) >= first ? s[cw][r] : 0.f;
                }
            }
#pragma unroll
            for (int cw = 0; cw < CW; ++cw)
#pragma unroll
                for (int r = 0; r < T::NR; ++r) ds[cw][r] *= s[cw][r];
#pragma unroll
            for (int kk = 0; kk < NKK; ++kk) {
                typename T::Frag pf[CW], sf[CW];
#pragma unroll
                for (int cw = 0; cw < CW; ++cw) {
                    if constexpr (DV) pf[cw] = pack<DT>(s[cw], kk);
                    if constexpr (DK) sf[cw] = pack<DT>(ds[cw], kk);
                }
#pragma unroll
                for (int dt = 0; dt < ND; ++dt) {
                    if constexpr (DV) {
                        const typename T::Frag ad = ld_tr<DT, RB>(Ds, lane, kk, dt);
#pragma unroll
                        for (int cw = 0; cw < CW; ++cw) dv[cw][dt] = T::mma(ad, pf[cw], dv[cw][dt]);
                    }
                    if constexpr (DK) {
                        const typename T::Frag aq = ld_tr<DT, RB>(Qs, lane, kk, dt);
#pragma unroll
                        for (int cw = 0; cw < CW; ++cw) dk[cw][dt] = T::mma(aq, sf[cw], dk[cw][dt]);
                    }
                }
            }
        }
        settle();
    };
    if (begin < end) {
        issue(0, 0, last);
        for (int head = 0; head < group; ++head) {
            int r0 = last;
            for (; r0 >= open; r0 -= BM) body(head, r0, no{});
            for (; r0 >= begin; r0 -= BM) body(head, r0, yes{});
        }
    }

    const float pm = 1.f / (float)(1 << T::PSHIFT);
#pragma unroll
    for (int cw = 0; cw < CW; ++cw) {
        const int col = wc0 + cw * T::TILE + cl;
        const bool out = col < p.Tk, some = col < m;
        const long long kr = ((long long)split * p.B * p.Hkv + z) * p.Tk + col;
        auto put = [&](const Ten& w, float* part, int u, f32x4 v) {
            const int d = Units<DT, ND>::d(u, g);
            if (!out || d >= p.D) return;
            if (!some) v = f32x4{};
            if (p.splits > 1) *reinterpret_cast<f32x4*>(part + kr * p.D + d) = v;
            else st4<DT>(const_cast<char*>(w.p) + b * w.b + hk * w.h + col * w.t, d, v);
        };
        if constexpr (DK) {
            if constexpr (RS > 1) __syncthreads();
            join_units<DT, ND, RS>(dk[cw], p.scale * pm, smem, wave, rw, lane, [&](int u, f32x4 v) { put(p.w0, p.part0, u, v); });
        }
        if constexpr (DV) {
            if constexpr (RS > 1) __syncthreads();
            join_units<DT, ND, RS>(dv[cw], pm, smem, wave, rw, lane, [&](int u, f32x4 v) { put(p.w1, p.part1, u, v); });
        }
    }
}

template <int DT, int DP, int CW, int RS, int RT>
__global__ __launch_bounds__(256) AL_WAVES(DP > 128 ? 1 : DT && DP == 64 && RS == 1 ? 3 : 2) void attn_lse_dkv_kernel(Args p) {
    __shared__ __attribute__((aligned(1024))) typename Dkv<DT, DP, CW, RS, RT>::Shared sh;
    const int bid = logical_block(p.xcd_map);
    if constexpr (two_roles(DP)) {
        if (bid & 1) dkv_block<DT, DP, CW, RS, RT, 2>(p, bid >> 1, sh);
        else dkv_block<DT, DP, CW, RS, RT, 1>(p, bid >> 1, sh);
    } else dkv_block<DT, DP, CW, RS, RT, 3>(p, bid, sh);
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
        st4<DT>(const_cast<char*>(w.p) + b * w.b + h * w.h + t * w.t, d, v);
    }
}

template <int DT, int DP>
void launch_bwd(const Args& a, const Ten& dq, const Ten& dk, const Ten& dv, hipStream_t s) {
    constexpr int TILE = Tr<DT>::TILE, WIDE = DP > 128 ? 2 : 4, RT = DT == 0 ? 2 : 1;
    const dim3 wg(256);
    Args x = a;
    x.w0 = dq;
    const QPlan pq = q_plan(a.B, a.Tq, a.Tk, a.Hq, a.Hkv, DP, TILE);
    x.packed = pq.packed;
    x.splits = pq.splits;
    x.split_rows = pq.split_rows;
    x.stripes = stripes_of((long long)a.B * (pq.packed ? a.Hkv : a.Hq));
    const dim3 gq((unsigned)(pq.blocks * pq.splits));
    if (pq.rs == 1) hipLaunchKernelGGL((attn_lse_dq_kernel<DT, DP, 1, 1, 1>), gq, wg, 0, s, x);
    else hipLaunchKernelGGL((attn_lse_dq_kernel<DT, DP, 1, WIDE, 1>), gq, wg, 0, s, x);
    if (pq.splits > 1) {
        const long long items = (long long)a.B * a.Hq * a.Tq * (a.D / 4);
        hipLaunchKernelGGL(attn_lse_sum_kernel<DT>, dim3((unsigned)((items + 255) / 256)), wg, 0, s, x, 0);
    }
    x.w0 = dk;
    x.w1 = dv;
    x.packed = 0;
    const KPlan pk = k_plan(a.B, a.Tq, a.Tk, a.Hkv, DP, TILE, DT == 0, a.causal);
    x.stripes = stripes_of((long long)a.B * a.Hkv);
    x.splits = pk.splits;
    x.part1 = x.part0 + (long long)pk.splits * a.B * a.Hkv * a.Tk * a.D;
    const dim3 gk((unsigned)(pk.blocks * pk.splits * (two_roles(DP) ? 2 : 1)));
    if (pk.rs == 1) hipLaunchKernelGGL((attn_lse_dkv_kernel<DT, DP, 1, 1, RT>), gk, wg, 0, s, x);
    else hipLaunchKernelGGL((attn_lse_dkv_kernel<DT, DP, 1, WIDE, 1>), gk, wg, 0, s, x);
    if (pk.splits > 1) {
        const long long items = (long long)a.B * a.Hkv * a.Tk * (a.D / 4);
        hipLaunchKernelGGL(attn_lse_sum_kernel<DT>, dim3((unsigned)((items + 255) / 256)), wg, 0, s, x, 1);
    }
}
template <int DT>
void launch_bwd(const Args& a, const Ten& dq, const Ten& dk, const Ten& dv, hipStream_t s) {
    if (a.D <= 32) launch_bwd<DT, 32>(a, dq, dk, dv, s);
    else if (a.D <= 64) launch_bwd<DT, 64>(a, dq, dk, dv, s);
    else if (a.D <= 96) launch_bwd<DT, 96>(a, dq, dk, dv, s);
    else if (a.D <= 128) launch_bwd<DT, 128>(a, dq, dk, dv, s);
    else launch_bwd<DT, 256>(a, dq, dk, dv, s);
}

}  // namespace

extern "C" long long dp_attention_lse_bwd_workspace(int dtype, int B, int Tq, int Tk, int Hq, int Hkv, int D) {
    if (dtype < 0 || dtype > 2 || B <= 0 || Tq <= 0 || Tk <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || D <= 0 || D > 256) return 0;
    const int tile = dtype == 0 ? 16 : 32, DP = al::padded_dim(D);
    const al::QPlan pq = al::q_plan(B, Tq, Tk, Hq, Hkv, DP, tile);
    const al::KPlan pk = al::k_plan(B, Tq, Tk, Hkv, DP, tile, dtype == 0, 1), pk0 = al::k_plan(B, Tq, Tk, Hkv, DP, tile, dtype == 0, 0);
    const long long rows = 2LL * B * Hq * ((Tq + 127LL) / 128 * 128);
    const long long q = pq.splits > 1 ? (long long)pq.splits * B * Hq * Tq * D : 0;
    const int ks = pk.splits > pk0.splits ? pk.splits : pk0.splits;
    const long long k = ks > 1 ? 2LL * ks * B * Hkv * Tk * D : 0;
    return (rows + (q > k ? q : k)) * 4;                // the partial sums of dQ are read before those of dK and dV are written
}

extern "C" int dp_attention_lse_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out, const float* lse, const long long* strides,
                                    int dtype, int B, int Tq, int Tk, int Hq, int Hkv, int D, const int* q_lens, const int* kv_lens, float scale, int causal,
                                    void* dq, void* dk, void* dv, void* work, long long work_bytes, void* stream) {
    const char* fn = "dp_attention_lse_bwd";
    al::Args a{};
    if (int rc = dp_attn_lse_common(fn, q, k, v, strides, dtype, B, Tq, Tk, Hq, Hkv, D, q_lens, kv_lens, scale, causal, &a)) return rc;
    const int es = dtype == 0 ? 4 : 2;
    al::Ten tq, tk, tv;
    DP_REQUIRE(lse, "%s: lse missing", fn);
    if (!dp_attn_lse_tensor(fn, "out", out, strides + 9, es, B, Tq, Hq, false, &a.o) || !dp_attn_lse_tensor(fn, "dout", dout, strides + 12, es, B, Tq, Hq, false, &a.dout) ||
        !dp_attn_lse_tensor(fn, "dq", dq, strides + 15, es, B, Tq, Hq, true, &tq) || !dp_attn_lse_tensor(fn, "dk", dk, strides + 18, es, B, Tk, Hkv, true, &tk) ||
        !dp_attn_lse_tensor(fn, "dv", dv, strides + 21, es, B, Tk, Hkv, true, &tv))
        return 1;
    const long long need = dp_attention_lse_bwd_workspace(dtype, B, Tq, Tk, Hq, Hkv, D);
    DP_REQUIRE(work && dp_aligned16(work) && work_bytes >= need, "%s: workspace of %lld bytes needed (got %lld)", fn, need, work_bytes);
    a.lse = const_cast<float*>(lse);
    a.rows = static_cast<float*>(work);
    a.part0 = a.rows + 2LL * B * Hq * a.Tqp;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == 0) launch_bwd<0>(a, tq, tk, tv, s);
    else if (dtype == 1) launch_bwd<1>(a, tq, tk, tv, s);
    else launch_bwd<2>(a, tq, tk, tv, s);
    DP_LAUNCH_CHECK("attn_lse_bwd");
    return 0;
}
