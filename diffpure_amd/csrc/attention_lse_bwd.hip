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

#define BWD_WAVES(DT, DP) ((DP) <= ((DT) == 0 ? 128 : 64) ? 2 : 1)

template <int DT, int DP, int CW>
__global__ __launch_bounds__(256) AL_WAVES(BWD_WAVES(DT, DP)) void attn_lse_dq_kernel(Args p) {
    using T = Tr<DT>;
    constexpr int NW = 4, BM = T::TILE, RB = DP * T::ES, KS = DP / 16, ND = DP / T::TILE, NKK = T::TILE / 16, COLS = NW * CW * T::TILE;
    using St = Stream<RB, BM, NW>;
    __shared__ __attribute__((aligned(1024))) char smem[2 * St::STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cl = lane & (T::TILE - 1), g = lane / T::TILE;
    const int nblk = (p.Tq + COLS - 1) / COLS;
    const int bid = logical_block(p.xcd_map);
    const int z = bid / nblk, blk = p.causal ? nblk - 1 - (bid - z * nblk) : bid - z * nblk;
    const int b = z / p.Hq, h = z - b * p.Hq, hk = h / (p.Hq / p.Hkv);
    const int n = clamp_len(p.q_lens, b, p.Tq), m = clamp_len(p.kv_lens, b, p.Tk), off = m - n;
    const int c0 = blk * COLS, wc0 = c0 + wave * CW * T::TILE;
    const int row_slots = p.D * T::ES / 16;
    const float c = p.scale * LOG2E;

    typename T::Frag qf[CW][KS], df[CW][KS];
    typename T::Acc dq[CW][ND], nd[CW];
    float l2[CW];
#pragma unroll
    for (int cw = 0; cw < CW; ++cw) {
        const int col = wc0 + cw * T::TILE + cl, row = col < n ? col : (n > 0 ? n - 1 : 0);
        ld_kept<DT, KS>(qf[cw], p.q.p + b * p.q.b + h * p.q.h + (long long)row * p.q.t, row_slots, g);
        ld_kept<DT, KS>(df[cw], p.dout.p + b * p.dout.b + h * p.dout.h + (long long)row * p.dout.t, row_slots, g);
        float delta = 0.f;
        {
            typename T::Frag of[KS];
            ld_kept<DT, KS>(of, p.o.p + b * p.o.b + h * p.o.h + (long long)row * p.o.t, row_slots, g);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int j = 0; j < 16 / T::ES; ++j) delta = fmaf((float)df[cw][ks][j], (float)of[ks][j], delta);
        }
        delta = col_sum<T::TILE>(delta);
        const float lse = p.lse[(long long)z * p.Tq + row];
        const bool some = col < n && lse > -INFINITY;
        l2[cw] = some ? lse * LOG2E - (float)T::PSHIFT : INFINITY;
        if (!some) delta = 0.f;
        if (g == 0 && col < p.Tqp) {
            float* w = p.ws + (long long)z * p.Tqp + col;
            w[0] = l2[cw];
            w[(long long)p.B * p.Hq * p.Tqp] = delta;
        }
#pragma unroll
        for (int r = 0; r < T::NR; ++r) nd[cw][r] = -delta;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) dq[cw][dt] = typename T::Acc{};
    }

    int rows_end = c0 < n ? m : 0;
    if (p.causal) {
        const int last = (c0 + COLS < n ? c0 + COLS : n) - 1 + off;
        rows_end = last + 1 < rows_end ? last + 1 : rows_end;
    }
    St st;
    st.init(p.k.p + b * p.k.b + hk * p.k.h, p.k.t, p.v.p + b * p.v.b + hk * p.v.h, p.v.t, row_slots, wave, lane);
    if (rows_end > 0) st.issue(smem, 0, m, 0, 0, wave);
    int cur = 0;
    for (int r0 = 0; r0 < rows_end; r0 += BM, cur ^= 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (r0 + BM < rows_end) st.issue(smem + (cur ^ 1) * St::STAGE, r0 + BM, m, 0, 0, wave);
        const char* Ks = smem + cur * St::STAGE;
        const char* Vs = Ks + St::TILE_BYTES;
        auto tile = [&](auto masked) {
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
                int end = p.causal ? wc0 + cw * T::TILE + cl + off + 1 : m;
                end = (end < m ? end : m) - r0 - 4 * g;
#pragma unroll
                for (int r = 0; r < T::NR; ++r) s[cw][r] = reg_row<DT>(r) < end ? s[cw][r] : 0.f;
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
        settle();
        };
        if (p.causal && r0 > wc0 + CW * T::TILE - 1 + off) {}
        else if (r0 + BM > m || (p.causal && r0 + BM - 1 > wc0 + off)) tile(yes{});
        else tile(no{});
    }
    const float mul = p.scale / (float)(1 << T::PSHIFT);
#pragma unroll
    for (int cw = 0; cw < CW; ++cw) {
        const int col = wc0 + cw * T::TILE + cl;
        if (col >= p.Tq) continue;
        if (col >= n) {
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) dq[cw][dt] = typename T::Acc{};
        }
        st_col<DT, ND>(dq[cw], mul, const_cast<char*>(p.w0.p) + b * p.w0.b + h * p.w0.h + (long long)col * p.w0.t, p.D, g);
    }
}

template <int DT, int DP, int CW>
__global__ __launch_bounds__(256) AL_WAVES(BWD_WAVES(DT, DP)) void attn_lse_dkv_kernel(Args p) {
    using T = Tr<DT>;
    constexpr int NW = 4, BM = T::TILE, RB = DP * T::ES, KS = DP / 16, ND = DP / T::TILE, NKK = T::TILE / 16, COLS = NW * CW * T::TILE;
    using St = Stream<RB, BM, NW>;
    __shared__ __attribute__((aligned(1024))) char smem[2 * St::STAGE];
    __shared__ __attribute__((aligned(16))) float rows[2][2][BM];       // stage: log-sum-exp, delta of the streamed queries
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cl = lane & (T::TILE - 1), g = lane / T::TILE;
    const int nblk = (p.Tk + COLS - 1) / COLS, group = p.Hq / p.Hkv;
    const int bid = logical_block(p.xcd_map);
    const int z = bid / nblk, blk = bid - z * nblk;                    // causal: the first blocks are the long ones
    const int b = z / p.Hkv, hk = z - b * p.Hkv;
    const int n = clamp_len(p.q_lens, b, p.Tq), m = clamp_len(p.kv_lens, b, p.Tk), off = m - n;
    const int c0 = blk * COLS, wc0 = c0 + wave * CW * T::TILE;
    const int row_slots = p.D * T::ES / 16;
    const float c = p.scale * LOG2E;

    typename T::Frag kf[CW][KS], vf[CW][KS];
    typename T::Acc dk[CW][ND], dv[CW][ND];
#pragma unroll
    for (int cw = 0; cw < CW; ++cw) {
        const int col = wc0 + cw * T::TILE + cl, row = col < m ? col : (m > 0 ? m - 1 : 0);
        ld_kept<DT, KS>(kf[cw], p.k.p + b * p.k.b + hk * p.k.h + (long long)row * p.k.t, row_slots, g);
        ld_kept<DT, KS>(vf[cw], p.v.p + b * p.v.b + hk * p.v.h + (long long)row * p.v.t, row_slots, g);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) dk[cw][dt] = dv[cw][dt] = typename T::Acc{};
    }

    int first = 0;                                                     // first query tile that sees a key of this workgroup
    if (p.causal && c0 - off > 0) first = (c0 - off) / BM * BM;
    const int per_head = c0 < m && first < n ? (n - first + BM - 1) / BM : 0;
    const int steps = per_head * group;                                // the query tiles of every head of the group, one after the other
    St st;
    st.init(p.q.p + b * p.q.b + hk * group * p.q.h, p.q.t, p.dout.p + b * p.dout.b + hk * group * p.dout.h, p.dout.t, row_slots, wave, lane);
    const float* ws = p.ws + ((long long)b * p.Hq + hk * group) * p.Tqp;
    const long long half = (long long)p.B * p.Hq * p.Tqp;
    // thread t < 2 BM carries one value of a tile: log-sum-exp (t < BM) or delta of query t % BM
    const float* my = ws + (tid >= BM ? half : 0) + (tid & (BM - 1));
    int head = 0, r0 = first;
    if (steps > 0) {
        st.issue(smem, r0, n, 0, 0, wave);
        if (tid < 2 * BM) rows[0][tid / BM][tid & (BM - 1)] = my[r0];
    }
    for (int it = 0; it < steps; ++it) {
        const int cur = it & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        int nr = r0 + BM, nh = head;
        if (nr >= n) {
            nr = first;
            ++nh;
        }
        float next = 0.f;
        if (it + 1 < steps) {
            st.issue(smem + (cur ^ 1) * St::STAGE, nr, n, nh * p.q.h, nh * p.dout.h, wave);
            if (tid < 2 * BM) next = my[(long long)nh * p.Tqp + nr];
        }
        const char* Qs = smem + cur * St::STAGE;
        const char* Ds = Qs + St::TILE_BYTES;
        auto tile = [&](auto masked) {
            typename T::Acc l2, nd;
#pragma unroll
            for (int r = 0; r < T::NR; r += 4) {
                const f32x4 a = *reinterpret_cast<const f32x4*>(&rows[cur][0][r * T::G + 4 * g]);
                const f32x4 d = *reinterpret_cast<const f32x4*>(&rows[cur][1][r * T::G + 4 * g]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    l2[r + j] = a[j];
                    nd[r + j] = -d[j];
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
                const typename T::Frag aq = ld_row<DT, RB>(Qs, lane, ks), ad = ld_row<DT, RB>(Ds, lane, ks);
#pragma unroll
                for (int cw = 0; cw < CW; ++cw) {
                    s[cw] = T::mma(aq, kf[cw][ks], s[cw]);
                    ds[cw] = T::mma(ad, vf[cw][ks], ds[cw]);
                }
            }
#pragma unroll
            for (int cw = 0; cw < CW; ++cw)
#pragma unroll
                for (int r = 0; r < T::NR; ++r) s[cw][r] = __builtin_amdgcn_exp2f(fmaf(s[cw][r], c, -l2[r]));
            if constexpr (masked.value) {
#pragma unroll
                for (int cw = 0; cw < CW; ++cw) {
                    const int begin = wc0 + cw * T::TILE + cl - off - r0 - 4 * g;       // first row of the tile that sees this key
#pragma unroll
                    for (int r = 0; r < T::NR; ++r) s[cw][r] = reg_row<DT>(r) >= begin ? s[cw][r] : 0.f;
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
                    pf[cw] = pack<DT>(s[cw], kk);
                    sf[cw] = pack<DT>(ds[cw], kk);
                }
#pragma unroll
                for (int dt = 0; dt < ND; ++dt) {
                    const typename T::Frag ad = ld_tr<DT, RB>(Ds, lane, kk, dt), aq = ld_tr<DT, RB>(Qs, lane, kk, dt);
#pragma unroll
                    for (int cw = 0; cw < CW; ++cw) {
                        dv[cw][dt] = T::mma(ad, pf[cw], dv[cw][dt]);
                        dk[cw][dt] = T::mma(aq, sf[cw], dk[cw][dt]);
                    }
                }
            }
            settle();
        };
        if (p.causal && r0 + BM - 1 + off < wc0) {}                    // no query of the tile sees a key of this wave
        else if (p.causal && r0 + off < wc0 + CW * T::TILE - 1) tile(yes{});
        else tile(no{});
        if (it + 1 < steps && tid < 2 * BM) rows[cur ^ 1][tid / BM][tid & (BM - 1)] = next;
        r0 = nr;
        head = nh;
    }
    const float pm = 1.f / (float)(1 << T::PSHIFT);
#pragma unroll
    for (int cw = 0; cw < CW; ++cw) {
        const int col = wc0 + cw * T::TILE + cl;
        if (col >= p.Tk) continue;
        if (col >= m) {
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) dk[cw][dt] = dv[cw][dt] = typename T::Acc{};
        }
        st_col<DT, ND>(dk[cw], p.scale * pm, const_cast<char*>(p.w0.p) + b * p.w0.b + hk * p.w0.h + (long long)col * p.w0.t, p.D, g);
        st_col<DT, ND>(dv[cw], pm, const_cast<char*>(p.w1.p) + b * p.w1.b + hk * p.w1.h + (long long)col * p.w1.t, p.D, g);
    }
}

template <int DT, int DP>
void launch_bwd(const Args& a, const Ten& dq, const Ten& dk, const Ten& dv, hipStream_t s) {
    constexpr int COLS = 4 * Tr<DT>::TILE;
    Args x = a;
    x.w0 = dq;
    hipLaunchKernelGGL((attn_lse_dq_kernel<DT, DP, 1>), dim3((unsigned)((long long)a.B * a.Hq * ((a.Tq + COLS - 1) / COLS))), dim3(256), 0, s, x);
    x.w0 = dk;
    x.w1 = dv;
    hipLaunchKernelGGL((attn_lse_dkv_kernel<DT, DP, 1>), dim3((unsigned)((long long)a.B * a.Hkv * ((a.Tk + COLS - 1) / COLS))), dim3(256), 0, s, x);
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

extern "C" long long dp_attention_lse_bwd_workspace(int B, int Tq, int Hq) {
    if (B <= 0 || Tq <= 0 || Hq <= 0) return 0;
    return 2LL * B * Hq * ((Tq + 63LL) / 64 * 64) * 4;
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
    DP_REQUIRE(work && dp_aligned16(work) && work_bytes >= dp_attention_lse_bwd_workspace(B, Tq, Hq), "%s: workspace of %lld bytes needed (got %lld)", fn,
               dp_attention_lse_bwd_workspace(B, Tq, Hq), work_bytes);
    a.lse = const_cast<float*>(lse);
    a.ws = static_cast<float*>(work);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == 0) launch_bwd<0>(a, tq, tk, tv, s);
    else if (dtype == 1) launch_bwd<1>(a, tq, tk, tv, s);
    else launch_bwd<2>(a, tq, tk, tv, s);
    DP_LAUNCH_CHECK("attn_lse_bwd");
    return 0;
}
