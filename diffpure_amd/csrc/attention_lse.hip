// out = softmax(scale q k^T + mask) v with the log-sum-exp of every row, for [B, T, H, D] tensors of any strides, token counts, head
// dimensions up to 256 and types: what a backward pass that recomputes the probabilities (attention_lse_bwd.hip) starts from.
#include "attention_lse.h"

namespace {
using namespace al;

// One workgroup = 4 waves, each CW tiles of query columns; K and V tiles of TILE rows stream through LDS (double buffered).
// The running maximum is only moved when a row's maximum has grown by more than 8 (in log2): until then the probabilities are taken
// against the old one - at most 2^8, exact in every type's range - and neither sum nor output is rescaled.
template <int DT, int DP, int CW>
__global__ __launch_bounds__(256) AL_WAVES(DP <= 128 ? 2 : 1) void attn_lse_fwd_kernel(Args p) {
    using T = Tr<DT>;
    constexpr int NW = 4, BM = T::TILE, RB = DP * T::ES, KS = DP / 16, ND = DP / T::TILE, NKK = T::TILE / 16, COLS = NW * CW * T::TILE;
    using St = Stream<RB, BM, NW>;
    __shared__ __attribute__((aligned(1024))) char smem[2 * St::STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cl = lane & (T::TILE - 1), g = lane / T::TILE;
    const int nblk = (p.Tq + COLS - 1) / COLS;
    const int bid = logical_block(p.xcd_map);
    const int z = bid / nblk, blk = p.causal ? nblk - 1 - (bid - z * nblk) : bid - z * nblk;     // causal: the long blocks first
    const int b = z / p.Hq, h = z - b * p.Hq, hk = h / (p.Hq / p.Hkv);
    const int n = clamp_len(p.q_lens, b, p.Tq), m = clamp_len(p.kv_lens, b, p.Tk), off = m - n;
    const int c0 = blk * COLS, wc0 = c0 + wave * CW * T::TILE;       // first column of the workgroup / of this wave
    const int row_slots = p.D * T::ES / 16;
    const float c = fabsf(p.scale) * LOG2E;

    typename T::Frag qf[CW][KS];
#pragma unroll
    for (int cw = 0; cw < CW; ++cw) {
        const int col = wc0 + cw * T::TILE + cl, row = col < n ? col : (n > 0 ? n - 1 : 0);
        ld_kept<DT, KS>(qf[cw], p.q.p + b * p.q.b + h * p.q.h + (long long)row * p.q.t, row_slots, g);
        if (p.scale < 0.f) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) qf[cw][ks] = -qf[cw][ks];
        }
    }
    typename T::Acc o[CW][ND];
    float mx[CW], l[CW];
#pragma unroll
    for (int cw = 0; cw < CW; ++cw) {
        mx[cw] = -INFINITY;
        l[cw] = 0.f;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) o[cw][dt] = typename T::Acc{};
    }

    int rows_end = c0 < n ? m : 0;
    if (p.causal) {
        const int last = (c0 + COLS < n ? c0 + COLS : n) - 1 + off;      // last key of the last query
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
        typename T::Acc s[CW];
#pragma unroll
        for (int cw = 0; cw < CW; ++cw) s[cw] = typename T::Acc{};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const typename T::Frag a = ld_row<DT, RB>(Ks, lane, ks);
#pragma unroll
            for (int cw = 0; cw < CW; ++cw) s[cw] = T::mma(a, qf[cw][ks], s[cw]);
        }
        if constexpr (masked.value) {
#pragma unroll
            for (int cw = 0; cw < CW; ++cw) {
                int end = p.causal ? wc0 + cw * T::TILE + cl + off + 1 : m;
                end = (end < m ? end : m) - r0 - 4 * g;
#pragma unroll
                for (int r = 0; r < T::NR; ++r) s[cw][r] = reg_row<DT>(r) < end ? s[cw][r] : -INFINITY;
            }
        }
#pragma unroll
        for (int cw = 0; cw < CW; ++cw) {
            float mb = s[cw][0];
#pragma unroll
            for (int r = 1; r < T::NR; ++r) mb = fmaxf(mb, s[cw][r]);
            mb = col_max<T::TILE>(mb);
            const bool grow = mb * c > mx[cw] * c + 8.f;
            if (__any(grow)) {
                const float nm = grow ? mb : mx[cw];
                const float alpha = mx[cw] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mx[cw] - nm) * c);
                mx[cw] = nm;
                l[cw] *= alpha;
#pragma unroll
                for (int dt = 0; dt < ND; ++dt)
#pragma unroll
                    for (int r = 0; r < T::NR; ++r) o[cw][dt][r] *= alpha;
            }
            const float mc = mx[cw] == -INFINITY ? 0.f : mx[cw] * c;
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < T::NR; ++r) {
                s[cw][r] = __builtin_amdgcn_exp2f(fmaf(s[cw][r], c, -mc));
                sum += s[cw][r];
            }
            l[cw] += sum;
        }
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) {
            typename T::Frag pf[CW];
#pragma unroll
            for (int cw = 0; cw < CW; ++cw) pf[cw] = pack<DT>(s[cw], kk);
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) {
                const typename T::Frag a = ld_tr<DT, RB>(Vs, lane, kk, dt);
#pragma unroll
                for (int cw = 0; cw < CW; ++cw) o[cw][dt] = T::mma(a, pf[cw], o[cw][dt]);
            }
        }
        settle();
        };
        if (p.causal && r0 > wc0 + CW * T::TILE - 1 + off) {}            // every key of the tile lies behind this wave's queries
        else if (r0 + BM > m || (p.causal && r0 + BM - 1 > wc0 + off)) tile(yes{});
        else tile(no{});
    }

#pragma unroll
    for (int cw = 0; cw < CW; ++cw) {
        const int col = wc0 + cw * T::TILE + cl;
        const float sum = col_sum<T::TILE>(l[cw]);
        if (col >= p.Tq) continue;
        const bool some = col < n && sum > 0.f;
        if (!some) {
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) o[cw][dt] = typename T::Acc{};
        }
        st_col<DT, ND>(o[cw], some ? 1.f / sum : 0.f, const_cast<char*>(p.w0.p) + b * p.w0.b + h * p.w0.h + (long long)col * p.w0.t, p.D, g);
        if (g == 0) p.lse[(long long)z * p.Tq + col] = some ? mx[cw] * fabsf(p.scale) + logf(sum) : -INFINITY;
    }
}

template <int DT, int DP>
void launch_fwd(const Args& a, hipStream_t s) {
    constexpr int COLS = 4 * Tr<DT>::TILE;
    const long long blocks = (long long)a.B * a.Hq * ((a.Tq + COLS - 1) / COLS);
    hipLaunchKernelGGL((attn_lse_fwd_kernel<DT, DP, 1>), dim3((unsigned)blocks), dim3(256), 0, s, a);
}
template <int DT>
void launch_fwd(const Args& a, hipStream_t s) {
    if (a.D <= 32) launch_fwd<DT, 32>(a, s);
    else if (a.D <= 64) launch_fwd<DT, 64>(a, s);
    else if (a.D <= 96) launch_fwd<DT, 96>(a, s);
    else if (a.D <= 128) launch_fwd<DT, 128>(a, s);
    else launch_fwd<DT, 256>(a, s);
}

}  // namespace

// strides: 3 per tensor (batch, token, head) in elements
bool dp_attn_lse_tensor(const char* fn, const char* name, const void* ptr, const long long* st, int es, int B, int Tn, int H, bool written, al::Ten* t) {
    if (!ptr || !dp_aligned16(ptr)) {
        dp_set_error("%s: %s is null or not 16-byte aligned", fn, name);
        return false;
    }
    const int n[3] = {B, Tn, H};
    for (int i = 0; i < 3; ++i) {
        if (st[i] < 0 || (st[i] * es) % 16 != 0 || st[i] > (1LL << 40) || (written && n[i] > 1 && st[i] == 0)) {
            dp_set_error("%s: %s strides must be multiples of 16 bytes, of a written tensor also positive (got %lld elements at position %d)", fn, name, st[i], i);
            return false;
        }
    }
    *t = al::Ten{static_cast<const char*>(ptr), st[0] * es, st[1] * es, st[2] * es};
    return true;
}

int dp_attn_lse_common(const char* fn, const void* q, const void* k, const void* v, const long long* strides, int dtype, int B, int Tq, int Tk, int Hq,
                       int Hkv, int D, const int* q_lens, const int* kv_lens, float scale, int causal, al::Args* a) {
    DP_REQUIRE(strides, "%s: strides missing", fn);
    DP_REQUIRE(dtype >= 0 && dtype <= 2, "%s: dtype %d (0 = fp32, 1 = fp16, 2 = bf16)", fn, dtype);
    DP_REQUIRE(B > 0 && Tq > 0 && Tk > 0 && Hq > 0 && Hkv > 0, "%s: sizes must be positive (B %d, Tq %d, Tk %d, Hq %d, Hkv %d)", fn, B, Tq, Tk, Hq, Hkv);
    DP_REQUIRE(Hq % Hkv == 0, "%s: %d query heads are not a multiple of %d key heads", fn, Hq, Hkv);
    DP_REQUIRE(D > 0 && D % 8 == 0 && D <= 256, "%s: the head dimension must be a multiple of 8 up to 256 (got %d)", fn, D);
    DP_REQUIRE(Tq <= (1 << 30) && Tk <= (1 << 30), "%s: at most 2^30 tokens (got %d, %d)", fn, Tq, Tk);
    DP_REQUIRE((long long)B * Hq * ((Tq + 63) / 64) < (1LL << 31) && (long long)B * Hkv * ((Tk + 63) / 64) < (1LL << 31), "%s: too many blocks", fn);
    DP_REQUIRE(scale != 0.f && scale - scale == 0.f, "%s: the scale must be finite and not zero", fn);
    const int es = dtype == 0 ? 4 : 2;
    if (!dp_attn_lse_tensor(fn, "q", q, strides, es, B, Tq, Hq, false, &a->q) || !dp_attn_lse_tensor(fn, "k", k, strides + 3, es, B, Tk, Hkv, false, &a->k) ||
        !dp_attn_lse_tensor(fn, "v", v, strides + 6, es, B, Tk, Hkv, false, &a->v))
        return 1;
    a->q_lens = q_lens;
    a->kv_lens = kv_lens;
    a->B = B; a->Tq = Tq; a->Tk = Tk; a->Hq = Hq; a->Hkv = Hkv; a->D = D;
    a->Tqp = (Tq + 63) / 64 * 64;
    a->scale = scale;
    a->causal = causal != 0;
    a->xcd_map = dp_tune(DP_T_XCD_MAP) != 0;
    return 0;
}

extern "C" int dp_attention_lse(const void* q, const void* k, const void* v, const long long* strides, int dtype, int B, int Tq, int Tk, int Hq, int Hkv,
                                int D, const int* q_lens, const int* kv_lens, float scale, int causal, void* out, float* lse, void* stream) {
    al::Args a{};
    if (int rc = dp_attn_lse_common("dp_attention_lse", q, k, v, strides, dtype, B, Tq, Tk, Hq, Hkv, D, q_lens, kv_lens, scale, causal, &a)) return rc;
    DP_REQUIRE(lse, "dp_attention_lse: lse missing");
    if (!dp_attn_lse_tensor("dp_attention_lse", "out", out, strides + 9, dtype == 0 ? 4 : 2, B, Tq, Hq, true, &a.w0)) return 1;
    a.lse = lse;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == 0) launch_fwd<0>(a, s);
    else if (dtype == 1) launch_fwd<1>(a, s);
    else launch_fwd<2>(a, s);
    DP_LAUNCH_CHECK("attn_lse_fwd");
    return 0;
}
