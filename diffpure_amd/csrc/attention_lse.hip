// out = softmax(scale q k^T + mask) v with the log-sum-exp of every row, for [B, T, H, D] tensors of any strides, token counts, head
// dimensions up to 256 and types: what a backward pass that recomputes the probabilities (attention_lse_bwd.hip) starts from.
//
// One pass over the keys with a running maximum and sum per query; the scores of a tile never leave the registers.  Measured on MI355X:
//   64 x 1024 tokens, 8 heads of 64, fp16    192 us (whole call), 715 TFLOP/s: by the counters vector instructions keep a SIMD busy for 75 % of the launch and matrix
//                                            instructions for 36 %, so the two hardly overlap, though 119 registers leave four waves per SIMD; 108 vector
//                                            instructions per 32 x 32 tile, of which 16 exponentials (16 cycles each)
//   64 x 197 tokens, 12 heads of 64, bf16    24 us: 1.48 times the work (128-column blocks, 32-key tiles), short workgroups
//   4 x 1 query, 50 001 keys, 16 / 4 heads of 128, bf16    90.5 us = 4.5 TB/s: the heads of a group packed into one tile, four waves on different rows,
//                                            16 ranges of keys joined by a second launch (5 us)
//   32 x 1024 tokens, 8 heads of 64, fp32    604 us = 114 TFLOP/s of the 154 that a large fp32 product reaches
// Above 128 channels the fp32 form spills 27 registers (128 x 256 tokens x 1 head of 256: 92 us, its operations 56).
#include "attention_lse.h"

namespace {
using namespace al;

// One workgroup = 4 waves; K and V tiles stream through LDS (double buffered).  RS = 1: every wave has its own tile of query columns and sees every
// streamed row.  RS > 1 (few columns): RS waves share their columns and take different rows of a stage; they join at the end.
// The running maximum is only moved when a row's maximum has grown by more than 8 (in log2): until then the probabilities are taken
// against the old one - at most 2^8, exact in every type's range - and neither sum nor output is rescaled.
template <int DT, int DP, int RS>
__global__ __launch_bounds__(256) AL_WAVES(2) void attn_lse_fwd_kernel(Args p) {
    using T = Tr<DT>;
    constexpr int NW = 4, BM = RS * T::ROWS, RB = DP * T::ES, KS = DP / T::KSTEP, ND = DP / T::TILE, NKK = T::ROWS / T::KROWS, COLS = NW / RS * T::TILE;
    using St = Stream<RB, T::ES, BM, NW>;
    __shared__ __attribute__((aligned(1024))) char smem[2 * St::STAGE];
    __shared__ float ml[RS > 1 ? 2 : 1][NW][T::TILE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rw = wave % RS, cl = lane & (T::TILE - 1), g = lane / T::TILE;
    const int bid0 = logical_block(p.xcd_map), split = bid0 % p.splits, bid = bid0 / p.splits;
    const int cols0 = p.packed ? p.Hq / p.Hkv * p.Tq : p.Tq, nblk = (cols0 + COLS - 1) / COLS;
    const int z = bid / nblk, blk = block_of(p, bid - z * nblk, nblk, true);
    if (z >= p.B * (p.packed ? p.Hkv : p.Hq)) return;
    const Kept kept(p, z);
    const int b = kept.b;
    const int n = clamp_len(p.q_lens, b, p.Tq), m = clamp_len(p.kv_lens, b, p.Tk), off = m - n;
    const int c0 = blk * COLS, col = c0 + wave / RS * T::TILE + cl;       // first column of the workgroup, this lane's
    const int row_slots = p.D * T::ES / 16;
    const float c = fabsf(p.scale) * LOG2E;

    typename T::Frag qf[KS];
    int head, tok;
    kept.col(p, col < kept.cols ? col : kept.cols - 1, head, tok);
    ld_kept<DT, KS>(qf, p.q.p + b * p.q.b + head * p.q.h + (tok < n ? tok : (n > 0 ? n - 1 : 0)) * p.q.t, row_slots, g);
    if (p.scale < 0.f) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[ks] = -qf[ks];
    }
    typename T::Acc o[ND];
    float mx = -INFINITY, l = 0.f;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) o[dt] = typename T::Acc{};

    // streamed rows: [begin, open) are seen by every column, [open, end) through the mask
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
        const char *Ks = smem + cur * St::STAGE + rw * T::ROWS * RB, *Vs = Ks + St::TILE_BYTES;
        cur ^= 1;
        Score<DT> s{};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) mma_rows<DT, RB>(Ks, lane, ks, qf[ks], s);
        if constexpr (masked.value) {
            const int seen = min(end, p.causal ? tok + off + 1 : end) - r0 - rw * T::ROWS - 4 * g;
#pragma unroll
            for (int r = 0; r < s.N; ++r) s.set(r, reg_row<DT>(r) < seen ? s.get(r) : -INFINITY);
        }
        float mb = s.get(0);
#pragma unroll
        for (int r = 1; r < s.N; ++r) mb = fmaxf(mb, s.get(r));
        mb = col_max<T::TILE>(mb);
        const bool grow = mb * c > mx * c + 8.f;
        if (__any(grow)) {
            const float nm = grow ? mb : mx;
            const float alpha = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mx - nm) * c);
            mx = nm;
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < ND; ++dt)
#pragma unroll
                for (int r = 0; r < T::NR; ++r) o[dt][r] *= alpha;
        }
        const float mc = mx == -INFINITY ? 0.f : mx * c;
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < s.N; ++r) {
            s.set(r, __builtin_amdgcn_exp2f(fmaf(s.get(r), c, -mc)));
            sum += s.get(r);
        }
        l += sum;
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) {
            const typename T::Frag pf = s.pack(kk);
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) o[dt] = T::mma(ld_tr<DT, RB>(Vs, lane, kk, dt), pf, o[dt]);
        }
        settle();
    };
    int r0 = begin;
    for (; r0 < open; r0 += BM) body(r0, no{});
    for (; r0 < end; r0 += BM) body(r0, yes{});

    float sum = col_sum<T::TILE>(l), top = mx, mine = 1.f;
    if constexpr (RS > 1) {
        if (g == 0) {
            ml[0][wave][cl] = top;
            ml[1][wave][cl] = sum;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < RS; ++w) top = fmaxf(top, ml[0][wave - rw + w][cl]);
        const float tc = top == -INFINITY ? 0.f : top * c;
        mine = __builtin_amdgcn_exp2f(mx * c - tc);
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < RS; ++w) sum += ml[1][wave - rw + w][cl] * __builtin_amdgcn_exp2f(ml[0][wave - rw + w][cl] * c - tc);
    }
    // a range in which a row meets no key (or scores of -inf only) has weight 0 in the join; a row that sees keys and sums to 0 in all is 0 / 0
    const bool some = keys_seen(tok, n, m, p.causal) > 0 && (p.splits == 1 || sum != 0.f), out = col < kept.cols;
    const float inv = some ? 1.f / sum : 0.f, lse = some ? top * fabsf(p.scale) + logf(sum) : -INFINITY;
    const long long kr = (long long)z * kept.cols + col + (long long)split * (p.packed ? p.Hkv : p.Hq) * p.B * kept.cols;
    char* row = const_cast<char*>(p.w0.p) + b * p.w0.b + head * p.w0.h + tok * p.w0.t;
    if (RS == 1 && p.splits == 1) {
        __syncthreads();
        const int first = c0 + wave * T::TILE;
        store_cols<DT, ND, RB>(o, inv, smem + wave * T::TILE * RB, lane, row_slots, [&](int i) -> char* {
            int h, t;
            kept.col(p, min(first + i, kept.cols - 1), h, t);
            return first + i < kept.cols ? const_cast<char*>(p.w0.p) + b * p.w0.b + h * p.w0.h + t * p.w0.t : nullptr;
        });
    } else join_units<DT, ND, RS>(o, mine, smem, wave, rw, lane, [&](int u, f32x4 v) {
        const int d = Units<DT, ND>::d(u, g);
        if (!out || d >= p.D) return;
        v = some ? v * inv : f32x4{};
        if (p.splits > 1) *reinterpret_cast<f32x4*>(p.part0 + kr * p.D + d) = v;
        else st4<DT>(row, d, v);
    });
    if (out && g == 0 && rw == 0) {
        if (p.splits > 1) p.part_lse[kr] = lse;
        else p.lse[((long long)b * p.Hq + head) * p.Tq + tok] = lse;
    }
}

// joins the ranges of a split launch: out = sum_s 2^(lse_s - lse) out_s.  One thread per four channels of a kept row.
template <int DT>
__global__ __launch_bounds__(256) void attn_lse_join_kernel(Args p) {
    const int per = p.D / 4, heads = p.packed ? p.Hkv : p.Hq, cols = p.packed ? p.Hq / p.Hkv * p.Tq : p.Tq;
    const long long rows = (long long)p.B * heads * cols, id = (long long)blockIdx.x * 256 + threadIdx.x, kr = id / per;
    const int d = (int)(id - kr * per) * 4;
    if (kr >= rows) return;
    const int z = (int)(kr / cols);
    const Kept kept(p, z);
    int h, t;
    kept.col(p, (int)(kr - (long long)z * cols), h, t);
    const bool some = keys_seen(t, clamp_len(p.q_lens, kept.b, p.Tq), clamp_len(p.kv_lens, kept.b, p.Tk), p.causal) > 0;
    // eight loads under way at a time (ranges behind the last one repeat it with weight 0); a range that is NaN is not the largest, but its weight is NaN
    float top = -INFINITY, sum = 0.f;
    for (int s0 = 0; s0 < p.splits; s0 += 8) {
        float l[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) l[i] = p.part_lse[min(s0 + i, p.splits - 1) * rows + kr];
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, l[i]);
    }
    f32x4 v = {};
    if (top == -INFINITY) top = 0.f;
    if (some) {
        for (int s0 = 0; s0 < p.splits; s0 += 8) {
            float l[8];
            f32x4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const long long at = min(s0 + i, p.splits - 1) * rows + kr;
                l[i] = p.part_lse[at];
                x[i] = *reinterpret_cast<const f32x4*>(p.part0 + at * p.D + d);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float w = s0 + i < p.splits ? __builtin_amdgcn_exp2f((l[i] - top) * LOG2E) : 0.f;
                sum += w;
                v += w * x[i];
            }
        }
        v *= 1.f / sum;
    }
    st4<DT>(const_cast<char*>(p.w0.p) + kept.b * p.w0.b + h * p.w0.h + t * p.w0.t, d, v);
    if (d == 0) p.lse[((long long)kept.b * p.Hq + h) * p.Tq + t] = some ? top + logf(sum) : -INFINITY;
}

template <int DTYPE, int DP>
void launch_fwd(Args a, hipStream_t s) {
    constexpr int DT = shape_of(DTYPE, DP), FEW = DP > 128 ? 2 : 4;
    const QPlan pl = q_plan(DTYPE, a.B, a.Tq, a.Tk, a.Hq, a.Hkv, DP);
    a.packed = pl.packed;
    a.splits = pl.splits;
    a.split_rows = pl.split_rows;
    a.stripes = stripes_of((long long)a.B * (pl.packed ? a.Hkv : a.Hq));
    if (pl.rs == 1) hipLaunchKernelGGL((attn_lse_fwd_kernel<DT, DP, 1>), dim3((unsigned)(pl.blocks * pl.splits)), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((attn_lse_fwd_kernel<DT, DP, FEW>), dim3((unsigned)(pl.blocks * pl.splits)), dim3(256), 0, s, a);
    if (pl.splits > 1) {
        const long long items = (long long)a.B * a.Hq * a.Tq * (a.D / 4);
        hipLaunchKernelGGL(attn_lse_join_kernel<DTYPE>, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, s, a);
    }
}
template <int DTYPE>
void launch_fwd(const Args& a, hipStream_t s) {
    if (a.D <= 32) launch_fwd<DTYPE, 32>(a, s);
    else if (a.D <= 64) launch_fwd<DTYPE, 64>(a, s);
    else if (a.D <= 96) launch_fwd<DTYPE, 96>(a, s);
    else if (a.D <= 128) launch_fwd<DTYPE, 128>(a, s);
    else launch_fwd<DTYPE, 256>(a, s);
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
        if (i == 1 && st[i] * es > 1 << 24) {
            dp_set_error("%s: %s: tokens lie more than 2^24 bytes apart (%lld elements)", fn, name, st[i]);
            return false;
        }
        if (st[i] < 0 || (st[i] * es) % 16 != 0 || st[i] > (1LL << 40) || (written && n[i] > 1 && st[i] == 0)) {
            dp_set_error("%s: %s strides must be multiples of 16 bytes, of a written tensor also positive (got %lld elements at position %d)", fn, name, st[i], i);
            return false;
        }
    }
    *t = al::Ten{static_cast<const char*>(ptr), st[0] * es, st[1] * es, st[2] * es};
    return true;
}

dp::Region dp_attn_lse_region(const char* name, const al::Ten& t, int B, int Tn, int H, long long row) {
    return dp::Region{name, (intptr_t)t.p, {B, Tn, H}, {t.b, t.t, t.h}, row};
}

int dp_attn_lse_common(const char* fn, const void* q, const void* k, const void* v, const long long* strides, int dtype, int B, int Tq, int Tk, int Hq,
                       int Hkv, int D, const int* q_lens, const int* kv_lens, float scale, int causal, al::Args* a) {
    DP_REQUIRE(strides, "%s: strides missing", fn);
    DP_REQUIRE(dtype >= 0 && dtype <= 2, "%s: dtype %d (0 = fp32, 1 = fp16, 2 = bf16)", fn, dtype);
    DP_REQUIRE(B > 0 && Tq > 0 && Tk > 0 && Hq > 0 && Hkv > 0, "%s: sizes must be positive (B %d, Tq %d, Tk %d, Hq %d, Hkv %d)", fn, B, Tq, Tk, Hq, Hkv);
    DP_REQUIRE(Hq % Hkv == 0, "%s: %d query heads are not a multiple of %d key heads", fn, Hq, Hkv);
    DP_REQUIRE(D > 0 && D % 8 == 0 && D <= 256, "%s: the head dimension must be a multiple of 8 up to 256 (got %d)", fn, D);
    DP_REQUIRE(Tq <= (1 << 30) && Tk <= (1 << 30), "%s: at most 2^30 tokens (got %d, %d)", fn, Tq, Tk);
    const int cols = 4 * al::tile_of(dtype, al::padded_dim(D));       // a grid has fewer than 2^32 threads; the launch that keeps keys has up to two workgroups of 256 per block
    DP_REQUIRE((long long)B * Hq * ((Tq + cols - 1) / cols) < (1LL << 23) && (long long)B * Hkv * ((Tk + cols - 1) / cols) < (1LL << 23), "%s: too many blocks", fn);
    DP_REQUIRE(scale != 0.f && scale - scale == 0.f, "%s: the scale must be finite and not zero", fn);
    const int es = dtype == 0 ? 4 : 2;
    if (!dp_attn_lse_tensor(fn, "q", q, strides, es, B, Tq, Hq, false, &a->q) || !dp_attn_lse_tensor(fn, "k", k, strides + 3, es, B, Tk, Hkv, false, &a->k) ||
        !dp_attn_lse_tensor(fn, "v", v, strides + 6, es, B, Tk, Hkv, false, &a->v))
        return 1;
    a->q_lens = q_lens;
    a->kv_lens = kv_lens;
    a->B = B; a->Tq = Tq; a->Tk = Tk; a->Hq = Hq; a->Hkv = Hkv; a->D = D;
    a->Tqp = (Tq + 127) / 128 * 128;
    a->splits = 1;
    a->split_rows = 1 << 30;
    a->scale = scale;
    a->causal = causal != 0;
    a->xcd_map = dp_tune(DP_T_XCD_MAP) != 0;
    return 0;
}

extern "C" long long dp_attention_lse_workspace(int dtype, int B, int Tq, int Tk, int Hq, int Hkv, int D) {
    if (dtype < 0 || dtype > 2 || B <= 0 || Tq <= 0 || Tk <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || D <= 0 || D > 256) return 0;
    const al::QPlan pl = al::q_plan(dtype, B, Tq, Tk, Hq, Hkv, al::padded_dim(D));
    return pl.splits > 1 ? (long long)pl.splits * B * Hq * Tq * (D + 1) * 4 : 0;
}

extern "C" int dp_attention_lse(const void* q, const void* k, const void* v, const long long* strides, int dtype, int B, int Tq, int Tk, int Hq, int Hkv,
                                int D, const int* q_lens, const int* kv_lens, float scale, int causal, void* out, float* lse, void* work,
                                long long work_bytes, void* stream) {
    const char* fn = "dp_attention_lse";
    al::Args a{};
    if (int rc = dp_attn_lse_common(fn, q, k, v, strides, dtype, B, Tq, Tk, Hq, Hkv, D, q_lens, kv_lens, scale, causal, &a)) return rc;
    DP_REQUIRE(lse, "%s: lse missing", fn);
    if (!dp_attn_lse_tensor(fn, "out", out, strides + 9, dtype == 0 ? 4 : 2, B, Tq, Hq, true, &a.w0)) return 1;
    const long long need = dp_attention_lse_workspace(dtype, B, Tq, Tk, Hq, Hkv, D);
    DP_REQUIRE(need == 0 || (work && dp_aligned16(work) && work_bytes >= need), "%s: workspace of %lld bytes needed (got %lld)", fn, need, work_bytes);
    const long long row = (long long)D * (dtype == 0 ? 4 : 2);
    const dp::Region written[] = {dp_attn_lse_region("out", a.w0, B, Tq, Hq, row), dp::flat("lse", lse, 4LL * B * Hq * Tq), dp::flat("work", work, need)},
                     read[] = {dp_attn_lse_region("q", a.q, B, Tq, Hq, row), dp_attn_lse_region("k", a.k, B, Tk, Hkv, row), dp_attn_lse_region("v", a.v, B, Tk, Hkv, row),
                               dp::flat("q_lens", q_lens, 4LL * B), dp::flat("kv_lens", kv_lens, 4LL * B)};
    if (dp::check_apart(fn, written, 3, read, 5)) return 1;
    a.lse = lse;
    a.part0 = static_cast<float*>(work);
    a.part_lse = need ? a.part0 + need / 4 / (D + 1) * D : nullptr;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == 0) launch_fwd<0>(a, s);
    else if (dtype == 1) launch_fwd<1>(a, s);
    else launch_fwd<2>(a, s);
    DP_LAUNCH_CHECK("attn_lse_fwd");
    return 0;
}
