// Shared pieces of the attention kernels that work from a log-sum-exp (attention_lse.hip, attention_lse_bwd.hip).
//
// Every product of the three passes has one STREAMED operand (row tiles that come through LDS) and one operand that a wave keeps:
//     forward   S^T = K Q^T,   O^T  += V^T P^T           streamed: K, V    kept: 32 queries (16 in fp32)
//     dQ        S^T, dP^T = V dO^T,  dQ^T += K^T dS^T    streamed: K, V    kept: queries
//     dK, dV    S = Q K^T, dP = dO V^T,  dV^T += dO^T P,  dK^T += Q^T dS   streamed: Q, dO   kept: keys
// i.e. a score tile is always [streamed rows] x [kept columns]: in the accumulator layout a lane owns ONE kept column and a few streamed
// rows, and its registers - rounded to the operand type - are the B operand of the second product as they stand (no shuffle, no LDS).  The
// A operand of the second product is the transposed view of the streamed tile: 16-bit types read it with the transposing LDS read
// (ds_read_b64_tr_b16: a group of 16 lanes gets the 4 x 16 block that its addresses name, transposed), fp32 with four plain reads.
//
// fp32 runs on the fp32 matrix instruction (16 x 16 x 4): full fp32 products, no splitting, no range limits.
#pragma once
#include "dp_common.h"
#include "dp_region.h"
#include "dp_tune.h"

namespace al {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

// The masked and the unmasked form of a tile are two instances of its whole body: a branch BETWEEN a matrix instruction and the first read of
// its result is to be avoided (where both arms lead from the instruction to the read, the compiler counts the wait along one of them only).
struct yes { static constexpr bool value = true; };
struct no { static constexpr bool value = false; };

// the end of such a body: its last results are settled before any branch (12 wait states at most, with the branch and what follows it)
__device__ __forceinline__ void settle() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 9");
    __builtin_amdgcn_sched_barrier(0);
}

// at least `n` waves per SIMD: with 2 the registers of a wave end at 256 and the matrix instructions take their accumulators from the ordinary
// ones (with one wave they move through the accumulation registers and score tiles are copied).  Forms whose waves share columns miss that from 96 channels on: their
// stages fill 98 KB of LDS and more, one workgroup to a CU, and the compiler then spreads over the accumulation registers too (28 to 123 of them).
#define AL_WAVES(n) __attribute__((amdgpu_waves_per_eu(n)))

constexpr float LOG2E = 1.44269504088896341f;

// DT: element type of q, k, v, out and the gradients, and the shape of a score tile
//   0 fp32, 1 fp16, 2 bf16; 3, 4: fp16, bf16 with 16 columns (above 128 channels: half the registers for the kept operand and the accumulators)
//   TILE columns of a tile, G lane groups of TILE lanes; an accumulator holds TILE rows in NR registers:
//   register r of lane l is row (r & 3) + 4 G (r >> 2) + 4 (l / TILE), column l % TILE; a score tile is SUB of them, ROWS = SUB TILE rows.
//   KSTEP channels per step of the first product, KROWS rows per step of the second.
//   PSHIFT: the backward pass forms 2^PSHIFT P (an addend of the exponent, free) - see attention_lse_bwd.hip.
template <int DT> struct Tr;
struct Half {
    typedef _Float16 E;
    typedef f16x8 Frag;
    typedef f16x4 E4;
    static constexpr int ES = 2, PSHIFT = 6;
};
struct Bf {
    typedef __bf16 E;
    typedef bf16x8 Frag;
    typedef bf16x4 E4;
    static constexpr int ES = 2, PSHIFT = 0;
};
struct Wide {
    typedef f32x16 Acc;
    static constexpr int TILE = 32, G = 2, NR = 16, SUB = 1, ROWS = 32, KSTEP = 16, KROWS = 16;
};
struct Narrow {
    typedef f32x4 Acc;
    static constexpr int TILE = 16, G = 4, NR = 4, SUB = 2, ROWS = 32, KSTEP = 32, KROWS = 32;
};
template <> struct Tr<1> : Half, Wide {
    static __device__ __forceinline__ Acc mma(Frag a, Frag b, Acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Tr<2> : Bf, Wide {
    static __device__ __forceinline__ Acc mma(Frag a, Frag b, Acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Tr<3> : Half, Narrow {
    static __device__ __forceinline__ Acc mma(Frag a, Frag b, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Tr<4> : Bf, Narrow {
    static __device__ __forceinline__ Acc mma(Frag a, Frag b, Acc c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Tr<0> {
    typedef float E;
    typedef f32x4 Frag;
    typedef f32x4 E4;
    typedef f32x4 Acc;
    static constexpr int TILE = 16, G = 4, NR = 4, SUB = 1, ROWS = 16, KSTEP = 16, KROWS = 16, ES = 4, PSHIFT = 0;
    static __device__ __forceinline__ Acc mma(Frag a, Frag b, Acc c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};
// the shape of a type at a (padded) head dimension
constexpr int shape_of(int dtype, int DP) { return dtype && DP > 128 ? dtype + 2 : dtype; }
constexpr int tile_of(int dtype, int DP) { return dtype == 0 || DP > 128 ? 16 : 32; }

// a score tile: [ROWS streamed rows] x [TILE kept columns]
template <int DT> struct Score {
    using T = Tr<DT>;
    static constexpr int N = T::SUB * T::NR;
    typename T::Acc a[T::SUB];
    __device__ __forceinline__ float get(int r) const { return a[r / T::NR][r % T::NR]; }
    __device__ __forceinline__ void set(int r, float v) { a[r / T::NR][r % T::NR] = v; }
    __device__ __forceinline__ void fill(float v) {
#pragma unroll
        for (int r = 0; r < N; ++r) set(r, v);
    }
    // -> B operand of step kk of the second product
    __device__ __forceinline__ typename T::Frag pack(int kk) const {
        if constexpr (DT == 0) return a[0];
        else {
            typename T::Frag f;
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = (typename T::E)get(kk * 8 + j);
            return f;
        }
    }
};

// LDS image of a streamed tile: rows of RB bytes, the 16-byte slots of a row XOR-ed with bits of the row.  The 64 banks take 16 slots at a time, so
//   - a row read (one slot of 16 consecutive rows) wants 16 different places for the rows, and
//   - a transposing read (4 slots of 4 rows: consecutive ones for 16-bit types, 4 apart in fp32) wants the four rows in different groups of 4 slots.
// Rows of 256 bytes and more: the row bits that such a read runs over go to the upper two bits of the XOR, the other two to the lower ones.  Shorter rows
// already differ by their start; the remaining row bits go the same way.  (Rows of 128 bytes in fp32 keep a two-way conflict in the transposing read.)
template <int RB, int ES> struct Lds {
    static constexpr int SLOTS = RB / 16;
    static __device__ __forceinline__ int swz(int row) {
        if constexpr (SLOTS % 16 == 0) return ES == 4 ? row & 15 : ((row & 3) << 2) | ((row >> 1) & 2) | ((row >> 3) & 1);
        else if constexpr (SLOTS % 8 == 0) return ES == 4 ? (row >> 1) & 7 : ((row & 2) << 1) | ((row >> 2) & 3);
        else return (row >> 2) & 3;
    }
    static __device__ __forceinline__ int at(int row, int slot) { return row * RB + ((slot ^ swz(row)) << 4); }
};

// A operand, rows as they stand: row = lane % TILE, 16 bytes of step ks
template <int DT, int RB>
__device__ __forceinline__ typename Tr<DT>::Frag ld_row(const char* tile, int lane, int ks) {
    using T = Tr<DT>;
    return *reinterpret_cast<const typename T::Frag*>(tile + Lds<RB, T::ES>::at(lane & (T::TILE - 1), ks * T::G + lane / T::TILE));
}

// the first product, one step: score += [streamed rows] x [kept columns]
template <int DT, int RB>
__device__ __forceinline__ void mma_rows(const char* tile, int lane, int ks, typename Tr<DT>::Frag kept, Score<DT>& s) {
    using T = Tr<DT>;
#pragma unroll
    for (int i = 0; i < T::SUB; ++i) s.a[i] = T::mma(ld_row<DT, RB>(tile + i * T::TILE * RB, lane, ks), kept, s.a[i]);
}

// A operand, transposed: row = d of block dt, k = the KROWS streamed rows of step kk in the accumulator's order
template <int DT, int RB>
__device__ __forceinline__ typename Tr<DT>::Frag ld_tr(const char* tile, int lane, int kk, int dt) {
    using T = Tr<DT>;
    const int g = lane / T::TILE;
    typename T::Frag f;
    if constexpr (DT == 0) {
        const int byte = (dt * 16 + (lane & 15)) * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = *reinterpret_cast<const float*>(tile + Lds<RB, T::ES>::at(4 * g + j, byte >> 4) + (byte & 12));
    } else {
        const int i = lane & 15, byte = (dt * T::TILE + (lane & (T::TILE - 16)) + 4 * (i & 3)) * 2;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int row = kk * 16 + half * 4 * T::G + 4 * g + (i >> 2);
            const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(tile + Lds<RB, T::ES>::at(row, byte >> 4) + (byte & 8)));
            const typename T::E4 e = __builtin_bit_cast(typename T::E4, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) f[half * 4 + j] = e[j];
        }
    }
    return f;
}

#define AL_GLDS(src, dst, bytes)                                                               \
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src),     \
                                     (__attribute__((address_space(3))) void*)(dst), bytes, 0, 0)

// Streams BM rows of two matrices into LDS (asynchronous copies, 1 KB per wave and instruction): a uniform base that walks down the rows and 32-bit
// offsets per lane.  In the last tile, rows behind the last one are read from the last one, and slots behind the head dimension always from its last
// slot: the copies stay inside the tensors and bring in finite values, which the masks (rows) and the zeroed kept operand (slots) take out again.
template <int RB, int ES, int BM, int NW> struct Stream {
    static constexpr int TILE_BYTES = BM * RB, STAGE = 2 * TILE_BYTES, PIECES = STAGE / (1024 * NW);
    static_assert(TILE_BYTES % 1024 == 0 && STAGE % (1024 * NW) == 0, "a wave's copy lies in one matrix, and the waves share the copies evenly");
    using L = Lds<RB, ES>;
    const char *x0, *x1;                // row 0 of the two matrices
    long long s0, s1;                   // bytes per row (at most 2^24: BM rows stay within 32 bits)
    unsigned off[PIECES];
    int row_slots, wave, lane;

    __device__ __forceinline__ bool second(int i) const { return (i * NW + wave) * 1024 >= TILE_BYTES; }
    __device__ __forceinline__ int slot_id(int i) const { return (((i * NW + wave) * 1024 - (second(i) ? TILE_BYTES : 0)) >> 4) + lane; }
    __device__ __forceinline__ unsigned offset(int i, int rows) const {       // rows: how many there are from the tile's first on
        const int id = slot_id(i), row = id / L::SLOTS, slot = (id % L::SLOTS) ^ L::swz(row);
        return (unsigned)(row < rows ? row : rows - 1) * (unsigned)(second(i) ? s1 : s0) + (slot < row_slots ? slot : row_slots - 1) * 16;
    }
    __device__ __forceinline__ void init(const char* x0_, long long s0_, const char* x1_, long long s1_, int row_slots_, int wave_, int lane_) {
        x0 = x0_; x1 = x1_; s0 = s0_; s1 = s1_; row_slots = row_slots_; wave = wave_; lane = lane_;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) off[i] = offset(i, BM);
    }
    // rows r0 .. r0 + BM - 1 of n (r0 < n) of the matrices moved by o0 / o1 bytes
    __device__ __forceinline__ void issue(char* stage, int r0, int n, long long o0, long long o1) const {
        const char *b0 = x0 + o0 + r0 * s0, *b1 = x1 + o1 + r0 * s1;
        if (r0 + BM <= n) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) AL_GLDS((second(i) ? b1 : b0) + off[i], stage + (i * NW + wave) * 1024, 16);
        } else {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) AL_GLDS((second(i) ? b1 : b0) + offset(i, n - r0), stage + (i * NW + wave) * 1024, 16);
        }
    }
};

// workgroups are dealt to the 8 XCDs round-robin by blockIdx: XCD x gets a contiguous range of logical blocks, so that the blocks of one
// head - which stream the same rows - share an L2
__device__ __forceinline__ int logical_block(int xcd_map) {
    int bid = blockIdx.x;
    if (xcd_map) {
        const int x = bid & 7, per = gridDim.x >> 3, rem = gridDim.x & 7;
        bid = (x < rem ? x * (per + 1) : rem * (per + 1) + (x - rem) * per) + (bid >> 3);
    }
    return bid;
}

// keys that query `tok` of a sample with n queries and m keys sees: lengths and the causal diagonal alone decide which rows are empty (a sum of
// probabilities does not: it is NaN where a score is, and 0 where every score is -inf)
__device__ __forceinline__ int keys_seen(int tok, int n, int m, int causal) { return tok >= n ? 0 : causal ? min(m, tok + m - n + 1) : m; }

__device__ __forceinline__ int clamp_len(const int* lens, int b, int t) {
    if (!lens) return t;
    const int n = lens[b];
    return n < 0 ? 0 : (n > t ? t : n);
}

// reductions over the lane groups that share a column (lane ^ 32; fp32 tiles of 16 also lane ^ 16): register swaps, no LDS
template <int TILE, typename F> __device__ __forceinline__ float col_reduce(float v, F f) {
    const unsigned u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned lo = r[0], hi = r[1];
    v = f(__uint_as_float(lo), __uint_as_float(hi));
    if constexpr (TILE == 16) {
        const unsigned w = __float_as_uint(v);
        const auto q = __builtin_amdgcn_permlane16_swap(w, w, false, false);
        const unsigned a = q[0], b = q[1];
        v = f(__uint_as_float(a), __uint_as_float(b));
    }
    return v;
}
template <int TILE> __device__ __forceinline__ float col_sum(float v) {
    return col_reduce<TILE>(v, [](float a, float b) { return a + b; });
}
template <int TILE> __device__ __forceinline__ float col_max(float v) {
    return col_reduce<TILE>(v, [](float a, float b) { return fmaxf(a, b); });
}

// kept operand: 16 bytes per step of one row of a tensor, slots behind the head dimension zero
template <int DT, int KS>
__device__ __forceinline__ void ld_kept(typename Tr<DT>::Frag (&f)[KS], const char* rowp, int row_slots, int g) {
    using T = Tr<DT>;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int slot = ks * T::G + g;
        typename T::Frag v = {};
        if (slot < row_slots) v = *reinterpret_cast<const typename T::Frag*>(rowp + slot * 16);
        f[ks] = v;
    }
}

// An accumulator block [d][column] is stored in units of four consecutive d: unit u = block dt, registers 4 i .. 4 i + 3.
template <int DT, int ND> struct Units {
    using T = Tr<DT>;
    static constexpr int PER = T::NR / 4, N = ND * PER;
    static __device__ __forceinline__ int d(int u, int g) { return (u / PER) * T::TILE + (u % PER) * 4 * T::G + 4 * g; }
    static __device__ __forceinline__ f32x4 get(const typename T::Acc (&acc)[ND], int u) {
        const int r = (u % PER) * 4;
        return f32x4{acc[u / PER][r], acc[u / PER][r + 1], acc[u / PER][r + 2], acc[u / PER][r + 3]};
    }
};
template <int DT> __device__ __forceinline__ void st4(char* rowp, int d, f32x4 v) {
    typename Tr<DT>::E4 e;
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = (typename Tr<DT>::E)v[j];
    *reinterpret_cast<typename Tr<DT>::E4*>(rowp + (long long)d * Tr<DT>::ES) = e;
}
// ... or in fp32 whatever the type is
template <int DT> __device__ __forceinline__ void st4(char* rowp, int d, f32x4 v, int wide) {
    if (wide) *reinterpret_cast<f32x4*>(rowp + (long long)d * 4) = v;
    else st4<DT>(rowp, d, v);
}
// The waves that took different rows for the same columns (RS of them, rank rw) join their accumulators: every wave leaves its units in LDS and sums a
// share of them, in the order of the ranks.  sink(unit, sum) gets each unit once.  smem: Units::N KB per wave; a barrier must lie before the call.
template <int DT, int ND, int RS, typename Sink>
__device__ __forceinline__ void join_units(const typename Tr<DT>::Acc (&acc)[ND], float mul, char* smem, int wave, int rw, int lane, Sink sink) {
    using U = Units<DT, ND>;
    if constexpr (RS == 1) {
#pragma unroll
        for (int u = 0; u < U::N; ++u) sink(u, mul != 0.f ? U::get(acc, u) * mul : f32x4{});
    } else {
        f32x4* mine = reinterpret_cast<f32x4*>(smem) + (long long)wave * U::N * 64 + lane;
#pragma unroll
        for (int u = 0; u < U::N; ++u) mine[u * 64] = mul != 0.f ? U::get(acc, u) * mul : f32x4{};
        __syncthreads();
        const f32x4* first = reinterpret_cast<const f32x4*>(smem) + (long long)(wave - rw) * U::N * 64 + lane;
        for (int u = rw; u < U::N; u += RS) {
            f32x4 s = first[u * 64];
#pragma unroll
            for (int w = 1; w < RS; ++w) s += first[(w * U::N + u) * 64];
            sink(u, s);
        }
    }
}

// The kept columns of a wave, [d][column] in its accumulators, to rows of global memory: through LDS (smem: TILE rows of RB bytes of this wave's own), so that
// a row leaves in whole 16-byte pieces of consecutive lanes.  Straight from the accumulators a store instruction writes 8 bytes here and there of 32 rows.
// row_of(i) -> address of column i's row, or null.  A barrier must lie before the call (the region held streamed rows).
template <int DT, int ND, int RB, typename Row>
__device__ __forceinline__ void store_cols(const typename Tr<DT>::Acc (&acc)[ND], float mul, char* smem, int lane, int row_slots, Row row_of) {
    using T = Tr<DT>;
    using U = Units<DT, ND>;
    using L = Lds<RB, T::ES>;
    const int cl = lane & (T::TILE - 1), g = lane / T::TILE;
#pragma unroll
    for (int u = 0; u < U::N; ++u) {
        const f32x4 v = mul != 0.f ? U::get(acc, u) * mul : f32x4{};        // (0: a row that is to be zero whatever its accumulator holds)
        const int byte = U::d(u, g) * T::ES;
        typename T::E4 e;
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = (typename T::E)v[j];
        *reinterpret_cast<typename T::E4*>(smem + L::at(cl, byte >> 4) + (byte & 8)) = e;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    constexpr int ITEMS = T::TILE * L::SLOTS;
#pragma unroll
    for (int i = 0; i < ITEMS / 64; ++i) {
        const int id = i * 64 + lane, row = id / L::SLOTS, slot = id % L::SLOTS;
        const f32x4 v = *reinterpret_cast<const f32x4*>(smem + L::at(row, slot));
        char* to = row_of(row);
        if (to && slot < row_slots) *reinterpret_cast<f32x4*>(to + slot * 16) = v;
    }
}

// row of the tile that register r of a score holds (plus 4 g)
template <int DT> __device__ __forceinline__ constexpr int reg_row(int r) { return (r & 3) + 4 * Tr<DT>::G * (r >> 2); }

// [B, T, H, D] tensor: byte strides
struct Ten {
    const char* p;
    long long b, t, h;
};

struct Args {
    Ten q, k, v, o, dout;         // out / dout: backward only
    Ten w0, w1;                   // what the kernel writes: out (forward), dq, or dk and dv
    float* lse;                   // [B, Hq, Tq]
    float* rows;                  // backward: [2][B, Hq, Tqp] log2-domain log-sum-exp (+inf: no such row) and -delta
    int *lost_q, *lost_k;         // backward, fp16: did a wave of the dQ / dK launch lose an element to infinity?  Those of a key head side by side, lost_qn / lost_kn
    int lost_qn, lost_kn;
    float *part0, *part1;         // split launches: partial results, [split][kept row][D] (the order of kept rows: see Kept)
    float* part_lse;              // forward: [split][kept row]
    const int *q_lens, *kv_lens;
    int B, Tq, Tk, Hq, Hkv, D, Tqp;
    int wide;                     // backward: the gradients are fp32 whatever the operands are
    const float* sample_scale;    // wide: [B] factors of the samples' gradients, or null
    int packed;                   // 1: the queries of all heads of a group are the columns of one block (heads share their keys)
    int splits, split_rows;       // the streamed rows are cut into `splits` ranges of split_rows
    float scale;
    int causal, xcd_map;
    int stripes;                  // causal: see block_of
};

// Block i of the nblk blocks of one head, longest first where a causal mask makes their work differ.  Contiguous ranges of blocks go to one XCD, so the
// blocks of a head are dealt into `stripes` interleaved runs (as many as make every XCD's share a whole number of runs): each XCD gets long and short ones.
__device__ __forceinline__ int block_of(const Args& p, int i, int nblk, bool longest_last) {
    if (!p.causal) return i;
    const int q = nblk / p.stripes, r = nblk - q * p.stripes, cut = r * (q + 1);
    const int run = i < cut ? i / (q + 1) : r + (i - cut) / q, at = i < cut ? i % (q + 1) : (i - cut) % q;
    const int blk = at * p.stripes + run;
    return longest_last ? nblk - 1 - blk : blk;
}

// The kept queries of a workgroup.  Not packed: z = one query head, column = token.  Packed: z = one key head, column = head of the group * Tq + token.
struct Kept {
    int b, hk, h0, cols;
    __device__ __forceinline__ Kept(const Args& p, int z) {
        const int heads = p.packed ? p.Hkv : p.Hq;
        b = z / heads;
        const int h = z - b * heads, group = p.Hq / p.Hkv;
        hk = p.packed ? h : h / group;
        h0 = p.packed ? h * group : h;
        cols = p.packed ? group * p.Tq : p.Tq;
    }
    __device__ __forceinline__ void col(const Args& p, int c, int& h, int& t) const {
        const int i = p.packed ? c / p.Tq : 0;
        h = h0 + i;
        t = c - i * p.Tq;
    }
};

}  // namespace al

namespace al {

inline int padded_dim(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : 256; }

inline int stripes_of(long long heads) {
    int s = 8;
    while (s > 1 && heads % 2 == 0) {
        heads /= 2;
        s /= 2;
    }
    return s;
}

// How a launch covers the chip's 256 CUs.
//   rs:     waves of a workgroup that share one tile of columns and divide the streamed rows (1: every wave has a tile of its own).  Sharing makes more
//           workgroups with fewer rows each, but their stages fill the LDS: fewer of them fit a CU.
//   splits: ranges of the streamed rows that workgroups of their own take; a second launch joins their partial results.
// The cheapest by this estimate in microseconds: a round of workgroups costs 4 to begin and end and, per stage, the matrix time c of a wave as often as
// waves share its SIMD - at least twice, the latency of a stage that nothing hides - or the stage's own way into LDS, 0.7 and 60 GB/s per CU; a join costs 5 and the
// partial results' way to memory and back.
// A causal mask leaves the blocks half their rows on average, and the longest, begun first, bounds the launch.
// (One head of 256 channels, 4133 keys and queries, bf16, backward: 145 us, and 409 us without ranges; 1006 queries, 9 keys, fp32: 60 and 120 us.)
struct Cover {
    int rs, splits;
    long long blocks;             // workgroups of one range
};
inline Cover cover(int dtype, int DP, long long heads, long long cols, int rows, int times, int roles, double out_bytes, bool causal) {
    const int tile = tile_of(dtype, DP), srows = dtype == 0 ? 16 : 32, few = DP > 128 ? 2 : 4;
    const double c = (dtype == 0 ? 1.5 : 0.38 * tile / 32) * DP / 128;
    static const int cuts[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
    Cover best{1, 1, 0};
    double best_t = 1e30;
    for (int rs = 1; rs <= few; rs += few - 1) {
        const long long wide = 4 * tile / rs, blocks = heads * ((cols + wide - 1) / wide) * roles;
        const int resident = rs > 1 ? (DP <= 64 ? 2 : 1) : (DP <= 64 ? 3 : dtype == 0 && DP > 128 ? 1 : 2);
        const int stages = (rows + rs * srows - 1) / (rs * srows);
        const double slots = 256.0 * resident;
        for (int cut : cuts) {
            if (cut > stages) break;
            if (blocks * cut * 256 >= 1LL << 32) break;             // threads of a grid; the first candidate always fits (dp_attn_lse_common)
            const double wgs = (double)blocks * cut, per = (double)((stages + cut - 1) / cut) * times;
            const double share = wgs <= 256 ? 1 : wgs >= slots ? resident : (wgs + 255) / 256, copy = 0.7 + 2.0 * rs * srows * DP * (dtype == 0 ? 4 : 2) * share / 60e3;
            const double turn = (share < 2 ? 2 : share) * c > copy ? (share < 2 ? 2 : share) * c : copy;
            double t;
            if (causal) t = 4 + turn * (per / 2 * wgs / slots > per ? per / 2 * wgs / slots : per);
            else t = (wgs <= 2 * slots ? (double)(long long)((wgs + slots - 1) / slots) : wgs / slots + 0.4) * (4 + turn * per);       // (many rounds run into each other)
            if (cut > 1) t += 5 + cut * out_bytes * 2 / 4e6;
            if (t < best_t * 0.999) {
                best_t = t;
                best = Cover{rs, cut, blocks};
            }
        }
    }
    return best;
}

// The launches that keep queries (forward, dQ).  packed: heads that share their keys are columns of one block where all their queries fit two tiles
// (a key is then read once per group).
struct QPlan {
    int packed, rs, splits, split_rows;
    long long blocks;
};
inline QPlan q_plan(int dtype, int B, int Tq, int Tk, int Hq, int Hkv, int DP) {
    QPlan pl;
    const int group = Hq / Hkv;
    pl.packed = group > 1 && (long long)group * Tq <= 2 * tile_of(dtype, DP);
    const Cover c = cover(dtype, DP, (long long)B * (pl.packed ? Hkv : Hq), pl.packed ? (long long)group * Tq : Tq, Tk, 1, 1, 4.0 * B * Hq * Tq * DP, false);
    pl.rs = c.rs;
    pl.blocks = c.blocks;
    const int stage = pl.rs * (dtype == 0 ? 16 : 32), stages = (Tk + stage - 1) / stage;
    pl.split_rows = (stages + c.splits - 1) / c.splits * stage;
    pl.splits = (Tk + pl.split_rows - 1) / pl.split_rows;
    return pl;
}

// The launch that keeps keys (dK, dV).
// Above 64 channels the two gradients are formed by different workgroups, each of which recomputes the scores: a wave that holds both has 64 accumulators
// more and leaves no room for a second wave on its SIMD (8191 causal, heads of 128: 1434 us together, 1160 us apart; 128 heads of 256 channels x 256: 78.6 and
// 76.4 us; heads of 64, where both fit: 182 us together for 32 x 1024 x 8 heads, and 5 products instead of 4 apart).
constexpr bool two_roles(int DP) { return DP > 64; }
inline Cover k_plan(int dtype, int B, int Tq, int Tk, int Hq, int Hkv, int DP, int causal) {
    const int roles = two_roles(DP) ? 2 : 1;
    return cover(dtype, DP, (long long)B * Hkv, Tk, Tq, Hq / Hkv, roles, 8.0 * B * Hkv * Tk * DP, causal != 0);
}

}  // namespace al

// argument checks shared by the two entry points (attention_lse.hip): message and non-zero / false on a refusal
bool dp_attn_lse_tensor(const char* fn, const char* name, const void* ptr, const long long* st, int es, int B, int Tn, int H, bool written, al::Ten* t);
dp::Region dp_attn_lse_region(const char* name, const al::Ten& t, int B, int Tn, int H, long long row);
int dp_attn_lse_common(const char* fn, const void* q, const void* k, const void* v, const long long* strides, int dtype, int B, int Tq, int Tk, int Hq,
                       int Hkv, int D, const int* q_lens, const int* kv_lens, float scale, int causal, al::Args* a);
