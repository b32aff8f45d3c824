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
// ones (with more, they move through the accumulation registers and every score tile is copied)
#define AL_WAVES(n) __attribute__((amdgpu_waves_per_eu(n)))

constexpr float LOG2E = 1.44269504088896341f;

// DT: element type of q, k, v, out and the gradients (0 fp32, 1 fp16, 2 bf16).
//   TILE columns / rows of a score tile, G lane groups of TILE lanes, NR accumulator registers per tile.
//   Register r of lane l is row (r & 3) + 4 G (r >> 2) + 4 (l / TILE), column l % TILE.
//   PSHIFT: the backward pass forms 2^PSHIFT P (an addend of the exponent, free) - see attention_lse_bwd.hip.
template <int DT> struct Tr;
template <> struct Tr<1> {
    typedef _Float16 E;
    typedef f16x8 Frag;
    typedef f16x4 E4;
    typedef f32x16 Acc;
    static constexpr int TILE = 32, G = 2, NR = 16, ES = 2, PSHIFT = 6;
    static __device__ __forceinline__ Acc mma(Frag a, Frag b, Acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Tr<2> {
    typedef __bf16 E;
    typedef bf16x8 Frag;
    typedef bf16x4 E4;
    typedef f32x16 Acc;
    static constexpr int TILE = 32, G = 2, NR = 16, ES = 2, PSHIFT = 0;
    static __device__ __forceinline__ Acc mma(Frag a, Frag b, Acc c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Tr<0> {
    typedef float E;
    typedef f32x4 Frag;
    typedef f32x4 E4;
    typedef f32x4 Acc;
    static constexpr int TILE = 16, G = 4, NR = 4, ES = 4, PSHIFT = 0;
    static __device__ __forceinline__ Acc mma(Frag a, Frag b, Acc c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};

// registers 8 kk .. 8 kk + 7 (fp32: all four) of a score tile -> B operand of step kk of the second product
template <int DT>
__device__ __forceinline__ typename Tr<DT>::Frag pack(const typename Tr<DT>::Acc& p, int kk) {
    if constexpr (DT == 0) return p;
    else {
        typename Tr<DT>::Frag f;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = (typename Tr<DT>::E)p[kk * 8 + j];
        return f;
    }
}

// LDS image of a streamed tile: rows of RB bytes, the 16-byte slots of a row XOR-ed with the row so that the lanes of a read (one slot of
// many rows, or two slots of four rows in the transposing read) fall on different banks.  SWM + 1 divides the slots of a row.
template <int RB> struct Lds {
    static constexpr int SLOTS = RB / 16;
    static constexpr int POW2 = SLOTS & -SLOTS;
    static constexpr int SWM = (POW2 < 8 ? POW2 : 8) - 1;
    // rows of 64 bytes: four of them span the banks, so the XOR takes the row's upper bits
    static __device__ __forceinline__ int swz(int row) { return SLOTS == 4 ? (row >> 2) & SWM : row & SWM; }
    static __device__ __forceinline__ int at(int row, int slot) { return row * RB + ((slot ^ swz(row)) << 4); }
};

// A operand, rows as they stand: row = lane % TILE, 16 bytes of step ks
template <int DT, int RB>
__device__ __forceinline__ typename Tr<DT>::Frag ld_row(const char* tile, int lane, int ks) {
    using T = Tr<DT>;
    return *reinterpret_cast<const typename T::Frag*>(tile + Lds<RB>::at(lane & (T::TILE - 1), ks * T::G + lane / T::TILE));
}

// A operand, transposed: row = d of block dt, k = the 16 streamed rows of step kk in the accumulator's order
template <int DT, int RB>
__device__ __forceinline__ typename Tr<DT>::Frag ld_tr(const char* tile, int lane, int kk, int dt) {
    using T = Tr<DT>;
    const int g = lane / T::TILE;
    typename T::Frag f;
    if constexpr (DT == 0) {
        const int byte = (dt * 16 + (lane & 15)) * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = *reinterpret_cast<const float*>(tile + Lds<RB>::at(4 * g + j, byte >> 4) + (byte & 12));
    } else {
        const int i = lane & 15, byte = (dt * 32 + (lane & 16) + 4 * (i & 3)) * 2;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int row = kk * 16 + half * 8 + 4 * g + (i >> 2);
            const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(tile + Lds<RB>::at(row, byte >> 4) + (byte & 8)));
            const typename T::E4 e = __builtin_bit_cast(typename T::E4, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) f[half * 4 + j] = e[j];
        }
    }
    return f;
}

#define AL_GLDS(src, dst)                                                                      \
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src),     \
                                     (__attribute__((address_space(3))) void*)(dst), 16, 0, 0)

// Streams BM rows of two matrices into LDS (asynchronous copies, 1 KB per wave and instruction).  Rows behind the last one are read from
// the last one and slots behind the head dimension from its last slot: the copies stay inside the tensors and bring in finite values,
// which the masks (rows) and the zeroed kept operand (slots) take out again.
template <int RB, int BM, int NW> struct Stream {
    static constexpr int TILE_BYTES = BM * RB, STAGE = 2 * TILE_BYTES, PIECES = STAGE / (1024 * NW);
    static_assert(TILE_BYTES % 1024 == 0 && STAGE % (1024 * NW) == 0, "a wave's copy lies in one matrix, and the waves share the copies evenly");
    const char* base[PIECES];
    long long stride[PIECES];
    int row[PIECES];

    __device__ __forceinline__ void init(const char* x0, long long s0, const char* x1, long long s1, int row_slots, int wave, int lane) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int byte = (i * NW + wave) * 1024;
            const bool second = byte >= TILE_BYTES;
            const int id = ((byte - (second ? TILE_BYTES : 0)) >> 4) + lane;
            row[i] = id / Lds<RB>::SLOTS;
            const int slot = (id % Lds<RB>::SLOTS) ^ Lds<RB>::swz(row[i]);
            base[i] = (second ? x1 : x0) + (slot < row_slots ? slot : row_slots - 1) * 16;
            stride[i] = second ? s1 : s0;
        }
    }
    // rows r0 .. r0 + BM - 1 (n > 0 rows exist) of the matrices moved by o0 / o1 bytes
    __device__ __forceinline__ void issue(char* stage, int r0, int n, long long o0, long long o1, int wave) const {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const bool second = (i * NW + wave) * 1024 >= TILE_BYTES;
            const int r = r0 + row[i] < n ? r0 + row[i] : n - 1;
            AL_GLDS(base[i] + (second ? o1 : o0) + (long long)r * stride[i], stage + (i * NW + wave) * 1024);
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

__device__ __forceinline__ int clamp_len(const int* lens, int b, int t) {
    if (!lens) return t;
    const int n = lens[b];
    return n < 0 ? 0 : (n > t ? t : n);
}

// reduction over the lane groups that share a column
template <int TILE> __device__ __forceinline__ float col_sum(float v) {
#pragma unroll
    for (int o = TILE; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}
template <int TILE> __device__ __forceinline__ float col_max(float v) {
#pragma unroll
    for (int o = TILE; o < 64; o <<= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
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

// one kept column of an accumulator block [d][column], times `mul`, to a row of D elements
template <int DT, int ND>
__device__ __forceinline__ void st_col(const typename Tr<DT>::Acc (&acc)[ND], float mul, char* rowp, int D, int g) {
    using T = Tr<DT>;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int r = 0; r < T::NR; r += 4) {
            const int d = dt * T::TILE + r * T::G + 4 * g;
            typename T::E4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = (typename T::E)(acc[dt][r + j] * mul);
            if (d < D) *reinterpret_cast<typename T::E4*>(rowp + (long long)d * T::ES) = v;
        }
}

// row of the tile that register r holds (plus 4 g)
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
    float* ws;                    // backward: [2][B, Hq, Tqp] log2-domain log-sum-exp (+inf: no such row) and delta; forward: see there
    const int *q_lens, *kv_lens;
    int B, Tq, Tk, Hq, Hkv, D, Tqp;
    float scale;
    int causal, xcd_map;
};

}  // namespace al

// argument checks shared by the two entry points (attention_lse.hip): message and non-zero / false on a refusal
bool dp_attn_lse_tensor(const char* fn, const char* name, const void* ptr, const long long* st, int es, int B, int Tn, int H, bool written, al::Ten* t);
int dp_attn_lse_common(const char* fn, const void* q, const void* k, const void* v, const long long* strides, int dtype, int B, int Tq, int Tk, int Hq,
                       int Hkv, int D, const int* q_lens, const int* kv_lens, float scale, int causal, al::Args* a);
