// 8-bit integer products with a scale for each row of A (a token) and each row of W (an output channel):
//   C[m][n] = epi( sa[m] * sw[n] * sum_k A8[m][k] * W8[n][k] )
// The sums are exact 32-bit integers (k <= 131072), so neither the order of summation nor a split of K over waves
// changes a bit of the result; the only roundings are the integer's conversion to float32, the two scales' products,
// the epilogue and the output type.
//
// Weights are packed once (oasr_gemm_pack_w_i8): pieces of 16 rows x 64 k, 1 KiB each, ordered [row group][K slice],
// rows and k padded with zeros; a piece holds its 16-byte chunks in the order in which the lanes of a fragment take them
// (lane = (row lane & 15, chunk lane >> 4)), so a fragment is one contiguous KiB, in memory as in LDS.  A's rows stay
// row-major: a copy brings 16 rows x 64 k with four neighbouring lanes per row (whole 64-byte segments) and its source
// addresses put chunk c of row r at place c ^ (-(r >> 2) & 3) of the row, which keeps the fragment reads free of bank
// conflicts (with (r >> 2) & 3 they take twice as long: a read's groups of sixteen lanes are not lanes 0 .. 15).
// The weight fragment is the matrix instruction's A operand (v_mfma_i32_16x16x64_i8), so a lane ends up with four
// consecutive n of one row m: C[m = lane & 15][n = 4 (lane >> 4) + e].
#include "oasr_common.h"
#include "quant_i8.h"

namespace oasr {
namespace i8 {

constexpr int kSlice = 64;                 // k per slice: one MFMA step
constexpr int kPiece = 16 * kSlice;        // bytes of 16 rows of a slice
constexpr int64_t kMaxK = 131072;          // 128 * 127 * k < 2^31
constexpr int64_t kMaxGroups = (int64_t)7 << 20;        // of 512 threads, and an eighth more: a launch has fewer than 2^32 threads
constexpr int64_t kMaxRows = (int64_t)1 << 24;          // one of 256 threads each at most
constexpr int64_t kMaxWideTiles = (int64_t)1 << 30;     // walked by 256 work-groups, counted in 32 bits

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void gbl_void;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;

struct GemmArgs {
    const int8_t* a;        // [m][lda], zeros from k to round_up(k, 64)
    const int8_t* w;        // packed
    const float* scale_a;
    const float* scale_w;
    const float* bias;      // may be null
    const float* resid;     // residual epilogue only
    void* c;
    int64_t lda, ldr, ldc, m, n;
    int ks;                 // K slices
    int ng;                 // groups of 16 rows of W
    float alpha;
    int vec;                // c and resid rows start on 16-byte boundaries
};

__device__ __forceinline__ uint32_t cvt_pk_bf16(float a, float b) {
    typedef __attribute__((ext_vector_type(2))) __bf16 bf2;
    bf2 v;
    v[0] = (__bf16)a;
    v[1] = (__bf16)b;
    return __builtin_bit_cast(uint32_t, v);
}

__device__ __forceinline__ int turned(int row) { return (4 - (row >> 2)) & 3; }      // of a piece's rows 0 .. 15

// Division of numbers below 2^32 by one that the host knows: a product with floor((2^32 - 1) / d), which is at most one too small,
// and a correction (the division itself takes some hundred cycles, and a kernel's first addresses wait for it).
// (Tiles of the 256 x 256 form found this way: 12032 x 16384 x 4096 669 -> 658 us, 48128 x 2048 x 1024 gated 123.9 -> 121.5.)
struct Divisor {
    uint32_t d, inv;

    Divisor() = default;
    __host__ __device__ explicit Divisor(int64_t by) : d((uint32_t)by), inv(0xffffffffu / d) {}
    __device__ __forceinline__ void split(int v, int& quotient, int& rest) const {
        uint32_t q = __umulhi((uint32_t)v, inv), r = (uint32_t)v - q * d;
        if (r >= d) ++q, r -= d;
        quotient = (int)q;
        rest = (int)r;
    }
};

// Which tile a work-group computes.  Work-groups with equal blockIdx % 8 share an XCD and its L2 (used for locality only): each
// XCD gets a block of `rows` x `cols` tiles and walks it row by row, so that it fetches few rows of A and few of W.  rows = 0: the
// whole matrix row by row.  (Column by column instead, the encoder's step at batch 4 takes 4.80 ms, and 4.50 this way.)
struct TileMap {
    int tiles_m, tiles_n, across, rows;         // 2^across blocks side by side along m
    Divisor cols;

    __device__ __forceinline__ bool tile(int& tm, int& tn) const {
        if (rows == 0) {
            cols.split((int)blockIdx.x, tm, tn);
            return true;
        }
        cols.split((int)(blockIdx.x >> 3), tm, tn);
        const int xcd = blockIdx.x & 7;
        tm += (xcd & ((1 << across) - 1)) * rows;
        tn += (xcd >> across) * (int)cols.d;
        return tm < tiles_m && tn < tiles_n;
    }
};

#define OASR_I8_BARRIER()                     \
    do {                                      \
        asm volatile("" ::: "memory");        \
        __builtin_amdgcn_sched_barrier(0);    \
        __builtin_amdgcn_s_barrier();         \
        __builtin_amdgcn_sched_barrier(0);    \
        asm volatile("" ::: "memory");        \
    } while (0)

// Four consecutive entries of a per-column vector, guarded at n unless the tile lies inside the matrix.
struct __attribute__((packed, aligned(4))) f32x4_any {
    float v[4];
};

template <bool FULL>
__device__ __forceinline__ f32x4 load_cols(const float* __restrict__ p, int64_t col, int64_t n) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (FULL) {
        const f32x4_any t = *reinterpret_cast<const f32x4_any*>(p + col);
        v = (f32x4){t.v[0], t.v[1], t.v[2], t.v[3]};
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < n) v[e] = p[col + e];
    }
    return v;
}

// Of what lies in a tile, what exists and how it is aligned: everything, on 16-byte boundaries or on those of its elements
// (16 bytes move at once either way; the latter is 1 - 2 % slower where both would do), or the first `count` of each piece.
enum { kGuarded, kAnyStart, kAligned };
typedef f32x4 __attribute__((aligned(4))) f32x4_at4;
typedef u32x4 __attribute__((aligned(2))) u32x4_at2;

// Four consecutive float32 values of a row.
template <int FULL, bool ONCE>
__device__ __forceinline__ f32x4 load_f32(const float* p, int64_t count) {
    if (FULL == kAligned) {
        const f32x4* q = reinterpret_cast<const f32x4*>(p);
        return ONCE ? __builtin_nontemporal_load(q) : *q;
    }
    if (FULL == kAnyStart) {
        const f32x4_at4* q = reinterpret_cast<const f32x4_at4*>(p);
        return ONCE ? __builtin_nontemporal_load(q) : *q;
    }
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < count) v[e] = p[e];
    return v;
}
template <int FULL, bool ONCE>
__device__ __forceinline__ void store_f32(float* p, f32x4 v, int64_t count) {
    if (FULL == kAligned) {
        f32x4* q = reinterpret_cast<f32x4*>(p);
        if (ONCE) __builtin_nontemporal_store(v, q);
        else *q = v;
    } else if (FULL == kAnyStart) {
        f32x4_at4* q = reinterpret_cast<f32x4_at4*>(p);
        if (ONCE) __builtin_nontemporal_store(v, q);
        else *q = v;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < count) p[e] = v[e];
    }
}
// Eight bf16 values of a row.
template <int FULL, bool ONCE>
__device__ __forceinline__ void store_bf16x8(uint16_t* p, u32x4 v, int64_t count) {
    if (FULL == kAligned) {
        u32x4* q = reinterpret_cast<u32x4*>(p);
        if (ONCE) __builtin_nontemporal_store(v, q);
        else *q = v;
    } else if (FULL == kAnyStart) {
        u32x4_at2* q = reinterpret_cast<u32x4_at2*>(p);
        if (ONCE) __builtin_nontemporal_store(v, q);
        else *q = v;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < count) p[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
    }
}

// Orders a wave's own LDS writes before its reads of them (LDS operations of a wave execute in order).
#define OASR_I8_WAVE_LDS()                                              \
    do {                                                                \
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local"); \
        __builtin_amdgcn_wave_barrier();                                \
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local"); \
    } while (0)

// x sigmoid(x) and the sigmoid.  The factor of the exponential is a product of its own: folded into the columns' scales and
// biases it saves up to 1.5 %, but a pre-activation past 2.36e38 overflows there, and a finite one would give infinity or NaN.
constexpr float kLog2e = 1.44269504088896340736f;
__device__ __forceinline__ float sigmoid_of(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * x)); }
__device__ __forceinline__ float swish_of(float x) { return x * sigmoid_of(x); }

constexpr int kSlab = 4096;     // LDS per wave of the epilogue: 16 rows x 64 columns of float32

// The epilogue of a wave's MT x NT tiles of 16 x 16, the first at (m0, n0): scales, bias, activation or residual, stores.
// FULL: whether the whole of it lies inside the matrix, so that nothing is guarded (rows of 777 float32: 12.5 -> 11.5 us at
// 1237 x 777 x 1000, rows of 1023 bf16: 150 -> 106 us at 48128 x 1023 x 1024).
// The matrix instruction leaves four columns of one row in a lane and the 16 rows of a tile in neighbouring lanes, which
// stored as it is costs a memory request per lane (measured: 16 bytes per clock and CU).  Each group of 16 rows therefore
// crosses a wave-private slab, and leaves with the columns of a row in neighbouring lanes: whole 128-byte lines.  The slab's
// 16-byte chunks are permuted by the row so that neither side has bank conflicts.
// ONCE: outputs and residual rows go past the caches (large problems, whose outputs the caches would not keep: products that end
// in float32 gain 3 - 10 %, the others 2 %, the encoder's step is the same either way).
template <int EPI, int MT, int NT, bool ONCE = false>
struct Epilogue {
    static_assert(NT == 4 || NT == 2, "a wave owns 64 or 32 columns");
    static constexpr bool kResidual = EPI == OASR_EPI_RESIDUAL_F32, kFloat = kResidual || EPI == OASR_EPI_BIAS_F32,
                          kGlu = EPI == OASR_EPI_GLU_BF16;
    static constexpr int kOut = kGlu ? 8 * NT : 16 * NT;                     // output columns of the wave
    static constexpr int kChunks = kFloat ? kOut / 4 : kOut / 8;             // 16-byte chunks per row: 16, 8, 4 or 2
    static constexpr int kRows = 64 / kChunks < 16 ? 64 / kChunks : 16;      // rows per store instruction
    static constexpr int kStores = 16 / kRows;
    static constexpr int kShift = kChunks == 16 ? 0 : kChunks == 8 ? 1 : kChunks == 4 ? 2 : 3;   // rows per 256 bytes, log2

    f32x4 sw[NT], bv[NT], resid[kStores];     // resid: of the row group whose turn is next
    float sa[MT];

    static __device__ __forceinline__ int full(const GemmArgs& p, int64_t m0, int64_t n0) {
        return m0 + 16 * MT <= p.m && n0 + 16 * NT <= p.n ? (p.vec ? kAligned : kAnyStart) : kGuarded;
    }
    static __device__ __forceinline__ int64_t out_col(int64_t n0, int lane) { return (kGlu ? n0 / 2 : n0) + lane % kChunks * (kFloat ? 4 : 8); }

    template <int FULL>
    __device__ __forceinline__ void load_resid(const GemmArgs& p, int64_t m0, int64_t n0, int lane, int i) {
        const int64_t col = out_col(n0, lane);
#pragma unroll
        for (int q = 0; q < kStores; ++q) {
            const int64_t row = m0 + 16 * i + kRows * q + lane / kChunks;
            if (FULL || row < p.m) resid[q] = load_f32<FULL, ONCE>(p.resid + row * p.ldr + col, p.n - col);
        }
    }

    template <int FULL>
    __device__ __forceinline__ void load_form(const GemmArgs& p, int64_t m0, int64_t n0, int lane) {
        const int r = lane & 15, g = lane >> 4;
#pragma unroll
        for (int i = 0; i < MT; ++i) sa[i] = p.scale_a && (FULL || m0 + 16 * i + r < p.m) ? p.scale_a[m0 + 16 * i + r] : 0.f;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            sw[j] = load_cols<FULL != kGuarded>(p.scale_w, n0 + 16 * j + 4 * g, p.n);
            bv[j] = p.bias ? load_cols<FULL != kGuarded>(p.bias, n0 + 16 * j + 4 * g, p.n) : (f32x4){0.f, 0.f, 0.f, 0.f};
        }
        if (kResidual) load_resid<FULL>(p, m0, n0, lane, 0);
    }
    __device__ __forceinline__ void load(const GemmArgs& p, int64_t m0, int64_t n0, int lane) {
        const int f = full(p, m0, n0);
        if (f == kAligned) load_form<kAligned>(p, m0, n0, lane);
        else if (f == kAnyStart) load_form<kAnyStart>(p, m0, n0, lane);
        else load_form<kGuarded>(p, m0, n0, lane);
    }

    template <int FULL>
    __device__ __forceinline__ void finish_form(const GemmArgs& p, const i32x4 (&acc)[MT][NT], int64_t m0, int64_t n0, int lane, char* slab) {
        const int r = lane & 15, g = lane >> 4;
        const int out_row = lane / kChunks, out_chunk = lane % kChunks;   // in the storing role (lanes past 16 rows idle)
        const bool storing = kRows * kChunks == 64 || out_row < kRows;
        const int64_t col = out_col(n0, lane), left = (kGlu ? p.n / 2 : p.n) - col;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            f32x4 o[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)      // the weight's scale first: a token's may be as large as float32 goes
                    o[j][e] = fmaf((float)acc[i][j][e] * sw[j][e], sa[i], bv[j][e]);
            const int turn = (r >> kShift) & (kChunks - 1);
            if (kFloat) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    *reinterpret_cast<f32x4*>(slab + r * (16 * kChunks) + (((4 * j + g) ^ turn) << 4)) = o[j];
            } else {
#pragma unroll
                for (int j = 0; j < NT; j += kGlu ? 2 : 1) {
                    f32x4 v = o[j];
                    if (kGlu) {                  // tile 2 q = 16 value columns, tile 2 q + 1 = their gates (n % 32 == 0)
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] *= sigmoid_of(o[j + 1][e]);
                    }
                    if (EPI == OASR_EPI_BIAS_SWISH_BF16) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = swish_of(v[e]);
                    }
                    const int half = 4 * (kGlu ? j / 2 : j) + g;          // 8-byte half of a chunk
                    *reinterpret_cast<u32x2*>(slab + r * (16 * kChunks) + (((half >> 1) ^ turn) << 4) + (half & 1) * 8) =
                        (u32x2){cvt_pk_bf16(v[0], v[1]), cvt_pk_bf16(v[2], v[3])};
                }
            }
            OASR_I8_WAVE_LDS();
            u32x4 v[kStores];
#pragma unroll
            for (int q = 0; q < kStores; ++q) {
                const int sr = kRows * q + out_row;
                v[q] = (u32x4){0, 0, 0, 0};
                if (storing) v[q] = *reinterpret_cast<const u32x4*>(slab + sr * (16 * kChunks) + ((out_chunk ^ ((sr >> kShift) & (kChunks - 1))) << 4));
                if (kResidual) {
                    f32x4 f = __builtin_bit_cast(f32x4, v[q]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) f[e] = fmaf(p.alpha, f[e], resid[q][e]);
                    v[q] = __builtin_bit_cast(u32x4, f);
                }
            }
            OASR_I8_WAVE_LDS();
            if (kResidual && i + 1 < MT) load_resid<FULL>(p, m0, n0, lane, i + 1);      // requested before this row group's stores
#pragma unroll
            for (int q = 0; q < kStores; ++q) {
                const int64_t row = m0 + 16 * i + kRows * q + out_row;
                if (!storing || !(FULL || row < p.m)) continue;
                if (kFloat) store_f32<FULL, ONCE>(reinterpret_cast<float*>(p.c) + row * p.ldc + col, __builtin_bit_cast(f32x4, v[q]), left);
                else store_bf16x8<FULL, ONCE>(reinterpret_cast<uint16_t*>(p.c) + row * p.ldc + col, v[q], left);
            }
        }
    }
    __device__ __forceinline__ void finish(const GemmArgs& p, const i32x4 (&acc)[MT][NT], int64_t m0, int64_t n0, int lane, char* slab) {
        const int f = full(p, m0, n0);
        if (f == kAligned) finish_form<kAligned>(p, acc, m0, n0, lane, slab);
        else if (f == kAnyStart) finish_form<kAnyStart>(p, acc, m0, n0, lane, slab);
        else finish_form<kGuarded>(p, acc, m0, n0, lane, slab);
    }
    // both at once
    static __device__ __forceinline__ void run(const GemmArgs& p, const i32x4 (&acc)[MT][NT], int64_t m0, int64_t n0, int lane, char* slab) {
        Epilogue e;
        const int f = full(p, m0, n0);
        if (f == kAligned) {
            e.template load_form<kAligned>(p, m0, n0, lane);
            e.template finish_form<kAligned>(p, acc, m0, n0, lane, slab);
        } else if (f == kAnyStart) {
            e.template load_form<kAnyStart>(p, m0, n0, lane);
            e.template finish_form<kAnyStart>(p, acc, m0, n0, lane, slab);
        } else {
            e.template load_form<kGuarded>(p, m0, n0, lane);
            e.template finish_form<kGuarded>(p, acc, m0, n0, lane, slab);
        }
    }
};

// One work-group of WM x WN waves computes a tile of (16 MT WM) x (16 NT WN).  K runs through a ring of RING slices in
// LDS, filled by direct copies RING - 1 slices ahead, one barrier per slice: behind the barrier of slice p every wave
// has seen its own copies of slice p land and has read slice p - 1, so the slot of p - 1 may be filled again.
// Rows of A past m repeat row m - 1 and row groups of W past the last repeat the last: read, multiplied, never stored.
template <int EPI, int WM, int WN, int MT, int NT, int RING>
__global__ __launch_bounds__(64 * WM * WN) void gemm_i8_tile_kernel(const GemmArgs p, const TileMap map) {
    constexpr int kWaves = WM * WN, BM = 16 * MT * WM, BN = 16 * NT * WN;
    constexpr int kPieces = (BM + BN) / 16, kCopies = kPieces / kWaves, kSlot = kPieces * kPiece;
    static_assert(kPieces % kWaves == 0, "every wave issues the same number of copies");
    __shared__ __attribute__((aligned(1024))) char ring[RING * kSlot];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    int tm, tn;
    if (!map.tile(tm, tn)) return;           // the whole work-group
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;

    const char* src[kCopies];
    int step[kCopies];
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
        const int q = wave * kCopies + i;
        if (q < BM / 16) {
            int64_t row = m0 + 16 * q + (lane >> 2);
            row = row < p.m ? row : p.m - 1;
            src[i] = reinterpret_cast<const char*>(p.a) + row * p.lda + (((lane & 3) ^ turned(lane >> 2)) << 4);
            step[i] = kSlice;
        } else {
            int64_t grp = n0 / 16 + (q - BM / 16);
            grp = grp < p.ng ? grp : p.ng - 1;
            src[i] = reinterpret_cast<const char*>(p.w) + grp * p.ks * kPiece + lane * 16;
            step[i] = kPiece;
        }
    }
    auto copy_next = [&](int slot) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            __builtin_amdgcn_global_load_lds((gbl_void*)src[i], (lds_void*)(ring + slot * kSlot + (wave * kCopies + i) * kPiece), 16, 0, 0);
            src[i] += step[i];
        }
    };

    i32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = (i32x4){0, 0, 0, 0};
    const int fr = lane & 15, frag = fr * 64 + (((lane >> 4) ^ turned(fr)) << 4);

    for (int t = 0; t < RING - 1 && t < p.ks; ++t) copy_next(t);
    int slot = 0, fill = RING - 1;
    for (int t = 0; t < p.ks; ++t) {
        if (t + RING - 1 <= p.ks)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((RING - 2) * kCopies) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the last slices: fewer copies than the ring are in flight
        OASR_I8_BARRIER();
        if (t + RING - 1 < p.ks) {
            copy_next(fill);
            fill = fill + 1 == RING ? 0 : fill + 1;
        }
        const char* sa = ring + slot * kSlot + wm * MT * kPiece;
        const char* sw = ring + slot * kSlot + (BM / 16 + wn * NT) * kPiece;
        i32x4 wf[NT], xf[MT];
#pragma unroll
        for (int j = 0; j < NT; ++j) wf[j] = *reinterpret_cast<const i32x4*>(sw + j * kPiece + lane * 16);
#pragma unroll
        for (int i = 0; i < MT; ++i) xf[i] = *reinterpret_cast<const i32x4*>(sa + i * kPiece + frag);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j], xf[i], acc[i][j], 0, 0, 0);
        slot = slot + 1 == RING ? 0 : slot + 1;
    }
    static_assert(RING * kSlot >= kWaves * kSlab, "the slabs take the ring's place");
    __syncthreads();                         // every wave has read its last slice
    Epilogue<EPI, MT, NT>::run(p, acc, m0 + wm * MT * 16, n0 + wn * NT * 16, lane, ring + wave * kSlab);
}

// Large problems: 256 x 256 tiles, eight waves as two groups (the upper and the lower 128 rows) one barrier apart, so that
// one group reads fragments and issues copies while the other multiplies (32 MFMAs per slice); a wave owns 128 x 64.  The
// grid is one work-group per CU; each walks its tiles in one continuous pipeline, the next tile's first slices being in
// flight during the epilogue.  A ring of four slices of 64 k (16 KiB per operand), copied two slices ahead.
// Work-groups with equal blockIdx % 8 share an XCD (used for locality only): an XCD owns a contiguous range of row tiles and
// walks it in bands of four column tiles, so that a band's weights stay in that XCD's L2.  From 16 row tiles on the ranges are whole
// row tiles, so some XCDs have one more than others, and with few rounds of tiles that is a round more than an even split would
// take: 9216 x 1024 x 4096 has 144 tiles, 16 or 20 to an XCD of 18 work-groups, two rounds instead of one.
// The residual form takes all 256 registers and spills nine (40 bytes of scratch, outside the loop over K).
constexpr int kWide = 256, kWideRing = 4, kWideSlice = kWide * kSlice;

template <int EPI>
__global__ __launch_bounds__(512) void gemm_i8_wide_kernel(const GemmArgs p, int tiles_m, int tiles_n) {
    __shared__ __attribute__((aligned(1024))) char ring[2 * kWideRing * kWideSlice + 8 * kSlab];      // A slots, W slots, slabs
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 2, wn = wave & 3;

    const int xcd = blockIdx.x & 7, first = blockIdx.x >> 3, stride = gridDim.x >> 3;
    const int n_tiles = tiles_m * tiles_n;
    const bool banded = tiles_m >= 16;
    const int m_lo = (int)((int64_t)tiles_m * xcd / 8), m_cnt = (int)((int64_t)tiles_m * (xcd + 1) / 8) - m_lo;
    const int flat_lo = (int)((int64_t)n_tiles * xcd / 8);
    const int local = banded ? m_cnt * tiles_n : (int)((int64_t)n_tiles * (xcd + 1) / 8) - flat_lo;
    if (first >= local) return;
    const int mine = (local - first + stride - 1) / stride;
    const Divisor by_band(banded ? m_cnt * 4 : tiles_n), by_rest(max(tiles_n & 3, 1));
    auto tile_at = [&](int i, int& tm, int& tn) {
        const int l = first + i * stride;
        if (!banded) {
            by_band.split(flat_lo + l, tm, tn);
            return;
        }
        int band, in;
        by_band.split(l, band, in);
        if (4 * band + 4 <= tiles_n) {
            tm = in >> 2;
            tn = in & 3;
        } else {
            by_rest.split(in, tm, tn);
        }
        tm += m_lo;
        tn += 4 * band;
    };

    i32x4 acc[8][4];
    const int nph = p.ks, total = mine * nph;
    const int fr = lane & 15, frag = fr * 64 + (((lane >> 4) ^ turned(fr)) << 4);
    // Copies: wave w brings rows 32 w .. 32 w + 31 of both operands' slices, two pieces each.  Rows past the last repeat it.
    const uint32_t chunk = (uint32_t)(((lane & 3) ^ turned(lane >> 2)) << 4);
    const char *src_a, *src_w0, *src_w1;
    uint32_t off0, off1;
    int st_i = 0, st_t = 0;
    auto seek = [&](int i) {
        int tm, tn;
        tile_at(i, tm, tn);
        int64_t row = (int64_t)tm * kWide + wave * 32;
        row = row < p.m ? row : p.m - 1;
        const int left = (int)min(p.m - 1 - row, (int64_t)31);
        src_a = reinterpret_cast<const char*>(p.a) + row * p.lda;
        off0 = (uint32_t)min(lane >> 2, left) * (uint32_t)p.lda + chunk;
        off1 = (uint32_t)min(16 + (lane >> 2), left) * (uint32_t)p.lda + chunk;
        const int grp = tn * (kWide / 16) + wave * 2;
        src_w0 = reinterpret_cast<const char*>(p.w) + (int64_t)min(grp, p.ng - 1) * p.ks * kPiece;
        src_w1 = reinterpret_cast<const char*>(p.w) + (int64_t)min(grp + 1, p.ng - 1) * p.ks * kPiece;
    };
    auto copy_next = [&](int ph) {
        char* da = ring + (ph & 3) * kWideSlice + wave * 2 * kPiece;
        char* dw = da + kWideRing * kWideSlice;
        __builtin_amdgcn_global_load_lds((gbl_void*)(src_a + off0), (lds_void*)da, 16, 0, 0);
        __builtin_amdgcn_global_load_lds((gbl_void*)(src_a + off1), (lds_void*)(da + kPiece), 16, 0, 0);
        __builtin_amdgcn_global_load_lds((gbl_void*)(src_w0 + (uint32_t)lane * 16), (lds_void*)dw, 16, 0, 0);
        __builtin_amdgcn_global_load_lds((gbl_void*)(src_w1 + (uint32_t)lane * 16), (lds_void*)(dw + kPiece), 16, 0, 0);
        src_a += kSlice;
        src_w0 += kPiece;
        src_w1 += kPiece;
        if (++st_t == nph) {
            st_t = 0;
            if (++st_i < mine) seek(st_i);
        }
    };
    seek(0);
    copy_next(0);
    if (total > 1) {
        copy_next(1);
        asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    OASR_I8_BARRIER();
    if (wm == 1) OASR_I8_BARRIER();          // the second group runs one barrier behind

    int ph = 0;
    const i32x4 zero = {0, 0, 0, 0};
    for (int i = 0; i < mine; ++i) {
        int tm, tn;
        tile_at(i, tm, tn);
        for (int t = 0; t < nph; ++t, ++ph) {
            const char* sa = ring + (ph & 3) * kWideSlice + wm * 8 * kPiece + frag;
            const char* sw = ring + (kWideRing + (ph & 3)) * kWideSlice + wn * 4 * kPiece + lane * 16;
            i32x4 wf[4], xf[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) wf[j] = *reinterpret_cast<const i32x4*>(sw + j * kPiece);
#pragma unroll
            for (int ii = 0; ii < 8; ++ii) xf[ii] = *reinterpret_cast<const i32x4*>(sa + ii * kPiece);
            if (ph + 2 < total) {
                copy_next(ph + 2);
                asm volatile("s_waitcnt vmcnt(4)" ::: "memory");     // own pieces of slice ph + 1 have landed
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            OASR_I8_BARRIER();
            __builtin_amdgcn_s_setprio(1);
            if (t == 0) {                    // a tile's first slice accumulates onto zero: no clearing pass
#pragma unroll
                for (int ii = 0; ii < 8; ++ii)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[ii][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j], xf[ii], zero, 0, 0, 0);
            } else {
#pragma unroll
                for (int ii = 0; ii < 8; ++ii)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[ii][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j], xf[ii], acc[ii][j], 0, 0, 0);
            }
            __builtin_amdgcn_s_setprio(0);
            // the second group holds the barrier that ends a tile's last slice until its epilogue is done, so that the two
            // groups' epilogues overlap
            if (!(wm == 1 && t == nph - 1)) OASR_I8_BARRIER();
        }
        // (loading the scales during the last slice instead costs more in the loop than it saves here)
        Epilogue<EPI, 8, 4, true>::run(p, acc, (int64_t)tm * kWide + wm * 128, (int64_t)tn * kWide + wn * 64, lane,
                                 ring + 2 * kWideRing * kWideSlice + wave * kSlab);
        if (wm == 1) OASR_I8_BARRIER();
    }
    if (wm == 0) OASR_I8_BARRIER();          // the same number of barriers in both groups
}

// Problems with few tiles (single tokens, one utterance): a work-group of eight waves owns 16 MT x 64 outputs, and the
// waves split K among them, slice by slice in turn.  Exact sums make the split free of consequences, and it is what keeps
// enough bytes in flight: no wave waits for another before the end.  A wave brings its A rows through an LDS ring of its own
// (DEPTH slices, no barriers) and its weight fragments straight to registers, both requested DEPTH - 1 slices ahead: up to
// 200 KiB per CU, where the ring shared by the waves of a tile holds 48 (1504 x 1024 x 4096: 15.2 against 25.4 us).  They are not on
// their way all the time: the weights are ordinary loads behind a condition, so at the loop's start the compiler waits for all that is
// in flight, the slice just requested included, once in DEPTH slices (matrix pipe busy 12 % there, waits 40 %).  At the end the partial
// sums cross LDS, and every wave finishes its share of the 16 x 32 outputs.
template <int MT>
struct SplitShape {
    static constexpr int kDepth = MT >= 8 ? 2 : 3;
    static constexpr int kRingBytes = kDepth * MT * kPiece;                // per wave
    static constexpr int kPasses = MT > 4 ? 2 : 1;                         // partial sums of 64 or, twice, of 32 columns
    static constexpr int kCols = 4 / kPasses;                              // column tiles per pass
    static constexpr int kUnits = MT * kCols / 2;                          // 16 x 32 outputs per pass, one per wave
    static constexpr int kSumBytes = 8 * MT * kCols * 1024;
    static constexpr int kLds = 8 * kRingBytes > kSumBytes + 8 * 2048 ? 8 * kRingBytes : kSumBytes + 8 * 2048;
};

template <int EPI, int MT>
__global__ __launch_bounds__(512) void gemm_i8_split_kernel(const GemmArgs p, const TileMap map) {
    typedef SplitShape<MT> Shape;
    constexpr int D = Shape::kDepth;
    __shared__ __attribute__((aligned(1024))) char lds[Shape::kLds];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tm, tn;
    if (!map.tile(tm, tn)) return;           // the whole work-group
    const int64_t m0 = (int64_t)tm * (16 * MT), n0 = (int64_t)tn * 64;

    char* const ring = lds + wave * Shape::kRingBytes;
    const char* src_a[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        int64_t row = m0 + 16 * i + (lane >> 2);
        row = row < p.m ? row : p.m - 1;
        src_a[i] = reinterpret_cast<const char*>(p.a) + row * p.lda + (((lane & 3) ^ turned(lane >> 2)) << 4) + wave * kSlice;
    }
    const char* src_w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        int64_t grp = n0 / 16 + j;
        grp = grp < p.ng ? grp : p.ng - 1;
        src_w[j] = reinterpret_cast<const char*>(p.w) + (grp * p.ks + wave) * kPiece + lane * 16;
    }
    i32x4 acc[MT][4], wf[D][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = (i32x4){0, 0, 0, 0};
    const int count = p.ks > wave ? (p.ks - wave + 7) / 8 : 0;            // this wave's slices
    auto request = [&](int slot, i32x4 (&w)[4]) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            __builtin_amdgcn_global_load_lds((gbl_void*)src_a[i], (lds_void*)(ring + (slot * MT + i) * kPiece), 16, 0, 0);
            src_a[i] += 8 * kSlice;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            w[j] = *reinterpret_cast<const i32x4*>(src_w[j]);
            src_w[j] += 8 * kPiece;
        }
    };
    const int fr = lane & 15, frag = fr * 64 + (((lane >> 4) ^ turned(fr)) << 4);
#pragma unroll
    for (int d = 0; d < D - 1; ++d)
        if (d < count) request(d, wf[d]);
    // the scales (and residual rows) of the 16 x 32 outputs that this wave will finish come along with the first slices
    const int unit_row = Shape::kCols == 4 ? (wave >> 1) % MT : wave % MT, unit_col = Shape::kCols == 4 ? 2 * (wave & 1) : 0;
    const int64_t mu = m0 + 16 * unit_row, nu = n0 + 16 * unit_col;
    Epilogue<EPI, 1, 2> out;
    out.load(p, mu, nu, lane);
    for (int t = 0; t < count; t += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (t + d >= count) break;
            // the slot of slice t + d - 1 is free: its fragments went into the products above
            if (t + d + D - 1 < count) {
                request((d + D - 1) % D, wf[(d + D - 1) % D]);
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"((D - 1) * (MT + 4)) : "memory");
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            i32x4 xf[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) xf[i] = *reinterpret_cast<const i32x4*>(ring + (d * MT + i) * kPiece + frag);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[d][j], xf[i], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // partial sums: [wave][row tile][column tile of the pass][lane]
#pragma unroll
    for (int pass = 0; pass < Shape::kPasses; ++pass) {
        __syncthreads();                     // the rings, or the pass before, have been read
        if (pass) out.load(p, mu, nu + 32 * pass, lane);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < Shape::kCols; ++j)
                *reinterpret_cast<i32x4*>(lds + ((wave * MT + i) * Shape::kCols + j) * 1024 + lane * 16) = acc[i][pass * Shape::kCols + j];
        __syncthreads();
        if (wave < Shape::kUnits) {
            i32x4 sum[1][2] = {};
#pragma unroll
            for (int w = 0; w < 8; ++w)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    sum[0][j] += *reinterpret_cast<const i32x4*>(lds + ((w * MT + unit_row) * Shape::kCols + unit_col + j) * 1024 + lane * 16);
            out.finish(p, sum, mu, nu + 32 * pass, lane, lds + Shape::kSumBytes + wave * 2048);
        }
    }
}

// Per-row quantisation of bf16 rows.  One wavefront per row with the row in registers (k <= 512 NV: NV loads of 16
// bytes per lane, all issued before the first use), or, for longer rows, in two sweeps of which the second reads from
// cache.  HBM-bound: 2 bytes in, 1 byte out per element.  Row starts need no alignment; the codes' rows are whole
// 64-byte slices, zero from k on.
// ONCE: read past the caches, for activations larger than they are (48128 x 4096 with its product 324 -> 315 us, since more
// of the codes stay in the memory-side cache; at 12 MB it costs 4 %).
template <bool ONCE = false>
__device__ __forceinline__ u32x4 load_row8(const uint16_t* __restrict__ xr, int64_t c, int64_t k) {
    typedef u32x4 __attribute__((aligned(2))) any;
    u32x4 v = {0, 0, 0, 0};
    if (c + 8 <= k) {
        const any* p = reinterpret_cast<const any*>(xr + c);
        v = ONCE ? __builtin_nontemporal_load(p) : *p;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < k) v[e >> 1] |= (uint32_t)xr[c + e] << (16 * (e & 1));
    }
    return v;
}

__device__ __forceinline__ uint32_t amax8(u32x4 v, uint32_t amax) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const uint32_t lo = (v[q] << 16) & 0x7fffffffu, hi = v[q] & 0x7fff0000u;
        amax = amax > lo ? amax : lo;
        amax = amax > hi ? amax : hi;
    }
    return amax;
}

__device__ __forceinline__ u32x2 codes8(u32x4 v, const RowScale& s) {
    uint32_t c[8];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        c[2 * q] = code_of_bf16(__uint_as_float(v[q] << 16), s);
        c[2 * q + 1] = code_of_bf16(__uint_as_float(v[q] & 0xffff0000u), s);
    }
    return (u32x2){pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7])};
}

template <int NV, bool ONCE>
__global__ __launch_bounds__(256) void quant_i8_rows_kernel(const uint16_t* __restrict__ x, int64_t ldx, int64_t rows,
                                                            int64_t k, int8_t* __restrict__ y, int64_t ldy,
                                                            float* __restrict__ scale) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const uint16_t* xr = x + row * ldx;
    int8_t* yr = y + row * ldy;
    const int64_t kp = (k + kSlice - 1) / kSlice * kSlice;
    uint32_t amax = 0;
    u32x4 v[NV > 0 ? NV : 1];
    if (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = load_row8<ONCE>(xr, 8 * lane + 512 * i, k);
#pragma unroll
        for (int i = 0; i < NV; ++i) amax = amax8(v[i], amax);
    } else {
        for (int64_t c = 8 * lane; c < k; c += 512) amax = amax8(load_row8(xr, c, k), amax);
    }
    const RowScale s = row_scale(wave_umax(amax));
    if (lane == 0) scale[row] = s.scale;
    if (NV > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = 8 * lane + 512 * i;
            if (c < kp) *reinterpret_cast<u32x2*>(yr + c) = codes8(v[i], s);
        }
    } else {
        for (int64_t c = 8 * lane; c < kp; c += 512) *reinterpret_cast<u32x2*>(yr + c) = codes8(load_row8(xr, c, k), s);
    }
}

// A few tokens: quantisation and product in one launch.  Every work-group (16 MT rows x 32 columns, eight waves that split K)
// quantises its rows itself - they are a few KiB that many of them read from L2 - into LDS, while its first weight slices are
// on their way; the codes and scales are bit for bit those of the quantiser.  Bound by the weights' way from HBM: 16384 x 4096 at
// one row (64 MiB) 12.8 us; small ones by latency (a second launch would cost more than the work).
constexpr int kFewColumns = 32;              // 64 at a time are 5 - 25 % slower at every size tried (1 x 4096 x 4096: 8.4 against 10.2 us)
constexpr int kFewDepth = 6;                 // slices requested ahead (4: up to 4 % slower; 8: faster on short n, slower on long)
                                             // (the first and last of six wait for all that is in flight, as above)

template <int MT>
struct FewShape {
    static constexpr int kCodes = 16384 * MT;                      // rows * k (rounded up to 64) of a work-group at most
    static constexpr int kItems = kCodes / 8 / 512;                // per thread, eight values each
    static constexpr int kCodeBytes = kCodes + 16 * 16 * MT, kSums = 8 * MT * 2 * 1024, kAll = kSums + MT * 2048;
    static constexpr int kLds = kAll > kCodeBytes ? kAll : kCodeBytes;
};

template <int EPI, int MT>
__global__ __launch_bounds__(512) void linear_i8_few_kernel(const GemmArgs p, const uint16_t* __restrict__ x, int64_t ldx, int k,
                                                            int tiles_m) {
    typedef FewShape<MT> Shape;
    constexpr int D = kFewDepth, CT = kFewColumns / 16;
    __shared__ __attribute__((aligned(1024))) char lds[Shape::kLds];
    __shared__ uint32_t row_amax[16 * MT];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (tid < 16 * MT) row_amax[tid] = 0;
    const int64_t m0 = (int64_t)(blockIdx.x % tiles_m) * (16 * MT), n0 = (int64_t)(blockIdx.x / tiles_m) * kFewColumns;
    const int rows = (int)min((int64_t)(16 * MT), p.m - m0), kp = p.ks * kSlice;
    const int pitch = kp + 16;               // 16 bytes apart: the rows' fragments in other banks
    x += m0 * ldx;

    const char* src_w[CT];
#pragma unroll
    for (int j = 0; j < CT; ++j) {
        int64_t grp = n0 / 16 + j;
        grp = grp < p.ng ? grp : p.ng - 1;
        src_w[j] = reinterpret_cast<const char*>(p.w) + (grp * p.ks + wave) * kPiece + lane * 16;
    }
    const int count = p.ks > wave ? (p.ks - wave + 7) / 8 : 0;
    i32x4 wf[D][CT];
    auto request = [&](i32x4 (&w)[CT]) {
#pragma unroll
        for (int j = 0; j < CT; ++j) {
            w[j] = *reinterpret_cast<const i32x4*>(src_w[j]);
            src_w[j] += 8 * kPiece;
        }
    };
#pragma unroll
    for (int d = 0; d < D - 1; ++d)
        if (d < count) request(wf[d]);
    const int64_t mu = m0 + 16 * (wave % MT);
    Epilogue<EPI, 1, 2> out;
    if (wave < MT) out.load(p, mu, n0, lane);

    // the rows, eight values to an item, all requested at once; a row is a multiple of eight items, so eight neighbouring lanes
    // always share one
    const int per_row = kp / 8, items = rows * per_row;
    u32x4 v[Shape::kItems];
#pragma unroll
    for (int i = 0; i < Shape::kItems; ++i) {
        const int id = tid + 512 * i, r = id / per_row;
        v[i] = id < items ? load_row8(x + r * ldx, 8 * (id - r * per_row), k) : (u32x4){0, 0, 0, 0};
    }
    __syncthreads();                         // row_amax is clear
#pragma unroll
    for (int i = 0; i < Shape::kItems; ++i) {
        const int id = tid + 512 * i;
        const uint32_t amax = eight_umax(amax8(v[i], 0));
        if (id < items && (lane & 7) == 0) atomicMax(&row_amax[id / per_row], amax);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < Shape::kItems; ++i) {
        const int id = tid + 512 * i, r = id / per_row;
        if (id >= items) break;
        *reinterpret_cast<u32x2*>(lds + r * pitch + 8 * (id - r * per_row)) = codes8(v[i], row_scale(row_amax[r]));
    }
    __syncthreads();
    const char* frag[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) frag[i] = lds + min(16 * i + (lane & 15), rows - 1) * pitch + wave * kSlice + (lane >> 4) * 16;
    out.sa[0] = row_scale(row_amax[min(16 * (wave % MT) + (lane & 15), rows - 1)]).scale;
    i32x4 acc[MT][CT] = {};
    for (int t = 0; t < count; t += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (t + d >= count) break;
            if (t + d + D - 1 < count) request(wf[(d + D - 1) % D]);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const i32x4 xf = *reinterpret_cast<const i32x4*>(frag[i] + (t + d) * 8 * kSlice);
#pragma unroll
                for (int j = 0; j < CT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[d][j], xf, acc[i][j], 0, 0, 0);
            }
        }
    }
    __syncthreads();                         // the rows have been read
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < CT; ++j) *reinterpret_cast<i32x4*>(lds + ((wave * MT + i) * CT + j) * 1024 + lane * 16) = acc[i][j];
    __syncthreads();
    if (wave < MT) {
        i32x4 sum[1][2] = {};
#pragma unroll
        for (int w = 0; w < 8; ++w)
#pragma unroll
            for (int j = 0; j < 2; ++j) sum[0][j] += *reinterpret_cast<const i32x4*>(lds + ((w * MT + wave) * CT + j) * 1024 + lane * 16);
        out.finish(p, sum, mu, n0, lane, lds + Shape::kSums + wave * 2048);
    }
}

// The same for few or very long rows: a work-group per row, so that a thousand rows occupy the whole chip and a thread holds a
// quarter of what a lane above does (1504 x 4096: 5.4 against 5.8 us, 1504 x 16384: 13.1 against 21.6, 12032 x 16384: 88
// against 130; but 12032 x 2048: 13.9 against 12.8 and 48128 x 4096: 101 against 89, where the barrier of each row costs more).
template <int NV, bool ONCE = false>
__global__ __launch_bounds__(256) void quant_i8_row_kernel(const uint16_t* __restrict__ x, int64_t ldx, int64_t k,
                                                           int8_t* __restrict__ y, int64_t ldy, float* __restrict__ scale) {
    __shared__ uint32_t wave_amax[4];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x, kp = (k + kSlice - 1) / kSlice * kSlice;
    const uint16_t* xr = x + row * ldx;
    int8_t* yr = y + row * ldy;
    u32x4 v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = load_row8<ONCE>(xr, 8 * tid + 2048 * i, k);
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) amax = amax8(v[i], amax);
    amax = wave_umax(amax);
    if ((tid & 63) == 0) wave_amax[tid >> 6] = amax;
    __syncthreads();
    const RowScale s = row_scale(max(max(wave_amax[0], wave_amax[1]), max(wave_amax[2], wave_amax[3])));
    if (tid == 0) scale[row] = s.scale;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int64_t c = 8 * tid + 2048 * i;
        if (c < kp) *reinterpret_cast<u32x2*>(yr + c) = codes8(v[i], s);
    }
}

// Row-major weight codes -> packed pieces, one 16-byte chunk per thread.
__global__ __launch_bounds__(256) void gemm_pack_w_i8_kernel(const int8_t* __restrict__ w, int64_t ldw, int64_t n, int64_t k,
                                                             int64_t ks, int64_t chunks, int8_t* __restrict__ out) {
    const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (idx >= chunks) return;
    const int lane = (int)(idx & 63);
    const int64_t piece = idx >> 6, grp = piece / ks, t = piece - grp * ks;
    const int64_t row = grp * 16 + (lane & 15), col = t * kSlice + (lane >> 4) * 16;
    struct __attribute__((packed, aligned(1))) Any {
        uint32_t v[4];
    } c = {{0, 0, 0, 0}};
    const int8_t* src = w + row * ldw + col;
    if (row < n) {
        if (col + 16 <= k) {
            c = *reinterpret_cast<const Any*>(src);
        } else {
            for (int e = 0; e < 16; ++e)
                if (col + e < k) c.v[e >> 2] |= (uint32_t)(uint8_t)src[e] << (8 * (e & 3));
        }
    }
    *reinterpret_cast<u32x4*>(out + idx * 16) = (u32x4){c.v[0], c.v[1], c.v[2], c.v[3]};
}

static int check_gemm(const char* what, const int8_t* w, const float* scale_w, const float* bias, const float* resid,
                      int64_t ldr, const void* c, int64_t ldc, int64_t m, int64_t n, int64_t k, int32_t epilogue) {
    OASR_REQUIRE(m >= 0 && n > 0 && k > 0, "%s: n and k must be positive, m not negative", what);
    OASR_REQUIRE(k <= kMaxK, "%s: k=%lld exceeds %lld (the sums are 32-bit integers)", what, (long long)k, (long long)kMaxK);
    OASR_REQUIRE(m < ((int64_t)1 << 31) && n < ((int64_t)1 << 31), "%s: m and n must be below 2^31", what);
    OASR_REQUIRE(epilogue >= OASR_EPI_BIAS_BF16 && epilogue <= OASR_EPI_BIAS_F32, "%s: unknown epilogue %d", what, epilogue);
    OASR_REQUIRE(epilogue != OASR_EPI_GLU_BF16 || n % 32 == 0, "%s: the GLU epilogue needs n=%lld to be a multiple of 32", what,
                 (long long)n);
    OASR_REQUIRE(ldc >= (epilogue == OASR_EPI_GLU_BF16 ? n / 2 : n), "%s: ldc=%lld is shorter than a row", what, (long long)ldc);
    OASR_REQUIRE(epilogue != OASR_EPI_RESIDUAL_F32 || ldr >= n, "%s: ldr=%lld is shorter than a row", what, (long long)ldr);
    if (m == 0) return OASR_OK;
    OASR_REQUIRE(w && scale_w && c, "%s: null pointer", what);
    OASR_REQUIRE(epilogue != OASR_EPI_RESIDUAL_F32 || resid, "%s: residual epilogue without resid", what);
    const int elt = epilogue == OASR_EPI_RESIDUAL_F32 || epilogue == OASR_EPI_BIAS_F32 ? 4 : 2;
    OASR_REQUIRE(((uintptr_t)w & 15) == 0, "%s: the packed weights must be 16-byte aligned", what);
    OASR_REQUIRE(((uintptr_t)c & (elt - 1)) == 0 && ((uintptr_t)scale_w & 3) == 0 && ((uintptr_t)bias & 3) == 0 &&
                     ((uintptr_t)resid & 3) == 0,
                 "%s: misaligned pointer", what);
    return OASR_OK;
}

// Which kernel runs a product: the one with the least estimated time, rounds * (begin + steps * step) microseconds.  A round is
// 256 work-groups (one per CU; where several share a CU a further round costs `share` of one), a step one slice (64 k), or
// for the splitting kernel eight.  The figures are fitted to times of all forms over 364 sizes (m 17 .. 4096, n 512 .. 16384,
// k 512 .. 16384) and pick within 1.4 % of the fastest form on average over those; larger m and smaller n are extrapolated, and the
// 256 x 256 form, which takes most of the large ones, is priced at ceil(tiles / 256) rounds although its whole row tiles per XCD
// may need one more (about a quarter of the sizes that it is picked for, up to twice the estimate).  E.g. 1504 x 1024 x 4096: 96 rows split 14.8 us, 128 x 128
// tiles 25.8, 256 x 256 43.4; 1504 x 4096 x 1024: 23.2 (32 rows split), 14.4, 20.1; 512 x 1024 x 512: 4.5, 6.2, 10.0.
// 16 rows split re-read the weights once per row tile: with more than 128 work-groups of them 32 rows are faster
// (300 x 4096 x 4096: 17.4 against 22.3 us).
struct Form {
    int bm, bn, slices;         // tile, slices per step
    double begin, step, share;
};
enum { kSplit16, kSplit32, kSplit64, kSplit96, kSplit128, kTile128, kTile256, kForms };
static const Form kFormTable[kForms] = {
    {16, 64, 8, 1.31, 0.50, 0.7}, {32, 64, 8, 1.69, 0.62, 0.8},  {64, 64, 8, 2.44, 0.79, 1.0},  {96, 64, 8, 3.93, 1.06, 1.0},
    {128, 64, 8, 4.49, 1.31, 1.0}, {128, 128, 1, 4.23, 0.32, 0.7}, {256, 256, 1, 10.4, 0.54, 1.0}};

static int choose_form(const GemmArgs& p) {
    int best = kTile128;
    double least = 1e300;
    for (int f = 0; f < kForms; ++f) {
        const Form& t = kFormTable[f];
        const int64_t groups = ((p.m + t.bm - 1) / t.bm) * ((p.n + t.bn - 1) / t.bn);
        if (groups >= (f == kTile256 ? kMaxWideTiles : kMaxGroups)) continue;       // more than a launch has: a form of larger tiles
        if (f == kSplit16 && p.m > 16 && groups > 128) continue;
        if (f == kTile256 && p.lda >= (1 << 26)) continue;       // 32 row pitches have to fit its 32-bit offsets
        const double rounds = (double)((groups + 255) / 256) * t.share;
        const double us = (rounds < 1.0 ? 1.0 : rounds) * (t.begin + (p.ks + t.slices - 1) / t.slices * t.step);
        if (us < least) {
            least = us;
            best = f;
        }
    }
    return best;
}

// The map of a launch of tm x tn tiles of bm x bn, and its work-groups (a few of which may have no tile).  Of the ways to deal
// the tiles to the eight XCDs as 1 x 8, 2 x 4, 4 x 2 or 8 x 1 blocks, the one that fetches least; rows of A count six times (they
// come in half lines, 64 bytes per slice: with a weight of one 1504 x 1024 x 4096 takes 22.1 us instead of 20.2, with four
// 1000 x 1000 x 4096 18.1 instead of 16.6).  A way that leaves an XCD more than an eighth above the average, or needs another
// round of work-groups, is out.  Against tiles not dealt at all, calls with their quantiser: 50 x 8192 x 8192 29.3 -> 18.3 us,
// 100 x 4096 x 16384 54.4 -> 26.0, 900 x 1024 x 8192 29.4 -> 24.6, 1504 x 4096 x 1024 19.5 -> 18.1; 2000 x 1024 x 4096 23.4 -> 24.0.
static int64_t map_tiles(int tm, int tn, int bm, int bn, TileMap& map) {
    const int64_t tiles = (int64_t)tm * tn;
    map = {tm, tn, 0, 0, Divisor(tn)};
    int64_t least = INT64_MAX;
    for (int a = 0; a < 4; ++a) {
        const int rows = (tm + (1 << a) - 1) >> a, cols = (tn + (8 >> a) - 1) / (8 >> a);
        const int64_t cost = 6 * (int64_t)rows * bm + (int64_t)cols * bn, most = (int64_t)rows * cols;
        if (64 * most > 9 * tiles || (most + 31) / 32 > (tiles + 255) / 256 || cost >= least) continue;
        least = cost;
        map = {tm, tn, a, rows, Divisor(cols)};
    }
    return map.rows ? 8 * (int64_t)map.rows * map.cols.d : tiles;
}

template <int EPI>
static void launch_form(int form, const GemmArgs& p, hipStream_t st) {
    const Form& t = kFormTable[form];
    const int tm = (int)((p.m + t.bm - 1) / t.bm), tn = (int)((p.n + t.bn - 1) / t.bn);
    const int64_t tiles = (int64_t)tm * tn;
    TileMap map;
    const dim3 grid((unsigned)map_tiles(tm, tn, t.bm, t.bn, map)), split(512);
    switch (form) {
        case kSplit16: hipLaunchKernelGGL((gemm_i8_split_kernel<EPI, 1>), grid, split, 0, st, p, map); break;
        case kSplit32: hipLaunchKernelGGL((gemm_i8_split_kernel<EPI, 2>), grid, split, 0, st, p, map); break;
        case kSplit64: hipLaunchKernelGGL((gemm_i8_split_kernel<EPI, 4>), grid, split, 0, st, p, map); break;
        case kSplit96: hipLaunchKernelGGL((gemm_i8_split_kernel<EPI, 6>), grid, split, 0, st, p, map); break;
        case kSplit128: hipLaunchKernelGGL((gemm_i8_split_kernel<EPI, 8>), grid, split, 0, st, p, map); break;
        case kTile128: hipLaunchKernelGGL((gemm_i8_tile_kernel<EPI, 2, 2, 4, 4, 4>), grid, dim3(256), 0, st, p, map); break;
        default:
            hipLaunchKernelGGL((gemm_i8_wide_kernel<EPI>), dim3((unsigned)(tiles < 256 ? (tiles + 7) / 8 * 8 : 256)), dim3(512), 0, st, p, tm, tn);
    }
}

// Whether a call quantises inside the product (and needs no workspace): the row tiles of 16 per work-group, or 0.  Up to 16
// rows always where they fit; more rows (32 to a work-group) while the work-groups fit the CUs once: 99 x 2048 x 1024 8.5 us on
// the device against 7.9 in two launches, but 8.4 against 12.4 per call made from a program (a launch costs the host 3.5).  Twice as
// many work-groups take twice as long (99 x 4096 x 1024: 16.7 against 8.7).
static int few_rows(int64_t m, int64_t n, int64_t k) {
    const int64_t kp = round_up(k, kSlice);
    if (m <= 16 && m * kp <= FewShape<1>::kCodes) return 1;
    if (32 * kp <= FewShape<2>::kCodes && (m + 31) / 32 * ((n + kFewColumns - 1) / kFewColumns) <= 256) return 2;
    return 0;
}

static int launch_few(int mt, const GemmArgs& p, const uint16_t* x, int64_t ldx, int64_t k, int32_t epilogue, hipStream_t st) {
    const int tm = (int)((p.m + 16 * mt - 1) / (16 * mt));
    const int64_t tn = (p.n + kFewColumns - 1) / kFewColumns;
    OASR_REQUIRE(tm * tn < kMaxGroups, "linear_i8: m=%lld x n=%lld is too large a result", (long long)p.m, (long long)p.n);
    const dim3 grid((unsigned)(tm * tn)), blk(512);
#define OASR_FEW(E)                                                                                             \
    do {                                                                                                        \
        if (mt == 1) hipLaunchKernelGGL((linear_i8_few_kernel<E, 1>), grid, blk, 0, st, p, x, ldx, (int)k, tm); \
        else hipLaunchKernelGGL((linear_i8_few_kernel<E, 2>), grid, blk, 0, st, p, x, ldx, (int)k, tm);         \
    } while (0)
    switch (epilogue) {
        case OASR_EPI_BIAS_BF16: OASR_FEW(OASR_EPI_BIAS_BF16); break;
        case OASR_EPI_BIAS_SWISH_BF16: OASR_FEW(OASR_EPI_BIAS_SWISH_BF16); break;
        case OASR_EPI_GLU_BF16: OASR_FEW(OASR_EPI_GLU_BF16); break;
        case OASR_EPI_RESIDUAL_F32: OASR_FEW(OASR_EPI_RESIDUAL_F32); break;
        default: OASR_FEW(OASR_EPI_BIAS_F32); break;
    }
#undef OASR_FEW
    OASR_CHECK_LAUNCH("linear_i8");
    return OASR_OK;
}

static int launch_gemm(const GemmArgs& p, int32_t epilogue, hipStream_t st) {
    const int form = choose_form(p);
    const Form& t = kFormTable[form];
    OASR_REQUIRE((p.m + t.bm - 1) / t.bm * ((p.n + t.bn - 1) / t.bn) < (form == kTile256 ? kMaxWideTiles : kMaxGroups),
                 "gemm_i8: m=%lld x n=%lld is too large a result", (long long)p.m, (long long)p.n);
    switch (epilogue) {
        case OASR_EPI_BIAS_BF16: launch_form<OASR_EPI_BIAS_BF16>(form, p, st); break;
        case OASR_EPI_BIAS_SWISH_BF16: launch_form<OASR_EPI_BIAS_SWISH_BF16>(form, p, st); break;
        case OASR_EPI_GLU_BF16: launch_form<OASR_EPI_GLU_BF16>(form, p, st); break;
        case OASR_EPI_RESIDUAL_F32: launch_form<OASR_EPI_RESIDUAL_F32>(form, p, st); break;
        default: launch_form<OASR_EPI_BIAS_F32>(form, p, st); break;
    }
    OASR_CHECK_LAUNCH("gemm_i8");
    return OASR_OK;
}

static GemmArgs gemm_args(const int8_t* a, int64_t lda, const int8_t* w, const float* scale_a, const float* scale_w,
                          const float* bias, const float* resid, int64_t ldr, void* c, int64_t ldc, int64_t m, int64_t n, int64_t k,
                          float alpha, int32_t epilogue) {
    GemmArgs p;
    p.a = a;
    p.w = w;
    p.scale_a = scale_a;
    p.scale_w = scale_w;
    p.bias = bias;
    p.resid = resid;
    p.c = c;
    p.lda = lda;
    p.ldr = ldr;
    p.ldc = ldc;
    p.m = m;
    p.n = n;
    p.ks = (int)((k + kSlice - 1) / kSlice);
    p.ng = (int)((n + 15) / 16);
    p.alpha = alpha;
    const int elt = epilogue == OASR_EPI_RESIDUAL_F32 || epilogue == OASR_EPI_BIAS_F32 ? 4 : 2;
    p.vec = ((uintptr_t)c & 15) == 0 && ((uintptr_t)resid & 15) == 0 && ldc * elt % 16 == 0 && ldr % 4 == 0;
    return p;
}

static int quant_rows(const uint16_t* x, int64_t ldx, int64_t rows, int64_t k, int8_t* y, int64_t ldy, float* scale,
                      hipStream_t st) {
    const dim3 grid((unsigned)((rows + 3) / 4)), blk(256);
    const bool once = rows * k >= ((int64_t)32 << 20);     // 64 MiB of activations
    if ((rows <= 8192 && k > 1024 && k <= 16384) || (k > 8192 && k <= 16384)) {
        const dim3 one((unsigned)rows);
        if (k <= 2048) hipLaunchKernelGGL(quant_i8_row_kernel<1>, one, blk, 0, st, x, ldx, k, y, ldy, scale);
        else if (k <= 4096) hipLaunchKernelGGL(quant_i8_row_kernel<2>, one, blk, 0, st, x, ldx, k, y, ldy, scale);
        else if (k <= 8192) hipLaunchKernelGGL(quant_i8_row_kernel<4>, one, blk, 0, st, x, ldx, k, y, ldy, scale);
        else if (once) hipLaunchKernelGGL((quant_i8_row_kernel<8, true>), one, blk, 0, st, x, ldx, k, y, ldy, scale);
        else hipLaunchKernelGGL(quant_i8_row_kernel<8>, one, blk, 0, st, x, ldx, k, y, ldy, scale);
        OASR_CHECK_LAUNCH("quant_i8_rows");
        return OASR_OK;
    }
#define OASR_QUANT_I8(NV)                                                                                              \
    do {                                                                                                               \
        if (once) hipLaunchKernelGGL((quant_i8_rows_kernel<NV, true>), grid, blk, 0, st, x, ldx, rows, k, y, ldy, scale); \
        else hipLaunchKernelGGL((quant_i8_rows_kernel<NV, false>), grid, blk, 0, st, x, ldx, rows, k, y, ldy, scale);     \
    } while (0)
    // the row in registers up to 8192 columns (16 loads per lane), the smallest form that covers it
    if (k <= 512) OASR_QUANT_I8(1);
    else if (k <= 1024) OASR_QUANT_I8(2);
    else if (k <= 2048) OASR_QUANT_I8(4);
    else if (k <= 4096) OASR_QUANT_I8(8);
    else if (k <= 8192) OASR_QUANT_I8(16);
    else hipLaunchKernelGGL((quant_i8_rows_kernel<0, false>), grid, blk, 0, st, x, ldx, rows, k, y, ldy, scale);   // two sweeps: caches wanted
#undef OASR_QUANT_I8
    OASR_CHECK_LAUNCH("quant_i8_rows");
    return OASR_OK;
}

}  // namespace i8
}  // namespace oasr

using namespace oasr;

extern "C" {

int oasr_quant_i8_rows(const uint16_t* x, int64_t ldx, int64_t rows, int64_t k, int8_t* y, int64_t ldy, float* scale,
                       void* stream) {
    OASR_REQUIRE(rows >= 0 && k > 0, "quant_i8_rows: k must be positive and rows not negative");
    OASR_REQUIRE(rows < i8::kMaxRows, "quant_i8_rows: rows must be below 2^24");
    OASR_REQUIRE(ldx >= k && ldy % 16 == 0 && ldy >= round_up(k, i8::kSlice),
                 "quant_i8_rows: ldx must cover k, ldy must be a multiple of 16 and cover k rounded up to 64");
    if (rows == 0) return OASR_OK;
    OASR_REQUIRE(x && y && scale, "quant_i8_rows: null pointer");
    OASR_REQUIRE(((uintptr_t)x & 1) == 0 && ((uintptr_t)y & 15) == 0 && ((uintptr_t)scale & 3) == 0,
                 "quant_i8_rows: misaligned pointer");
    return i8::quant_rows(x, ldx, rows, k, y, ldy, scale, (hipStream_t)stream);
}

int64_t oasr_gemm_i8_packed_bytes(int64_t n, int64_t k) {
    if (n <= 0 || k <= 0) return 0;
    return round_up(n, 16) * round_up(k, i8::kSlice);
}

int oasr_gemm_pack_w_i8(const int8_t* w, int64_t ldw, int64_t n, int64_t k, int8_t* out, void* stream) {
    OASR_REQUIRE(n > 0 && k > 0 && ldw >= k, "gemm_pack_w_i8: n and k must be positive and ldw cover k");
    OASR_REQUIRE(k <= i8::kMaxK && n < ((int64_t)1 << 31), "gemm_pack_w_i8: k must not exceed %lld and n must be below 2^31",
                 (long long)i8::kMaxK);
    OASR_REQUIRE(w && out && w != out, "gemm_pack_w_i8: null pointer or in-place call");
    OASR_REQUIRE(((uintptr_t)out & 15) == 0, "gemm_pack_w_i8: out must be 16-byte aligned");
    const int64_t chunks = oasr_gemm_i8_packed_bytes(n, k) / 16;
    OASR_REQUIRE(chunks < ((int64_t)1 << 32) - 256, "gemm_pack_w_i8: the packed weights must be below 64 GiB");
    hipLaunchKernelGGL(i8::gemm_pack_w_i8_kernel, dim3((unsigned)((chunks + 255) / 256)), dim3(256), 0, (hipStream_t)stream, w, ldw,
                       n, k, round_up(k, i8::kSlice) / i8::kSlice, chunks, out);
    OASR_CHECK_LAUNCH("gemm_pack_w_i8");
    return OASR_OK;
}

int oasr_gemm_i8(const int8_t* a, int64_t lda, const int8_t* w_packed, const float* scale_a, const float* scale_w,
                 const float* bias, const float* resid, int64_t ldr, void* c, int64_t ldc, int64_t m, int64_t n, int64_t k, float alpha,
                 int32_t epilogue, void* stream) {
    const int rc = i8::check_gemm("gemm_i8", w_packed, scale_w, bias, resid, ldr, c, ldc, m, n, k, epilogue);
    if (rc != OASR_OK) return rc;
    OASR_REQUIRE(lda % 16 == 0 && lda >= round_up(k, i8::kSlice), "gemm_i8: lda must be a multiple of 16 and cover k rounded up to 64");
    if (m == 0) return OASR_OK;
    OASR_REQUIRE(a && scale_a, "gemm_i8: null pointer");
    OASR_REQUIRE(((uintptr_t)a & 15) == 0 && ((uintptr_t)scale_a & 3) == 0, "gemm_i8: misaligned pointer");
    return i8::launch_gemm(i8::gemm_args(a, lda, w_packed, scale_a, scale_w, bias, resid, ldr, c, ldc, m, n, k, alpha, epilogue), epilogue,
                           (hipStream_t)stream);
}

int64_t oasr_linear_i8_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    if (m <= 0 || n <= 0 || k <= 0 || i8::few_rows(m, n, k)) return 0;
    return round_up(m * round_up(k, i8::kSlice), 256) + round_up(m * 4, 256);
}

int oasr_linear_i8(const uint16_t* x, int64_t ldx, const int8_t* w_packed, const float* scale_w, const float* bias,
                   const float* resid, int64_t ldr, void* c, int64_t ldc, int64_t m, int64_t n, int64_t k, float alpha, int32_t epilogue,
                   void* workspace, int64_t workspace_bytes, void* stream) {
    const int rc = i8::check_gemm("linear_i8", w_packed, scale_w, bias, resid, ldr, c, ldc, m, n, k, epilogue);
    if (rc != OASR_OK) return rc;
    OASR_REQUIRE(ldx >= k, "linear_i8: ldx must cover k");
    if (m == 0) return OASR_OK;
    OASR_REQUIRE(x, "linear_i8: null pointer");
    OASR_REQUIRE(((uintptr_t)x & 1) == 0, "linear_i8: misaligned pointer");
    if (const int mt = i8::few_rows(m, n, k))
        return i8::launch_few(mt, i8::gemm_args(nullptr, 0, w_packed, nullptr, scale_w, bias, resid, ldr, c, ldc, m, n, k, alpha, epilogue), x,
                              ldx, k, epilogue, (hipStream_t)stream);
    OASR_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0, "linear_i8: workspace missing or not 256-byte aligned");
    if (workspace_bytes < oasr_linear_i8_workspace_bytes(m, n, k)) {
        set_error("linear_i8: workspace needs %lld bytes, got %lld", (long long)oasr_linear_i8_workspace_bytes(m, n, k),
                  (long long)workspace_bytes);
        return OASR_ECAPACITY;
    }
    OASR_REQUIRE(m < i8::kMaxRows, "linear_i8: m must be below 2^24");
    const int64_t kp = round_up(k, i8::kSlice);
    int8_t* q = static_cast<int8_t*>(workspace);
    float* s = reinterpret_cast<float*>(q + round_up(m * kp, 256));
    const int rq = i8::quant_rows(x, ldx, m, k, q, kp, s, (hipStream_t)stream);
    if (rq != OASR_OK) return rq;
    return i8::launch_gemm(i8::gemm_args(q, kp, w_packed, s, scale_w, bias, resid, ldr, c, ldc, m, n, k, alpha, epilogue), epilogue,
                           (hipStream_t)stream);
}

}  // extern "C"
