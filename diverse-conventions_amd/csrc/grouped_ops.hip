// grouped_ops.hip -- linear layers of several networks over one batch whose rows are sorted by network (gfx950): the products of training
// that oc_policy_forward's tables do for inference, with the gradients.
//   forward   Y[m, n]      = sum_k X[m, k] W_g[n, k] + b_g[n]          for the rows m of group g
//   backward  dX[m, k]     = sum_n dY[m, n] W_g[n, k]
//             dW_g[n, k]   = sum_{m in g} dY[m, n] X[m, k],   db_g[n] = sum_{m in g} dY[m, n]
//
// One tile kernel does all three: out[j][i] = sum_r I(i, r) J(j, r), i along the output's contiguous dimension.  An operand is either
// contiguous along the reduction (W and X of the forward pass) or along its own index (W for dX, both operands of dW); the tile is
// staged in LDS as it lies in memory, and the second kind is transposed on the way to the registers (ds_read_b64_tr_b16; f32: four
// 4-byte reads).  The matrix instruction's first operand is I, so that a lane ends up with four consecutive elements of an output row.
//
// Which rows belong to which group is read from the offsets on the device: a workgroup counts the row tiles of all groups, finds its
// own, and leaves if there is none, so that ragged groups cost no host round trip and no tile crosses a group.  Tiles are dealt to the
// eight XCDs in contiguous runs: workgroups that share a network's weights share an L2.  (dW: every XCD gets its share of every group,
// because a group's tiles cost what its rows are: 583 -> 387 us on ragged groups.)
//
// What bounds it (MI355X).  16-bit, 256 x 256 tiles: 4096^3 bf16 122 us = 1120 TFLOP/s (the library's product 1350); 16 ragged groups, 16 k
// rows x 2048 x 4096: 323 - 329 us forward, 370 - 376 dx, 365 dw (the last round of tiles is half empty, a group's last tile too; even groups
// 270 us forward = 1018 TFLOP/s).  The even forward takes 200 us without the copies, 234 without the matrix instructions, 261 without the LDS
// reads and 260 without its stores: the copies from L2 into LDS (2.1 GB, 8 TB/s over all CUs) and the wavefronts' meeting at two barriers a
// step bound it.  f32: 4096^3 1013 us = 136 TFLOP/s (library 150).  One to three rows a group: the weights' bytes, 252 MB in 58 us =
// 4.3 TB/s.  Widths or addresses off 16 bytes go through registers one step ahead: 8192 rows of 2047 -> 2047 bf16 96 us forward and 517
// backward, of 2048 -> 2048 64 and 152; f32 574 and 1211 against 515 and 1111.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "overcooked_ops.h"
#include "oc_internal.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

struct GroupedArgs {
    const void *I, *J;                                     // operand of the output's contiguous index, operand of its rows
    const void *bias;                                      // forward: [groups][ni] or NULL
    void *out;                                             // in the operands' type, or f32 partial sums of a split reduction
    const void *offsets;                                   // [groups + 1] int32 or int64
    long long ld_i, ld_j, ld_out;                          // row lengths in memory, in elements
    long long rows;                                        // of the whole batch
    int groups, ni, nj, red;                               // ni: output row length; rows product: red; dW: nj = output rows per group
    int offsets64, splits;
    void *bias_out;                                        // dW: db or NULL, by further workgroups of the launch
    int bias_splits, weight_blocks;
};

__device__ __forceinline__ long long offset_at(const GroupedArgs &a, int g) {
    const long long o = a.offsets64 ? static_cast<const long long *>(a.offsets)[g] : static_cast<long long>(static_cast<const int *>(a.offsets)[g]);
    return o < 0 ? 0 : o > a.rows ? a.rows : o;            // never outside the batch, whatever the offsets say
}

template <typename T> struct Mat;
template <> struct Mat<__bf16> {
    typedef bf16x8 frag;
    static __device__ __forceinline__ void mma(f32x4 &c, const frag &a, const frag &b) { c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mat<_Float16> {
    typedef f16x8 frag;
    static __device__ __forceinline__ void mma(f32x4 &c, const frag &a, const frag &b) { c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mat<float> {
    typedef f32x4 frag;
    static __device__ __forceinline__ void mma(f32x4 &c, const frag &a, const frag &b) {
        // element s of the lanes' pieces is one step of four reduction indices: which ones does not matter as long as both operands agree
#pragma unroll
        for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
    }
};

// Place of 16-byte piece c of row r of a staged tile, in bytes.  Contiguous along the reduction: rows of RB (64 or 128) bytes, read by 16
// lanes at 16 different rows at once.  Otherwise: rows of N elements, read at four rows 8 apart (16-bit: and four neighbours of each).
// The exclusive or spreads those over the banks; the piece at place p of row r is piece p under the same operation.
template <typename T, bool TR, int N, int RB>
__device__ __forceinline__ int swap_piece(int r, int c) {
    if (!TR) return RB == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3);
    constexpr int kPieces = N * static_cast<int>(sizeof(T)) / 16;
    if (sizeof(T) == 2) return c ^ ((((r & 3) | (((r >> 3) & 3) << 2)) & (kPieces / 2 - 1)) << 1);
    return c ^ ((((r >> 2) & 3) << 2) & (kPieces - 1));
}
template <typename T, bool TR, int N, int RB>
__device__ __forceinline__ int place(int r, int c) {
    constexpr int kRow = TR ? N * static_cast<int>(sizeof(T)) : RB;
    return r * kRow + (swap_piece<T, TR, N, RB>(r, c) << 4);
}

__device__ __attribute__((aligned(16))) uint32_t g_zero_piece[4];           // where pieces behind the reduction's end are read from

// A tile of one operand, copied from memory to LDS without passing through registers (aligned rows): every thread asks for kPer pieces of
// 16 bytes, a wavefront's 64 land one behind the other.  Indexes behind the operand's end are read from its last row or piece -- their
// results are not stored --, reduction indexes behind the end from a piece of zeros, on both sides: what lies there may be anything.
// What the lanes add to the tile's address is worked out once; the address itself moves in scalar registers (32 bits for the lanes: the host
// takes the other way for rows beyond 2^31 bytes a tile).
template <typename T, bool TR, int N, int RB, int THREADS>
struct Copy {
    static constexpr int V = 16 / sizeof(T), BK = RB / sizeof(T);
    static constexpr int kRowPieces = TR ? N / V : RB / 16;
    static constexpr int kPer = N * RB / 16 / THREADS;
    static_assert(kPer * THREADS * 16 == N * RB, "every thread carries the same number of pieces");
    uint32_t off[kPer];
    const char *base;
    long long step;

    __device__ __forceinline__ void init(const T *first, long long ld, long long at, long long r0, long long own) {
        base = reinterpret_cast<const char *>(TR ? first + r0 * ld + at : first + at * ld + r0);
        step = (TR ? BK * ld : BK) * static_cast<long long>(sizeof(T));
        const int left = own > N ? N - 1 : static_cast<int>(own) - 1;
#pragma unroll
        for (int n = 0; n < kPer; ++n) {
            const int q = threadIdx.x + n * THREADS, row = q / kRowPieces, c = swap_piece<T, TR, N, RB>(row, q % kRowPieces);
            const int i = TR ? c * V : row, mine = i <= left ? i : TR ? left / V * V : left;
            off[n] = static_cast<uint32_t>(TR ? row * ld + mine : mine * ld + c * V) * static_cast<uint32_t>(sizeof(T));
        }
    }
    // wave: the wavefront's number, red: reduction indexes left from this step's first
    __device__ __forceinline__ void issue(char *lds, int wave, long long red) {
        char *to = lds + wave * 1024;
#pragma unroll
        for (int n = 0; n < kPer; ++n) {
            const char *from = base + off[n];
            if (red < BK) {
                const int q = threadIdx.x + n * THREADS, row = q / kRowPieces;
                const int r = TR ? row : swap_piece<T, TR, N, RB>(row, q % kRowPieces) * V;
                if (r >= red) from = reinterpret_cast<const char *>(g_zero_piece);
            }
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                             (__attribute__((address_space(3))) void *)(to + n * THREADS * 16), 16, 0, 0);
        }
        base += step;
    }
};

// The same through registers, for rows at any address and of any length: every thread carries kPer pieces of 16 bytes.
template <typename T, bool TR, int N, int THREADS>
struct Stage {
    static constexpr int V = 16 / sizeof(T), BK = 128 / sizeof(T);
    static constexpr int kRowPieces = TR ? N / V : 8;
    static constexpr int kPer = N * 8 / THREADS;
    static_assert(N * 8 % THREADS == 0, "every thread carries the same number of pieces");
    const T *src[kPer];
    u32x4 x[kPer];

    // `at`: index of the tile's first own index, `end`: their number; r0: first reduction index
    __device__ __forceinline__ void init(const T *base, long long ld, long long at, long long r0) {
#pragma unroll
        for (int n = 0; n < kPer; ++n) {
            const int q = threadIdx.x + n * THREADS, row = q / kRowPieces, c = q % kRowPieces;
            src[n] = TR ? base + (r0 + row) * ld + at + c * V : base + (at + row) * ld + r0 + c * V;
        }
    }
    // own: own indexes left from the tile's first, red: reduction indexes left from this step's first.  Outside: zeros.
    __device__ __forceinline__ void load(long long own, long long red) {
#pragma unroll
        for (int n = 0; n < kPer; ++n) {
            const int q = threadIdx.x + n * THREADS, row = q / kRowPieces, c = q % kRowPieces;
            const long long row_left = (TR ? red : own) - row, left = (TR ? own : red) - c * V;
            x[n] = u32x4{0, 0, 0, 0};
            if (row_left > 0 && left > 0) {
                if (left >= V) {
                    x[n] = *reinterpret_cast<const u32x4_a2 *>(src[n]);
                } else {
                    union { u32x4 raw; T e[V]; } p;
                    p.raw = x[n];
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (i < left) p.e[i] = src[n][i];
                    x[n] = p.raw;
                }
            }
        }
    }
    __device__ __forceinline__ void advance(long long ld) {
#pragma unroll
        for (int n = 0; n < kPer; ++n) src[n] += TR ? BK * ld : BK;
    }
    __device__ __forceinline__ void store(char *lds) const {
#pragma unroll
        for (int n = 0; n < kPer; ++n) {
            const int q = threadIdx.x + n * THREADS;
            *reinterpret_cast<u32x4 *>(lds + place<T, TR, N, 128>(q / kRowPieces, q % kRowPieces)) = x[n];
        }
    }
};

// The lanes' pieces of an operand for matrix step kk of a staged tile, COUNT own indexes 16 apart from `own0 + lane % 16` on; 16-bit:
// reduction indexes 32 kk + 8 (lane / 16) + 0..7, f32: 16 kk + 4 (lane / 16) + 0..3.
// The transposing reads are written out, four pieces and their wait at a time: in front of the builtin the compiler waits for every copy
// to LDS that is on its way (it cannot tell that they go to other buffers), and there would be no pipeline.
#define OC_READ_TR "ds_read_b64_tr_b16 "
template <int STEP>
__device__ __forceinline__ void read_transposed(uint64_t (&x)[2], uint32_t a) {
    asm volatile(OC_READ_TR "%0, %2\n\t" OC_READ_TR "%1, %2 offset:%3\n\ts_waitcnt lgkmcnt(0)" : "=&v"(x[0]), "=&v"(x[1]) : "v"(a), "n"(STEP) : "memory");
}
template <int STEP>
__device__ __forceinline__ void read_transposed(uint64_t (&x)[4], uint32_t a, uint32_t b) {
    asm volatile(OC_READ_TR "%0, %4\n\t" OC_READ_TR "%1, %4 offset:%6\n\t" OC_READ_TR "%2, %5\n\t" OC_READ_TR "%3, %5 offset:%6\n\ts_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]) : "v"(a), "v"(b), "n"(STEP) : "memory");
}
template <int STEP>
__device__ __forceinline__ void read_transposed(uint64_t (&x)[8], uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile(OC_READ_TR "%0, %8\n\t" OC_READ_TR "%1, %8 offset:%12\n\t" OC_READ_TR "%2, %9\n\t" OC_READ_TR "%3, %9 offset:%12\n\t"
                 OC_READ_TR "%4, %10\n\t" OC_READ_TR "%5, %10 offset:%12\n\t" OC_READ_TR "%6, %11\n\t" OC_READ_TR "%7, %11 offset:%12\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]), "=&v"(x[6]), "=&v"(x[7])
                 : "v"(a), "v"(b), "v"(c), "v"(d), "n"(STEP) : "memory");
}
#undef OC_READ_TR

// Places that do not change from step to step are kept in `off`.
template <typename T, bool TR, int N, int RB, int COUNT>
struct Frags {
    static constexpr int kOff = TR ? (sizeof(T) == 2 ? COUNT : 1) : RB / 64;
    uint32_t off[kOff];

    __device__ __forceinline__ void init(int own0) {
        const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
        if constexpr (!TR) {
#pragma unroll
            for (int kk = 0; kk < kOff; ++kk) off[kk] = place<T, false, N, RB>(own0 + i, g + 4 * kk);       // 16 rows on: the same swizzle
        } else if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int x = 0; x < COUNT; ++x) off[x] = place<T, true, N, RB>(8 * g + (i >> 2), ((own0 >> 4) + x) * 2 + ((i & 3) >> 1)) + (i & 1) * 8;
        } else {
            off[0] = own0 + i;
        }
    }
    // kk: the matrix step
    __device__ __forceinline__ void read(const char *lds, int kk, typename Mat<T>::frag (&out)[COUNT]) const {
        if constexpr (!TR) {
#pragma unroll
            for (int x = 0; x < COUNT; ++x) out[x] = *reinterpret_cast<const typename Mat<T>::frag *>(lds + off[kk] + x * 16 * RB);
        } else if constexpr (sizeof(T) == 2) {
            constexpr int kRow = N * 2, kStep = 4 * kRow;  // reduction indexes 4 on, and 32 on: the same swizzle
            const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char *)lds)) + kk * 32 * kRow;
            constexpr int kBatch = COUNT >= 4 ? 4 : COUNT;
            static_assert(COUNT % kBatch == 0, "whole batches");
#pragma unroll
            for (int x = 0; x < COUNT; x += kBatch) {
                union { uint64_t raw[2 * kBatch]; typename Mat<T>::frag v[kBatch]; } y;
                if constexpr (kBatch == 4) read_transposed<kStep>(y.raw, base + off[x], base + off[x + 1], base + off[x + 2], base + off[x + 3]);
                else if constexpr (kBatch == 2) read_transposed<kStep>(y.raw, base + off[x], base + off[x + 1]);
                else read_transposed<kStep>(y.raw, base + off[x]);
#pragma unroll
                for (int k = 0; k < kBatch; ++k) out[x + k] = y.v[k];
            }
        } else {
            const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
            for (int x = 0; x < COUNT; ++x)
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int r = 16 * kk + 4 * g + s, own = off[0] + 16 * x;
                    out[x][s] = *reinterpret_cast<const float *>(lds + place<T, true, N, RB>(r, own >> 2) + (own & 3) * 4);
                }
        }
    }
};

// The workgroup's place in the run of its XCD: workgroups go round robin over 8 XCDs, each gets a contiguous run of `total` tiles.
__device__ __forceinline__ int xcd_tile(int block, int total) {
    const int per = total >> 3, rest = total & 7, xcd = block & 7, k = block >> 3;
    return xcd * per + (xcd < rest ? xcd : rest) + k;
}
__device__ __forceinline__ bool xcd_has(int block, int total) { return (block >> 3) < (total >> 3) + ((block & 7) < (total & 7) ? 1 : 0); }

enum { PRODUCT_ROWS = 0, PRODUCT_WEIGHTS = 1 };

// Column sums of dY per group: a workgroup has 64 columns of one group and one split of its rows; 4 columns a thread.
template <typename T, int THREADS>
__device__ __forceinline__ void column_sums(const GroupedArgs &a, int block, float (*part)[64]) {
    const int blocks_n = (a.nj + 63) / 64;
    const int split = block % a.bias_splits, tile = block / a.bias_splits, group = tile / blocks_n;
    const int c0 = (tile % blocks_n) * 64 + (threadIdx.x & 15) * 4, lane_row = threadIdx.x >> 4;
    constexpr int kRows = THREADS / 16;
    const long long row0 = offset_at(a, group);
    long long rows = offset_at(a, group + 1) - row0;
    if (rows < 0) rows = 0;
    const long long len = (rows + a.bias_splits - 1) / a.bias_splits, first = split * len, last = first + len < rows ? first + len : rows;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const T *src = static_cast<const T *>(a.J);
    typedef T four_t __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    if (c0 + 4 <= a.nj) {
#pragma unroll 4
        for (long long r = first + lane_row; r < last; r += kRows) {
            const four_t v = *reinterpret_cast<const four_t *>(src + (row0 + r) * a.ld_j + c0);
#pragma unroll
            for (int k = 0; k < 4; ++k) s[k] += static_cast<float>(v[k]);
        }
    } else {
        for (long long r = first + lane_row; r < last; r += kRows)
            for (int k = 0; k < 4; ++k)
                if (c0 + k < a.nj) s[k] += static_cast<float>(src[(row0 + r) * a.ld_j + c0 + k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) part[lane_row][(threadIdx.x & 15) * 4 + k] = s[k];
    __syncthreads();
    const int c = (tile % blocks_n) * 64 + threadIdx.x;
    if (threadIdx.x < 64 && c < a.nj) {
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < kRows; ++k) sum += part[k][threadIdx.x];
        if (a.bias_splits > 1) static_cast<float *>(a.bias_out)[(static_cast<long long>(split) * a.groups + group) * a.nj + c] = sum;
        else static_cast<T *>(a.bias_out)[static_cast<long long>(group) * a.nj + c] = static_cast<T>(sum);
    }
}

// RB: bytes of the reduction that a step takes per index of its own; STAGES: tiles in LDS, STAGES - 1 of them on their way (0: through
// registers, two tiles).
template <typename T, int BI, int BJ, int WI, int WJ, bool TRI, bool TRJ, int PRODUCT, int RB, int STAGES>
__global__ __launch_bounds__((BI / WI) * (BJ / WJ) * 64) void oc_grouped_kernel(const GroupedArgs a) {
    constexpr int THREADS = (BI / WI) * (BJ / WJ) * 64, BK = RB / sizeof(T);
    constexpr int FI = WI / 16, FJ = WJ / 16;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_i = (a.ni + BI - 1) / BI;
    const T *base_i = static_cast<const T *>(a.I), *base_j = static_cast<const T *>(a.J);
    int it, group;
    long long j0, j_left, r0, red;                         // first output row and how many are left, first reduction index and their number
    long long out_row;
    bool first_split = true;
    if (PRODUCT == PRODUCT_ROWS) {
        int total = 0;                                     // row tiles of all groups
        for (int b = 0; b < a.groups; b += 64) {
            int n = 0;
            if (b + lane < a.groups) {
                const long long rows = offset_at(a, b + lane + 1) - offset_at(a, b + lane);
                n = rows > 0 ? static_cast<int>((rows + BJ - 1) / BJ) : 0;
            }
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off);
            total += __builtin_amdgcn_readfirstlane(n);
        }
        // rows of no group: before the first, behind the last
        const long long head = offset_at(a, 0), tail = offset_at(a, a.groups);
        const long long stray = (head + (a.rows - tail)) * a.ni;
        for (long long e = static_cast<long long>(blockIdx.x) * THREADS + threadIdx.x; e < stray; e += static_cast<long long>(gridDim.x) * THREADS) {
            const long long r = e / a.ni, row = r < head ? r : tail + (r - head), at = row * a.ld_out + e % a.ni;
            if (a.splits == 1) static_cast<T *>(a.out)[at] = static_cast<T>(0.0f);
            else
                for (int k = 0; k < a.splits; ++k) static_cast<float *>(a.out)[k * a.rows * a.ld_out + at] = 0.0f;
        }
        total *= tiles_i;
        const int split = blockIdx.x % a.splits, block = blockIdx.x / a.splits;
        if (!xcd_has(block, total)) return;
        const int tile = xcd_tile(block, total);
        int before = 0, mine = 0;
        group = 0;
        for (int b = 0; b < a.groups; b += 64) {
            int n = 0;
            if (b + lane < a.groups) {
                const long long rows = offset_at(a, b + lane + 1) - offset_at(a, b + lane);
                n = rows > 0 ? static_cast<int>((rows + BJ - 1) / BJ) : 0;
            }
            int upto = n;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int y = __shfl_up(upto, off);
                if (lane >= off) upto += y;
            }
            const unsigned long long past = __ballot((before + upto) * tiles_i > tile);
            if (past) {
                const int l = __ffsll(past) - 1;
                group = b + l;
                mine = __builtin_amdgcn_readlane(n, l);
                before += __builtin_amdgcn_readlane(upto, l) - mine;
                break;
            }
            before += __builtin_amdgcn_readlane(upto, 63);
        }
        // the row tiles of a group go fastest: they share the weights' tile
        const int local = tile - before * tiles_i;
        it = local / mine;
        const long long row0 = offset_at(a, group), rows = offset_at(a, group + 1) - row0;
        j0 = row0 + static_cast<long long>(local % mine) * BJ;
        j_left = row0 + rows - j0;
        const long long len = ((a.red + a.splits - 1) / a.splits + BK - 1) / BK * BK;
        r0 = split * len;
        red = a.red - r0 < len ? a.red - r0 : len;
        out_row = split * a.rows + j0;
        first_split = split == 0;
        base_i += static_cast<long long>(group) * (TRI ? a.red : a.ni) * a.ld_i;
    } else {
        const int tiles_j = (a.nj + BJ - 1) / BJ, per_group = tiles_i * tiles_j;
        if (blockIdx.x >= static_cast<unsigned>(a.weight_blocks)) {
            column_sums<T, THREADS>(a, blockIdx.x - a.weight_blocks, reinterpret_cast<float (*)[64]>(lds));
            return;
        }
        // groups differ in rows: every XCD gets its share of each group, the same tiles of all of them
        const int group_blocks = per_group * a.splits;
        group = blockIdx.x / group_blocks;
        const int in_group = xcd_tile(blockIdx.x - group * group_blocks, group_blocks);
        const int split = in_group % a.splits, local = in_group / a.splits;
        it = local % tiles_i;
        j0 = static_cast<long long>(local / tiles_i) * BJ;
        j_left = a.nj - j0;
        const long long row0 = offset_at(a, group);
        long long rows = offset_at(a, group + 1) - row0;
        if (rows < 0) rows = 0;
        const long long len = ((rows + a.splits - 1) / a.splits + BK - 1) / BK * BK;
        r0 = row0 + split * len;
        red = rows - split * len < len ? rows - split * len : len;
        out_row = (static_cast<long long>(split) * a.groups + group) * a.nj + j0;
    }
    const long long i0 = static_cast<long long>(it) * BI, i_left = a.ni - i0;

    f32x4 acc[FI][FJ];
#pragma unroll
    for (int fi = 0; fi < FI; ++fi)
#pragma unroll
        for (int fj = 0; fj < FJ; ++fj) acc[fi][fj] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int wi = (wave % (BI / WI)) * WI, wj = (wave / (BI / WI)) * WJ;
    constexpr int kBuffer = (BI + BJ) * RB, kJ = BI * RB;                   // a buffer has I's tile in front of J's
    const int steps = red > 0 ? static_cast<int>((red + BK - 1) / BK) : 0;
    Frags<T, TRI, BI, RB, FI> at_i;
    Frags<T, TRJ, BJ, RB, FJ> at_j;
    at_i.init(wi);
    at_j.init(wj);
    const auto multiply = [&](const char *li) {
        const char *lj = li + kJ;
#pragma unroll
        for (int kk = 0; kk < RB / 64; ++kk) {
            typename Mat<T>::frag fi[FI], fj[FJ];
            at_j.read(lj, kk, fj);
            at_i.read(li, kk, fi);
#pragma unroll
            for (int x = 0; x < FI; ++x)
#pragma unroll
                for (int y = 0; y < FJ; ++y) Mat<T>::mma(acc[x][y], fi[x], fj[y]);
        }
    };
    if constexpr (STAGES > 0) {
        Copy<T, TRI, BI, RB, THREADS> ci;
        Copy<T, TRJ, BJ, RB, THREADS> cj;
        constexpr int kLoads = ci.kPer + cj.kPer;          // of a wavefront and step
        if (steps > 0) {
            ci.init(base_i, a.ld_i, i0, r0, i_left);
            cj.init(base_j, a.ld_j, j0, r0, j_left);
        }
        int here = 0, there = 0;                           // the buffers of the step at hand and of the next one to be copied
        const auto next = [](int at) { return at + kBuffer == STAGES * kBuffer ? 0 : at + kBuffer; };
        const auto issue = [&](int t) {
            const long long left = red - static_cast<long long>(t) * BK;
            ci.issue(lds + there, wave, left);
            cj.issue(lds + there + kJ, wave, left);
            there = next(there);
        };
        for (int t = 0; t < STAGES - 1 && t < steps; ++t) issue(t);
        if constexpr (THREADS == 512) {
            // Two wavefronts a SIMD, half a step apart: while one multiplies the other reads its pieces of the next step, so that LDS and
            // the matrix unit work at the same time (side by side in the same phase they took turns: 2.8 times a step's matrix time).
            // Barriers b0, b1, ..: wavefronts 0-3 read step t between b(2t-1) and b(2t), wavefronts 4-7 one barrier later.  Every wavefront
            // has its copies of step t in LDS before b(2t-1), and the buffer of step t - 1 is read for the last time before it.
            static_assert(RB == 64, "one matrix step");
            if (steps > 0) {
                if (steps >= STAGES - 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 2) * kLoads) : "memory");
                else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                if (wave >= 4) __builtin_amdgcn_s_barrier();
                for (int t = 0; t < steps; ++t) {
                    const char *li = lds + here;
                    here = next(here);
                    typename Mat<T>::frag fi[FI], fj[FJ];
                    asm volatile("" ::: "memory");
                    at_j.read(li + kJ, 0, fj);
                    at_i.read(li, 0, fi);
                    if (t + STAGES - 1 < steps) {
                        issue(t + STAGES - 1);
                        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * kLoads) : "memory");
                    } else {
                        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    __builtin_amdgcn_s_barrier();
                    __builtin_amdgcn_sched_barrier(0);
                    __builtin_amdgcn_s_setprio(1);
#pragma unroll
                    for (int x = 0; x < FI; ++x)
#pragma unroll
                        for (int y = 0; y < FJ; ++y) Mat<T>::mma(acc[x][y], fi[x], fj[y]);
                    __builtin_amdgcn_s_setprio(0);
                    __builtin_amdgcn_sched_barrier(0);
                    __builtin_amdgcn_s_barrier();
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (wave < 4) __builtin_amdgcn_s_barrier();
            }
        } else
        for (int t = 0; t < steps; ++t) {
            // step t has arrived when at most the later ones are on their way; the barrier says so for the other wavefronts' parts, and
            // that all are through with step t - 1, whose buffer the next copies go to
            if (t + STAGES - 1 <= steps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 2) * kLoads) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (t + STAGES - 1 < steps) issue(t + STAGES - 1);
            multiply(lds + here);
            here = next(here);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");             // this wavefront has read its part before it says so
        }
    } else if (steps > 0) {
        Stage<T, TRI, BI, THREADS> si;
        Stage<T, TRJ, BJ, THREADS> sj;
        si.init(base_i, a.ld_i, i0, r0);
        sj.init(base_j, a.ld_j, j0, r0);
        si.load(i_left, red);
        sj.load(j_left, red);
        si.store(lds);
        sj.store(lds + kJ);
        __syncthreads();
        for (int t = 0; t < steps; ++t) {
            const bool more = t + 1 < steps;
            if (more) {
                si.advance(a.ld_i);
                sj.advance(a.ld_j);
                const long long left = red - static_cast<long long>(t + 1) * BK;
                si.load(i_left, left);
                sj.load(j_left, left);
            }
            multiply(lds + (t & 1) * kBuffer);
            if (more) {
                char *next = lds + ((t + 1) & 1) * kBuffer;
                si.store(next);
                sj.store(next + kJ);
            }
            __syncthreads();
        }
    }
    // a lane has elements i .. i + 3 of output row j
    if constexpr (sizeof(T) == 2) {
        if (a.splits == 1) {
            // 16-bit results go through LDS, rows of the tile in 16-byte pieces: as 8-byte pieces straight from the lanes, 32 bytes of a row
            // at a time, 292 us instead of 270 (16 groups x 1024 rows x 2048 x 4096)
            constexpr int kPieces = BI / 8, kSpread = kPieces < 16 ? kPieces - 1 : 15;
            __syncthreads();                               // all have read the last step
#pragma unroll
            for (int fi = 0; fi < FI; ++fi) {
                const int i = wi + 16 * fi + 4 * (lane >> 4);
                float b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (PRODUCT == PRODUCT_ROWS && a.bias) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (i + k < i_left) b[k] = static_cast<float>(static_cast<const T *>(a.bias)[static_cast<long long>(group) * a.ni + i0 + i + k]);
                }
#pragma unroll
                for (int fj = 0; fj < FJ; ++fj) {
                    const int j = wj + 16 * fj + (lane & 15);
                    typedef T four_t __attribute__((ext_vector_type(4)));
                    four_t v;
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] = static_cast<T>(acc[fi][fj][k] + b[k]);
                    *reinterpret_cast<four_t *>(lds + j * BI * 2 + (((i >> 3) ^ (j & kSpread)) << 4) + (i & 4) * 2) = v;
                }
            }
            __syncthreads();
#pragma unroll 4
            for (int q = threadIdx.x; q < BJ * kPieces; q += THREADS) {
                const int j = q / kPieces, c = q % kPieces;
                const long long left = i_left - c * 8;
                if (j >= j_left || left <= 0) continue;
                union { u32x4 raw; T e[8]; } x;
                x.raw = *reinterpret_cast<const u32x4 *>(lds + j * BI * 2 + ((c ^ (j & kSpread)) << 4));
                T *dst = static_cast<T *>(a.out) + (out_row + j) * a.ld_out + i0 + c * 8;
                if (left >= 8) {
                    *reinterpret_cast<u32x4_a2 *>(dst) = x.raw;
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (k < left) dst[k] = x.e[k];
                }
            }
            return;
        }
    }
#pragma unroll
    for (int fi = 0; fi < FI; ++fi) {
        const int i = wi + 16 * fi + 4 * (lane >> 4);
        float b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (PRODUCT == PRODUCT_ROWS && a.bias && first_split) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (i + k < i_left) b[k] = static_cast<float>(static_cast<const T *>(a.bias)[static_cast<long long>(group) * a.ni + i0 + i + k]);
        }
#pragma unroll
        for (int fj = 0; fj < FJ; ++fj) {
            const int j = wj + 16 * fj + (lane & 15);
            if (j >= j_left || i >= i_left) continue;
            const long long at = (out_row + j) * a.ld_out + i0 + i;
            if (a.splits > 1) {
                float *dst = static_cast<float *>(a.out) + at;
                typedef float four_t __attribute__((ext_vector_type(4), aligned(4)));
                four_t v = acc[fi][fj];
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] += b[k];
                if (i + 4 <= i_left) *reinterpret_cast<four_t *>(dst) = v;
                else
                    for (int k = 0; k < 4; ++k)
                        if (i + k < i_left) dst[k] = v[k];
            } else {
                T *dst = static_cast<T *>(a.out) + at;
                typedef T four_t __attribute__((ext_vector_type(4), aligned(sizeof(T))));
                four_t v;
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = static_cast<T>(acc[fi][fj][k] + b[k]);
                if (i + 4 <= i_left) *reinterpret_cast<four_t *>(dst) = v;
                else
                    for (int k = 0; k < 4; ++k)
                        if (i + k < i_left) dst[k] = v[k];
            }
        }
    }
}

// out[e] = sum over the splits, in their order; two arrays in one launch: dW's parts and db's behind them
template <typename T>
__global__ __launch_bounds__(256) void oc_grouped_join_kernel(const float *parts_w, T *out_w, long long n_w, int splits_w, const float *parts_b, T *out_b,
                                                              long long n_b, int splits_b) {
    const long long n = n_w + n_b;
    for (long long e = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; e < n; e += static_cast<long long>(gridDim.x) * 256) {
        const bool w = e < n_w;
        const float *src = w ? parts_w + e : parts_b + (e - n_w);
        const long long stride = w ? n_w : n_b;
        const int splits = w ? splits_w : splits_b;
        float s = 0.0f;
#pragma unroll 8
        for (int k = 0; k < splits; ++k) s += src[k * stride];
        if (w) out_w[e] = static_cast<T>(s);
        else out_b[e - n_w] = static_cast<T>(s);
    }
}

template <typename K>
hipError_t launch_tiles(K kernel, int threads, int lds_bytes, long long blocks, const GroupedArgs &a, hipStream_t s) {
    if (blocks <= 0) return hipSuccess;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    if (lds_bytes > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds_bytes);
        if (e != hipSuccess) return e;
    }
    kernel<<<dim3(static_cast<unsigned>(blocks)), threads, lds_bytes, s>>>(a);
    return hipGetLastError();
}

template <typename T, int BI, int BJ, int WI, int WJ, bool TRI, bool TRJ, int PRODUCT, int RB, int STAGES>
hipError_t launch_product(const GroupedArgs &a, bool aligned, hipStream_t s) {
    constexpr int threads = (BI / WI) * (BJ / WJ) * 64;
    const long long tiles_i = (a.ni + BI - 1) / BI;
    long long blocks = (a.rows / BJ + std::min<long long>(a.groups, a.rows)) * tiles_i * a.splits;
    GroupedArgs b = a;
    if (PRODUCT == PRODUCT_WEIGHTS) {
        const long long weight_blocks = b.out ? tiles_i * ((a.nj + BJ - 1) / BJ) * a.groups * a.splits : 0;
        blocks = weight_blocks + (b.bias_out ? static_cast<long long>((a.nj + 63) / 64) * a.groups * a.bias_splits : 0);
        if (weight_blocks > 0x7fffffffLL) return hipErrorInvalidValue;
        b.weight_blocks = static_cast<int>(weight_blocks);
    }
    return aligned ? launch_tiles(oc_grouped_kernel<T, BI, BJ, WI, WJ, TRI, TRJ, PRODUCT, RB, STAGES>, threads, STAGES * (BI + BJ) * RB, blocks, b, s)
                   : launch_tiles(oc_grouped_kernel<T, BI, BJ, WI, WJ, TRI, TRJ, PRODUCT, 128, 0>, threads, 2 * (BI + BJ) * 128, blocks, b, s);
}

// Which tile.  Few rows a group: narrow in rows, many workgroups, the weights stream through (32 networks of 2048 x 2048, bf16: 32 rows
// each 42 us against 57 with 128 x 128, 48 rows 60 against 57; f32: 64 rows 188 against 283, 96 rows 266 against 270).  Enough work for
// most of the 256 CUs with 256 x 256 tiles (16-bit types): those (K = 2048, bf16: 180 tiles 55 us against 72 with 128 x 128, 128 tiles 54
// against 48).  Short output rows: 64 x 64, f32 also up to 192 (61 k rows of 192: 31 us against 36); so are fewer than 128 tiles of
// 128 x 128 (1000 x 1000 x 1000: bf16 14 us against 22, f32 33 against 38).  Else 128 x 128.
// Few tiles and a long reduction: the reduction is cut, too, into pieces of 256 or more (f32: 128), and a second launch adds the f32 parts up.
enum { TILE_64x32, TILE_64, TILE_128, TILE_256 };
struct RowsPlan { int tile, splits; };

RowsPlan rows_plan(int type, long long rows, int groups, int ni, int red) {
    RowsPlan p;
    const bool f32 = type == OC_F32;
    int bi = 64, bj = 64;
    if (rows <= (f32 ? 80LL : 32LL) * groups) { p.tile = TILE_64x32; bj = 32; }
    else if (!f32 && ni > 128 && (rows / 256 + groups / 2) * ((ni + 255) / 256) >= 150) { p.tile = TILE_256; bi = bj = 256; }
    else if (ni <= 64 || (f32 && ni <= 192)) p.tile = TILE_64;
    else if ((rows / 128 + std::min<long long>(groups, rows)) * ((ni + 127) / 128) < 128) p.tile = TILE_64;
    else { p.tile = TILE_128; bi = bj = 128; }
    const long long tiles = (rows / bj + std::min<long long>(groups, rows)) * ((ni + bi - 1) / bi);
    p.splits = tiles < 1 || tiles > 128 ? 1 : static_cast<int>(std::max<long long>(1, std::min<long long>({256 / tiles, red / (f32 ? 128 : 256), 16})));
    return p;
}

// f32 parts of a rows product, in elements
long long rows_parts(const RowsPlan &p, long long rows, int ni) { return p.splits > 1 ? p.splits * rows * ni : 0; }

template <typename T>
hipError_t launch_join(const float *parts_w, void *out_w, long long n_w, int splits_w, const float *parts_b, void *out_b, long long n_b, int splits_b, hipStream_t s) {
    if (n_w + n_b == 0) return hipSuccess;
    oc_grouped_join_kernel<T><<<dim3(static_cast<unsigned>(std::min<long long>(4096, (n_w + n_b + 255) / 256))), 256, 0, s>>>(
        parts_w, static_cast<T *>(out_w), n_w, splits_w, parts_b, static_cast<T *>(out_b), n_b, splits_b);
    return hipGetLastError();
}

// `parts`: rows_parts() floats
template <typename T, bool TRI, bool TRJ>
hipError_t launch_rows(GroupedArgs a, const RowsPlan &p, float *parts, bool aligned, hipStream_t s) {
    void *const out = a.out;
    a.splits = p.splits;
    if (p.splits > 1) a.out = parts;
    hipError_t e = hipSuccess;
    if (p.tile == TILE_64x32) e = launch_product<T, 64, 32, 16, 32, TRI, TRJ, PRODUCT_ROWS, 128, 3>(a, aligned, s);
    else if (p.tile == TILE_64) e = launch_product<T, 64, 64, 32, 32, TRI, TRJ, PRODUCT_ROWS, 64, 4>(a, aligned, s);
    else if (p.tile == TILE_128) e = launch_product<T, 128, 128, 64, 64, TRI, TRJ, PRODUCT_ROWS, 64, 4>(a, aligned, s);
    if constexpr (sizeof(T) == 2) {
        if (p.tile == TILE_256) e = launch_product<T, 256, 256, 128, 64, TRI, TRJ, PRODUCT_ROWS, 64, 5>(a, aligned, s);
    }
    if (e != hipSuccess || p.splits == 1) return e;
    return launch_join<T>(parts, out, a.rows * a.ni, p.splits, nullptr, nullptr, 0, 1, s);
}

struct WeightPlan { int tile, splits, bias_splits; };

// The tile of dW and into how many pieces its rows are cut so that there are workgroups for every CU (a piece has 128 rows or more).
// 256 x 256 where they fill the CUs without cutting (bf16, 8192 rows: 192 tiles 101 us against 44 with 128 x 128, 256 tiles 76 against 85).
WeightPlan weight_plan(int type, long long rows, int groups, int ni, int nj) {
    WeightPlan p;
    const auto tiles = [&](int b) { return static_cast<long long>((ni + b - 1) / b) * ((nj + b - 1) / b) * groups; };
    p.tile = type != OC_F32 && ni > 128 && nj > 128 && tiles(256) >= 224 ? 256 : ni <= 64 || nj <= 64 ? 64 : 128;
    const long long most = std::max<long long>(1, rows / groups / 128);
    const auto cut = [&](long long blocks) { return static_cast<int>(std::max<long long>(1, std::min<long long>({most, (512 + blocks - 1) / blocks, 64}))); };
    p.splits = tiles(p.tile) >= 224 ? 1 : cut(tiles(p.tile));
    const long long bias_blocks = static_cast<long long>((nj + 63) / 64) * groups;
    p.bias_splits = bias_blocks >= 512 ? 1 : cut(bias_blocks);
    return p;
}

template <typename T>
hipError_t launch_weights(const GroupedArgs &a, const WeightPlan &p, bool aligned, hipStream_t s) {
    if constexpr (sizeof(T) == 2) {
        if (p.tile == 256) return launch_product<T, 256, 256, 128, 64, true, true, PRODUCT_WEIGHTS, 64, 5>(a, aligned, s);
    }
    if (p.tile == 64) return launch_product<T, 64, 64, 32, 32, true, true, PRODUCT_WEIGHTS, 64, 4>(a, aligned, s);
    return launch_product<T, 128, 128, 64, 64, true, true, PRODUCT_WEIGHTS, 64, 4>(a, aligned, s);
}

bool aligned_rows(const void *p, long long ld, int type) {
    const long long size = type == OC_F32 ? 4 : 2;
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * size % 16 == 0 && ld * size * 256 < 0x80000000LL;
}

int check_grouped(const oc_grouped_linear_args *p, const char *who) {
    if (!p) return oc_internal_fail(OC_ERR_INVALID_ARG, "%s: NULL arguments", who);
    if (p->rows < 0 || p->groups < 1 || p->in_features < 1 || p->out_features < 1 || p->type < OC_F32 || p->type > OC_F16 || p->x_stride < p->in_features)
        return oc_internal_fail(OC_ERR_INVALID_ARG, "%s: rows %lld, groups %d, in_features %d, out_features %d, type %d, x_stride %lld", who,
                                static_cast<long long>(p->rows), p->groups, p->in_features, p->out_features, p->type, static_cast<long long>(p->x_stride));
    if (!p->d_weight || !p->d_offsets || (p->rows > 0 && !p->d_x))
        return oc_internal_fail(OC_ERR_INVALID_ARG, "%s: a required pointer is NULL", who);
    return OC_OK;
}

// What a backward pass computes and where its f32 parts lie in the workspace: dx's, then dW's, then db's, each only where that gradient is
// asked for and its sums are cut.  The workspace's size and its use both come from here.
struct BackwardPlan {
    RowsPlan rows;
    WeightPlan weights;
    long long n_w, n_b;                                    // elements to be joined, 0: written at once
    long long at_w, at_b, floats;                          // dW's parts, db's parts, the end
};

BackwardPlan backward_plan(const oc_grouped_linear_args *p, bool dx, bool dw, bool db) {
    const int K = p->in_features, N = p->out_features;
    BackwardPlan b;
    b.rows = rows_plan(p->type, p->rows, p->groups, K, N);
    b.weights = weight_plan(p->type, p->rows, p->groups, K, N);
    b.n_w = dw && b.weights.splits > 1 ? static_cast<long long>(p->groups) * N * K : 0;
    b.n_b = db && b.weights.bias_splits > 1 ? static_cast<long long>(p->groups) * N : 0;
    b.at_w = dx ? rows_parts(b.rows, p->rows, K) : 0;
    b.at_b = b.at_w + b.n_w * b.weights.splits;
    b.floats = b.at_b + b.n_b * b.weights.bias_splits;
    return b;
}

template <typename T>
hipError_t backward_type(const oc_grouped_linear_args *p, const BackwardPlan &plan, const GroupedArgs &base, float *parts, hipStream_t s) {
    hipError_t e = hipSuccess;
    const int K = p->in_features, N = p->out_features, V = p->type == OC_F32 ? 4 : 8;
    if (p->d_dx && p->rows > 0) {
        GroupedArgs a = base;
        a.I = p->d_weight; a.J = p->d_dy; a.out = p->d_dx;
        a.ld_i = K; a.ld_j = N; a.ld_out = K;
        a.ni = K; a.red = N;
        e = launch_rows<T, true, false>(a, plan.rows, parts, aligned_rows(p->d_weight, K, p->type) && aligned_rows(p->d_dy, N, p->type) && K % V == 0 && N % V == 0, s);
        if (e != hipSuccess) return e;
    }
    if (p->d_dweight || p->d_dbias) {
        GroupedArgs a = base;
        a.I = p->d_x; a.J = p->d_dy;
        a.ld_i = p->x_stride; a.ld_j = N; a.ld_out = K;
        a.ni = K; a.nj = N; a.splits = plan.weights.splits; a.bias_splits = plan.weights.bias_splits;
        a.out = plan.n_w ? static_cast<void *>(parts + plan.at_w) : p->d_dweight;
        a.bias_out = plan.n_b ? static_cast<void *>(parts + plan.at_b) : p->d_dbias;
        e = launch_weights<T>(a, plan.weights, aligned_rows(p->d_x, p->x_stride, p->type) && aligned_rows(p->d_dy, N, p->type) && K % V == 0 && N % V == 0, s);
        if (e == hipSuccess)
            e = launch_join<T>(parts + plan.at_w, p->d_dweight, plan.n_w, plan.weights.splits, parts + plan.at_b, p->d_dbias, plan.n_b, plan.weights.bias_splits, s);
    }
    return e;
}

}  // namespace

extern "C" int64_t oc_grouped_linear_workspace_bytes(const oc_grouped_linear_args *p, int backward) {
    if (check_grouped(p, "oc_grouped_linear_workspace_bytes") != OC_OK) return -1;
    long long floats;
    if (!backward) {
        floats = rows_parts(rows_plan(p->type, p->rows, p->groups, p->out_features, p->in_features), p->rows, p->out_features);
    } else {
        const bool any = p->d_dx || p->d_dweight || p->d_dbias;            // no output known yet: room for all of them
        floats = backward_plan(p, p->d_dx || !any, p->d_dweight || !any, p->d_dbias || !any).floats;
    }
    return floats * static_cast<long long>(sizeof(float));
}

extern "C" int oc_grouped_linear(const oc_grouped_linear_args *p, void *d_workspace, void *stream) {
    if (const int rc = check_grouped(p, "oc_grouped_linear")) return rc;
    if (p->rows == 0) return OC_OK;
    if (!p->d_y) return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_grouped_linear: d_y is NULL");
    const RowsPlan plan = rows_plan(p->type, p->rows, p->groups, p->out_features, p->in_features);
    if (plan.splits > 1 && (!d_workspace || reinterpret_cast<uintptr_t>(d_workspace) % 4))
        return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_grouped_linear: needs a workspace of %lld bytes",
                                static_cast<long long>(oc_grouped_linear_workspace_bytes(p, 0)));
    GroupedArgs a = {};
    a.I = p->d_weight; a.J = p->d_x; a.bias = p->d_bias; a.out = p->d_y; a.offsets = p->d_offsets;
    a.ld_i = p->in_features; a.ld_j = p->x_stride; a.ld_out = p->out_features;
    a.rows = p->rows; a.groups = p->groups; a.ni = p->out_features; a.red = p->in_features;
    a.offsets64 = p->offsets64 != 0;
    const int V = p->type == OC_F32 ? 4 : 8;
    const bool aligned = aligned_rows(p->d_weight, p->in_features, p->type) && aligned_rows(p->d_x, p->x_stride, p->type) && p->in_features % V == 0;
    const OcDeviceScope on_device(oc_device_of_pointer(p->d_y));
    hipStream_t s = static_cast<hipStream_t>(stream);
    float *parts = static_cast<float *>(d_workspace);
    const hipError_t e = p->type == OC_F32    ? launch_rows<float, false, false>(a, plan, parts, aligned, s)
                         : p->type == OC_BF16 ? launch_rows<__bf16, false, false>(a, plan, parts, aligned, s)
                                              : launch_rows<_Float16, false, false>(a, plan, parts, aligned, s);
    return e == hipSuccess ? OC_OK : oc_internal_fail(OC_ERR_HIP, "oc_grouped_linear: %s", hipGetErrorString(e));
}

extern "C" int oc_grouped_linear_backward(const oc_grouped_linear_args *p, void *d_workspace, void *stream) {
    if (const int rc = check_grouped(p, "oc_grouped_linear_backward")) return rc;
    if (p->rows > 0 && !p->d_dy) return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_grouped_linear_backward: d_dy is NULL");
    if (!p->d_dx && !p->d_dweight && !p->d_dbias) return OC_OK;
    const BackwardPlan plan = backward_plan(p, p->d_dx, p->d_dweight, p->d_dbias);
    if (plan.floats > 0 && (!d_workspace || reinterpret_cast<uintptr_t>(d_workspace) % 4))
        return oc_internal_fail(OC_ERR_INVALID_ARG, "oc_grouped_linear_backward: needs a workspace of %lld bytes", plan.floats * static_cast<long long>(sizeof(float)));
    GroupedArgs a = {};
    a.offsets = p->d_offsets; a.rows = p->rows; a.groups = p->groups; a.offsets64 = p->offsets64 != 0; a.splits = 1;
    const OcDeviceScope on_device(oc_device_of_pointer(p->d_weight));
    hipStream_t s = static_cast<hipStream_t>(stream);
    float *parts = static_cast<float *>(d_workspace);
    const hipError_t e = p->type == OC_F32    ? backward_type<float>(p, plan, a, parts, s)
                         : p->type == OC_BF16 ? backward_type<__bf16>(p, plan, a, parts, s)
                                              : backward_type<_Float16>(p, plan, a, parts, s);
    return e == hipSuccess ? OC_OK : oc_internal_fail(OC_ERR_HIP, "oc_grouped_linear_backward: %s", hipGetErrorString(e));
}
