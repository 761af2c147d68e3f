// Product of 8-bit rows with 8-bit weights, a power-of-two scale for each
// block of 128 along the summed axis:
//
//   c[i, j] = sum over blocks b of 2^(ea[i,b] + ew[j,b]) * sum over k in b of a[i,k] w[j,k]
//
// One v_mfma_scale_f32_16x16x128 multiplies a whole block of 16 x 16 and
// applies both scale bytes in the matrix unit, so scales cost no arithmetic.
// Any order of the 128 values within a block is right as long as both
// operands use the same one, and a block has one scale, so a lane takes two
// pieces of 16 bytes that make its wave's loads whole 64-byte runs.
#include "head_common.h"

namespace tkh {

constexpr int kTile = 16;  // rows of a fragment

template <int N> struct Int {
    static constexpr int value = N;
};

// Bytes [0, left) of a lane's half fragment stay, the others become zero:
// for the block in which k ends. `at` is the half's first byte in the block.
__device__ __forceinline__ v4i keep_bytes(v4i v, int at, int left) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const int n = left - at - 4 * d;
        v[d] &= n >= 4 ? -1 : n <= 0 ? 0 : (1 << (8 * n)) - 1;
    }
    return v;
}

__device__ __forceinline__ v8i join(v4i lo, v4i hi) {
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// A lane's 32 bytes of block b of a row: pieces g and g + 4 of its 8 (g =
// lane / 16). Pieces that begin beyond k are not read.
__device__ __forceinline__ v8i load_fragment(const uint8_t* row, int b, int g, int k) {
    const int at = b * kBlock + g * 16, left = k - b * kBlock;
    if (left >= kBlock) {
        return join(*(const v4i*)(row + at), *(const v4i*)(row + at + 64));
    }
    v4i lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
    if (g * 16 < left) lo = keep_bytes(*(const v4i*)(row + at), g * 16, left);
    if (g * 16 + 64 < left) hi = keep_bytes(*(const v4i*)(row + at + 64), g * 16 + 64, left);
    return join(lo, hi);
}

template <typename T>
__device__ __forceinline__ void store_c(void* c, int64_t at, float v) {
    ((typename Raw<T>::type*)c)[at] = Num<T>::put(v);
}

// The products of blocks [C, CPW), each with its byte of the scales.
template <int C, int CPW>
__device__ __forceinline__ v4f multiply_blocks(const v8i (&w)[CPW], const v8i (&a)[CPW], v4f acc,
                                               const int (&ws)[(CPW + 3) / 4], const int (&as)[(CPW + 3) / 4]) {
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[C], a[C], acc, 0, 0, C & 3, ws[C / 4], C & 3, as[C / 4]);
    if constexpr (C + 1 < CPW) return multiply_blocks<C + 1>(w, a, acc, ws, as);
    return acc;
}

// The plain kernel: a wave makes one 16 x 16 piece of c from device memory, four
// blocks under way at a time. It takes up to 4 rows of a of no more than 8192
// values that k_mm_stream does not take, where it is bound by the weights'
// arrival (1 x 3000 x 100008 62 us, 4.8 TB/s), and rows too far apart for the tiles' 32-bit offsets.
template <typename T> __global__ __launch_bounds__(256) void k_mm_plain(const tkh_matmul p) {
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int64_t n0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * kTile;
    const int64_t m0 = (int64_t)blockIdx.y * kTile;
    if (n0 >= p.n) return;
    const int64_t wn = n0 + r < p.n ? n0 + r : p.n - 1, am = m0 + r < p.m ? m0 + r : p.m - 1;
    const uint8_t* w = (const uint8_t*)p.w + wn * p.w_stride;
    const uint8_t* a = (const uint8_t*)p.a + am * p.a_stride;
    const uint8_t* ws = (const uint8_t*)p.w_scale + wn * p.w_scale_stride;
    const uint8_t* as = (const uint8_t*)p.a_scale + am * p.a_scale_stride;
    const int k = (int)p.k, blocks = (k + kBlock - 1) / kBlock;
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    int b = 0;
    for (; (b + 4) * kBlock <= k; b += 4) {
        v8i wf[4], af[4];
        int wq[1], aq[1];
        __builtin_memcpy(wq, ws + b, 4);
        __builtin_memcpy(aq, as + b, 4);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int at = (b + c) * kBlock + g * 16;
            wf[c] = join(*(const v4i*)(w + at), *(const v4i*)(w + at + 64));
            af[c] = join(*(const v4i*)(a + at), *(const v4i*)(a + at + 64));
        }
        acc = multiply_blocks<0>(wf, af, acc, wq, aq);
    }
    for (; b < blocks; ++b)
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            load_fragment(w, b, g, k), load_fragment(a, b, g, k), acc, 0, 0, 0, ws[b], 0, as[b]);
    // a lane holds 4 neighbours along n of row m0 + r
    if (m0 + r < p.m)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n0 + g * 4 + i < p.n)
                store_c<T>(p.c, (m0 + r) * p.c_stride + n0 + g * 4 + i, acc[i]);
}

// ---- the tiled kernel

// 16 bytes a lane from base + offset straight into shared memory at `to` +
// 16 * lane. It has no result registers; the wait is wait_tiles'.
__device__ __forceinline__ void load_to_lds(const uint8_t* base, uint32_t offset, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(to), "v"(offset), "s"(base)
                 : "memory");
}

// Every wave's loads into shared memory have landed and every wave has read
// what it read before.
__device__ __forceinline__ void wait_tiles() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

typedef __attribute__((address_space(3))) const uint8_t* LdsPtr;

// Rows of an operand, brought 8 at a time, a lane its piece of one of them.
// Two offsets a lane do for all: those of 8 whole rows, and those of the 8
// among which the operand ends, whose last row stands for the missing ones.
// 8 rows that are all beyond the end are read as the first: nothing uses them.
struct Rows {
    const uint8_t* base;
    int64_t stride;
    int rows;
    uint32_t whole, last;

    __device__ __forceinline__ Rows(const uint8_t* base, int64_t stride, int rows, int row, int at)
        : base(base), stride(stride), rows(rows),
          whole(__umul24(row, (unsigned)stride) + at),
          last(__umul24(min(row, (rows - 1) & 7), (unsigned)stride) + at) {}

    __device__ __forceinline__ void bring(int row0, int at, uint32_t back, uint32_t to) const {
        const int from = row0 < rows ? row0 : 0;
        load_to_lds(base + from * stride + at, (rows - from >= 8 ? whole : last) - back, to);
    }
};

// A workgroup makes BM x BN of c, each of its WM x WN waves FM x FN fragments.
// 256 x 256 is the largest tile whose sums (128 registers a lane) and fragments
// fit two waves a SIMD, and with 64 KB of operands for 2^23 products a step
// comes closest to keeping the matrix units fed. 4096 x 4096 x 128256 takes
// 1967 to 2091 us by the run, 2060 to 2190 TF/s, the matrix units busy half of
// the clocks at 1.98 GHz: a step's end waits for the next tiles, which come from
// L2 (operands are read 6.3 times from beyond it). 200 x 4096 x 128256 takes 169
// us, 3.2 TB/s of weights: one tile of m, so that nothing is shared between
// workgroups. Where k is short so is the whole: 24 x 1000 x 50257 14 us, 53 MB
// at 3.8 TB/s.
//
// Tiles of one block of k lie in shared memory twice over, one being read while the
// next arrives: a row takes 128 bytes, its 16-byte piece p at place p ^ (row
// & 7), which spreads the 16 rows that a fragment's lanes read over the
// banks.
template <typename T, int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(WM * WN * 64, WM * WN / 4) void k_mm_tile(const tkh_matmul p, int tiles_m, int tiles_n, int per) {
    constexpr int BM = WM * FM * kTile, BN = WN * FN * kTile, kStage = (BM + BN) * kBlock;
    constexpr int kTileWaves = WM * WN, kLanes = kTileWaves * 64;
    static_assert(BM % (8 * kTileWaves) == 0 && BN % (8 * kTileWaves) == 0, "a wave brings 8 rows at a time");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * kStage];
    __shared__ int scales[2][(BM + BN + kLanes - 1) / kLanes * kLanes];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(LdsPtr)smem;

    // a die's workgroups (every eighth) take neighbouring tiles: 4 along n by
    // all of m, so that they share what its L2 holds
    const int index = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (index >= tiles_m * tiles_n) return;
    const int group = index / (4 * tiles_m), in = index - group * 4 * tiles_m;
    const int wide = min(4, tiles_n - group * 4);
    const int64_t m0 = (int64_t)(in / wide) * BM, n0 = (int64_t)(group * 4 + in % wide) * BN;

    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int k = (int)p.k, blocks = (k + kBlock - 1) / kBlock;
    const int rows_m = (int)min((int64_t)BM, p.m - m0), rows_n = (int)min((int64_t)BN, p.n - n0);
    const uint8_t* abase = (const uint8_t*)p.a + m0 * p.a_stride;
    const uint8_t* wbase = (const uint8_t*)p.w + n0 * p.w_stride;

    // the pieces that this wave brings: 8 rows of 8 pieces at a time
    constexpr int LA = BM / 8 / kTileWaves, LW = BN / 8 / kTileWaves;
    const int piece = (lane & 7) ^ (lane >> 3);
    const Rows arows{abase, p.a_stride, rows_m, lane >> 3, piece * 16};
    const Rows wrows{wbase, p.w_stride, rows_n, lane >> 3, piece * 16};
    // piece i of block b, straight into a buffer
    const auto bring = [&](int b, int buf, int i) {
        // one that begins beyond k is read as the block's first, and masked
        // when it is used
        const uint32_t back = b * kBlock + piece * 16 < k ? 0 : piece * 16;
        const uint32_t to = lds0 + buf * kStage;
        if (i < LW)
            wrows.bring((wave * LW + i) * 8, b * kBlock, back, to + (wave * LW + i) * 1024);
        else
            arows.bring((wave * LA + i - LW) * 8, b * kBlock, back, to + BN * kBlock + (wave * LA + i - LW) * 1024);
    };

    // Scales come four blocks at a time, a lane bringing those of one row
    // through a register into shared memory, from where every wave takes its
    // own: in registers they would be there four times over.
    // They are asked for in every step, wanted or not: a load under a branch
    // would be waited for at its end.
    constexpr int LS = (BM + BN + kLanes - 1) / kLanes;
    static_assert(BN % kLanes == 0 || LS == 1, "a wave's rows are of one operand");
    const bool short_row = blocks < 4;
    uint32_t sat[LS];
    const uint8_t* sbase[LS];
    int arriving[LS], sa[FM], sw[FN];
#pragma unroll
    for (int i = 0; i < LS; ++i) {
        const bool of_w = i * kLanes + wave * 64 < BN;
        const int row = i * kLanes + (int)threadIdx.x;
        sbase[i] = of_w ? (const uint8_t*)p.w_scale + n0 * p.w_scale_stride
                        : (const uint8_t*)p.a_scale + m0 * p.a_scale_stride;
        sat[i] = __umul24(of_w ? min(row, rows_n - 1) : min(row - BN, rows_m - 1),
                          (unsigned)(of_w ? p.w_scale_stride : p.a_scale_stride));
    }
    const auto bring_scales = [&](int quad) {
        // where a row ends within these four, its last four
#pragma unroll
        for (int i = 0; i < LS; ++i) {
            const uint8_t* from = short_row ? (const uint8_t*)p.w : sbase[i] + min(4 * quad, blocks - 4);
            __builtin_memcpy(&arriving[i], from + (short_row ? 0 : sat[i]), 4);
        }
    };
    const auto place_scales = [&](int quad) {
#pragma unroll
        for (int i = 0; i < LS; ++i) {
            asm volatile("" : "+v"(arriving[i]));  // waited for here, before other loads are under way
            // a short row's are all there from the start, and stay
            scales[short_row ? 1 : quad & 1][i * kLanes + threadIdx.x] =
                (int)((uint32_t)arriving[i] >> (8 * max(0, 4 * quad + 4 - blocks) & 31));
        }
    };
    const auto read_scales = [&](int b) {
        const uint8_t* at = (const uint8_t*)scales[b / 4 & 1] + (b & 3);
#pragma unroll
        for (int j = 0; j < FM; ++j) sa[j] = at[(BN + (wm * FM + j) * kTile + r) * 4];
#pragma unroll
        for (int i = 0; i < FN; ++i) sw[i] = at[((wn * FN + i) * kTile + r) * 4];
    };

    v4f acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

    const int swz0 = (g ^ (r & 7)) * 16, swz1 = ((g + 4) ^ (r & 7)) * 16;
    // `left`: how many of the block's values count, where it is the last
    const auto fragment = [&](auto part, uint32_t rows, int row, int left) {
        const LdsPtr at = (LdsPtr)(uintptr_t)(rows + row * kBlock + r * kBlock);
        v4i lo = *(__attribute__((address_space(3))) const v4i*)(at + swz0);
        v4i hi = *(__attribute__((address_space(3))) const v4i*)(at + swz1);
        if (decltype(part)::value) {
            lo = keep_bytes(lo, g * 16, left);
            hi = keep_bytes(hi, g * 16 + 64, left);
        }
        return join(lo, hi);
    };
    v8i fa[FM], fw;
    const auto read_a = [&](auto part, int b, int j) {
        fa[j] = fragment(part, lds0 + (b & 1) * kStage + BN * kBlock, (wm * FM + j) * kTile, k - b * kBlock);
    };
    const auto read_w = [&](auto part, int b, int i) {
        return fragment(part, lds0 + (b & 1) * kStage, (wn * FN + i) * kTile, k - b * kBlock);
    };
    const auto product = [&](int i, int j) {
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            fw, fa[j], acc[i][j], 0, 0, 0, sw[i], 0, sa[j]);
    };
    // The products of the fragments [0, last) of w. The next fragment arrives
    // behind this one's products; held to this order, two of them are all
    // that lie in registers.
    // The loads of block `then` are issued a few at a time between the
    // products of the first fragments: a wave waits while the address unit
    // takes a load (16 clocks), and would stand still through all of them.
    constexpr int kSpread = FN / 2, kEach = (LA + LW + kSpread - 1) / kSpread;
    const auto products = [&](auto part, int b, auto last, int then) {
#pragma unroll
        for (int i = 0; i < decltype(last)::value; ++i) {
            v8i next = fw;
            if (i + 1 < FN) next = read_w(part, b, i + 1);
            if (!decltype(part)::value)
#pragma unroll
                for (int q = i * kEach; q < (i + 1) * kEach && q < LA + LW; ++q) bring(then, (b + 1) & 1, q);
#pragma unroll
            for (int j = 0; j < FM; ++j) product(i, j);
            __builtin_amdgcn_sched_barrier(0);
            fw = next;
        }
    };
    const int whole = k / kBlock;
#pragma unroll
    for (int i = 0; i < LA + LW; ++i) bring(0, 0, i);
    bring_scales(0);
    place_scales(0);
    if (short_row) {
#pragma unroll
        for (int i = 0; i < LS; ++i) {
            int v = 0;
            for (int b = 0; b < blocks; ++b) v |= (int)sbase[i][sat[i] + b] << (8 * b);
            scales[0][i * kLanes + threadIdx.x] = v;
        }
    }
    wait_tiles();
    if (rows_m <= wm * FM * kTile) {
        // None of this wave's rows is there: it brings what is of its part of
        // the tiles, between the same waits as the others. Neighbouring waves
        // have the same rows and run on SIMDs of their own, so that the others
        // get the matrix units and the address unit for themselves: 777 x
        // 2560 x 200019 478 us instead of 562 (in turn), 300 x 4096 x 128256 240 / 276.
        bring_scales(0);
        if (whole) {
#pragma unroll 1
            for (int b = 0; b < whole; ++b) {
#pragma unroll
                for (int i = 0; i < LA + LW; ++i)
                    if (i < LW || (wave * LA + i - LW) * 8 < rows_m) bring(min(b + 1, blocks - 1), (b + 1) & 1, i);
                wait_tiles();
                if (b + 1 < whole) {
                    place_scales((b + 2) / 4);
                    bring_scales((b + 3) / 4);
                }
            }
        }
        if (whole < blocks) wait_tiles();
        return;
    }
    read_scales(0);
    bring_scales(0);
    if (whole) {
#pragma unroll
        for (int j = 0; j < FM; ++j) read_a(Int<0>{}, 0, j);
        fw = read_w(Int<0>{}, 0, 0);
#pragma unroll 1
        for (int b = 0; b + 1 < whole; ++b) {
            products(Int<0>{}, b, Int<FN - 1>{}, b + 1);
            // everything of block b has been read and the next one is there:
            // its first fragments are read behind the last products of this
            wait_tiles();
            place_scales((b + 2) / 4);
            bring_scales((b + 3) / 4);
            const v8i first = read_w(Int<0>{}, b + 1, 0);
#pragma unroll
            for (int j = 0; j < FM; ++j) {
                product(FN - 1, j);
                __builtin_amdgcn_sched_barrier(0);  // into the same registers
                read_a(Int<0>{}, b + 1, j);
            }
            fw = first;
            read_scales(b + 1);
        }
        // where none is left, a block that nobody reads
        products(Int<0>{}, whole - 1, Int<FN>{}, min(whole, blocks - 1));
        wait_tiles();
    }
    if (whole < blocks) {
        if (whole) read_scales(whole);
#pragma unroll
        for (int j = 0; j < FM; ++j) read_a(Int<1>{}, whole, j);
        fw = read_w(Int<1>{}, whole, 0);
        products(Int<1>{}, whole, Int<FN>{}, 0);
        wait_tiles();
    }

    typedef typename Raw<T>::type R;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
        const int m = (wm * FM + j) * kTile + r;
        if (m >= rows_m) continue;
        R* c = (R*)p.c + (m0 + m) * p.c_stride + n0;
#pragma unroll
        for (int i = 0; i < FN; ++i) {
            const int n = (wn * FN + i) * kTile + g * 4;
            R v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = Num<T>::put(acc[i][j][q]);
            if (n + 4 <= rows_n) {
                store_pack(c + n, v);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (n + q < rows_n) c[n + q] = v[q];
            }
        }
    }
}

template <typename T, int WM, int WN, int FM, int FN>
static int tiled(const tkh_matmul& p, void* stream) {
    const int tiles_m = (int)ceil_div(p.m, WM * FM * kTile), tiles_n = (int)ceil_div(p.n, WN * FN * kTile);
    const int per = (int)ceil_div((int64_t)tiles_m * tiles_n, 8);
    return launch("k_mm_tile", k_mm_tile<T, WM, WN, FM, FN>, dim3(per * 8), dim3(WM * WN * 64), 0, stream, p,
                  tiles_m, tiles_n, per);
}

// ---- few rows of a

// Up to 16 MT rows of a, against which w streams through registers once. The
// NW waves of a workgroup share k, which is CPW blocks for each, and keep their blocks of a
// in registers for good; the weights of the next NT x 16 rows are on their way
// while these are multiplied. The waves' parts of c meet in shared memory,
// added in the waves' order. Bound by memory: a byte of w is read once.
// Measured: 1 x 4096 x 151669 105 us, 627 MB read at 5.9 TB/s; 32 x 4096 x
// 128256 107 us, 5.0 TB/s.
// Workgroups take neighbouring rows in turn: a stretch of its own for each was
// 10% slower.
template <typename T, int NW, int MT, int CPW, int NT>
__global__ __launch_bounds__(NW * 64, NW / 4) void k_mm_stream(const tkh_matmul p, int fragments) {
    static_assert(CPW <= 4, "a row's scales are in one register");
    __shared__ v4f parts[2][NW][NT * MT][64];
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int b0 = wave * CPW;
    // fragment i of a turn; `fragments` or more: none
    const auto fragment_of = [&](int turn, int i) {
        return (turn * (int)gridDim.x + (int)blockIdx.x) * NT + i;
    };

    // this wave's blocks of a row, and their scales, a byte each
    const auto load = [&](v8i (&to)[CPW], const uint8_t* row) {
#pragma unroll
        for (int c = 0; c < CPW; ++c) {
            const uint8_t* at = row + (b0 + c) * kBlock + g * 16;
            to[c] = join(*(const v4i*)at, *(const v4i*)(at + 64));
        }
    };
    const auto load_scales = [&](int (&to)[1], const uint8_t* row) {
        to[0] = 0;
        __builtin_memcpy(to, row + b0, CPW);
    };

    v8i a[MT][CPW];
    int as[MT][1];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const int64_t m = min((int64_t)(j * kTile + r), p.m - 1);
        load(a[j], (const uint8_t*)p.a + m * p.a_stride);
        load_scales(as[j], (const uint8_t*)p.a_scale + m * p.a_scale_stride);
    }
    v8i w[NT][CPW];
    int ws[NT][1];
    const auto load_tile = [&](int turn) {
        // without a branch: past the end, the last row
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int64_t n = min((int64_t)fragment_of(turn, i) * kTile + r, p.n - 1);
            load(w[i], (const uint8_t*)p.w + n * p.w_stride);
            load_scales(ws[i], (const uint8_t*)p.w_scale + n * p.w_scale_stride);
        }
    };
    load_tile(0);
    for (int turn = 0; fragment_of(turn, 0) < fragments; ++turn) {
        v8i now[NT][CPW];
        int ns[NT][1];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
#pragma unroll
            for (int c = 0; c < CPW; ++c) now[i][c] = w[i][c];
            ns[i][0] = ws[i][0];
        }
        load_tile(turn + 1);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < MT; ++j)
                parts[turn & 1][wave][i * MT + j][lane] =
                    multiply_blocks<0>(now[i], a[j], v4f{0.0f, 0.0f, 0.0f, 0.0f}, ns[i], as[j]);
        // the other turn's parts have all been read before this barrier
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int q = 0; q < (NT * MT + NW - 1) / NW; ++q) {
            const int f = q * NW + wave, at = fragment_of(turn, f / MT);
            if (f >= NT * MT || at >= fragments) break;
            v4f sum = parts[turn & 1][0][f][lane];
#pragma unroll
            for (int v = 1; v < NW; ++v) sum += parts[turn & 1][v][f][lane];
            const int64_t n = (int64_t)at * kTile + g * 4;
            const int m = f % MT * kTile + r;
            if (m >= p.m) continue;
            typedef typename Raw<T>::type R;
            R* c = (R*)p.c + m * p.c_stride + n;
            R v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = Num<T>::put(sum[e]);
            if (n + 4 <= p.n) {
                store_pack(c, v);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < p.n) c[e] = v[e];
            }
        }
    }
}

template <typename T, int NW, int MT, int CPW> static int streamed(const tkh_matmul& p, void* stream) {
    // what is on its way and what is multiplied take 8 registers a fragment
    // each, beside those of a, of 256 (128 with 16 waves); the parts of c take
    // 2 KB a wave for each 256
    constexpr int kHeld = NW > 8 || MT * CPW > 8 ? 4 : 8, kMost = 4 / MT,
                  NT = CPW * kMost <= kHeld ? kMost : kHeld / CPW;
    const int fragments = (int)ceil_div(p.n, kTile), tiles = (int)ceil_div(fragments, NT);
    // what takes up to 128 registers fits a compute unit twice
    const int most = NW == 8 && CPW <= 2 ? 512 : 256;
    return launch("k_mm_stream", k_mm_stream<T, NW, MT, CPW, NT>, dim3((unsigned)(tiles < most ? tiles : most)),
                  dim3(NW * 64), 0, stream, p, fragments);
}

// Eight waves share k: a block each, or 2, 3 or 4.
template <typename T, int MT> static int streamed_by(const tkh_matmul& p, void* stream) {
    switch (p.k / (8 * kBlock)) {
    case 1: return streamed<T, 8, MT, 1>(p, stream);
    case 2: return streamed<T, 8, MT, 2>(p, stream);
    case 3: return streamed<T, 8, MT, 3>(p, stream);
    default: return streamed<T, 8, MT, 4>(p, stream);
    }
}

// Which kernel: by the rows of a, then by k. Times in us.
// Streamed or tiled, where k fills the waves evenly:
//   16 x 4096 x 128256 100 / 118, 32 x 4096 107 / 118, 64 x 4096 130 / 130,
//   40 x 2048 x 100008 47 / 50, with 16 waves 16 x 6144 x 50257 60 / 73 and
//   16 x 8192 82 / 101;
// where it does not, and every load asks whether it is beyond k:
//   24 x 1000 x 50257 18 / 14, 24 x 3000 x 100008 90 / 75, 8 x 3000 81 / 73,
//   with 16 waves 16 x 5000 x 50257 60 / 64.
// Streamed or plain, up to 4 rows: 1 x 2048 x 100008 40 / 40, 4 x 2048 41 / 44,
// 1 x 4096 x 151669 107 / 124, 1 x 6144 x 50257 54 / 70, 1 x 8192 74 / 111.
// Plain or tiled: 1 x 3000 x 100008 62 / 73, 4 x 3000 67 / 73, 1 x 7168 x 50257
// 80 / 84, 1 x 12288 160 / 153, 1 x 16384 x 128256 455 / 391. A few rows of a
// cost the plain kernel little, and its waves wait for nobody; long rows give
// the tiles time to make up for their start.
// Tiles of 128 x 128, two workgroups to a compute unit, or of 256 x 256, one:
// 100 x 1000 x 100008 30 / 34, 112 x 4862 x 128256 151 / 154, 140 x 4096 x
// 128256 209 / 155.
template <typename T> static int matmul_as(const tkh_matmul& p, void* stream) {
    const int64_t blocks = ceil_div(p.k, kBlock);
    if (p.k % (8 * kBlock) == 0 && blocks <= 32 && p.m <= 64)
        return p.m <= 16   ? streamed_by<T, 1>(p, stream)
               : p.m <= 32 ? streamed_by<T, 2>(p, stream)
                           : streamed_by<T, 4>(p, stream);
    if (p.m <= 16 && p.k == 16 * 3 * kBlock) return streamed<T, 16, 1, 3>(p, stream);
    if (p.m <= 16 && p.k == 16 * 4 * kBlock) return streamed<T, 16, 1, 4>(p, stream);
    // the tiles' offsets are of 32 bits
    if ((p.m > 4 || blocks > 64) && p.a_stride < (1 << 23) && p.w_stride < (1 << 23) &&
        p.a_scale_stride < (1 << 23) && p.w_scale_stride < (1 << 23))
        return p.m > 128 ? tiled<T, 4, 2, 4, 8>(p, stream) : tiled<T, 2, 2, 4, 4>(p, stream);
    const dim3 grid((unsigned)ceil_div(p.n, 4 * kTile), (unsigned)ceil_div(p.m, kTile));
    return launch("k_mm_plain", k_mm_plain<T>, grid, dim3(256), 0, stream, p);
}

}  // namespace tkh

extern "C" int tk_head_matmul(const tkh_matmul* args, void* stream) {
    using namespace tkh;
    if (!args) return fail(TKH_E_INVALID_ARG, "no arguments");
    const tkh_matmul& p = *args;
    // each kernel's workgroups fit a launch: the fewest rows a workgroup takes
    // are 64 of w, or 128 of both
    if (p.m < 0 || p.n < 0 || p.k < 1 || p.k > (1 << 24) || p.n > (1 << 30) - 64 || p.m > 1000000 ||
        ceil_div(p.m, 128) * ceil_div(p.n, 128) > (1 << 23))
        return fail(TKH_E_SHAPE, "m %lld, n %lld, k %lld", (long long)p.m, (long long)p.n, (long long)p.k);
    if (p.out_dtype != TKH_BF16 && p.out_dtype != TKH_F16)
        return fail(TKH_E_UNSUPPORTED, "out dtype %d", p.out_dtype);
    if (p.m == 0 || p.n == 0) return TKH_OK;
    if (!p.a || !p.a_scale || !p.w || !p.w_scale || !p.c) return fail(TKH_E_INVALID_ARG, "a null pointer");
    // a single row's stride is stepped over by no kernel
    if ((p.m > 1 && p.a_stride % 16) || (p.n > 1 && p.w_stride % 16) || (uintptr_t)p.a % 16 || (uintptr_t)p.w % 16)
        return fail(TKH_E_SHAPE, "rows of a and w are 16-byte aligned");
    const int64_t blocks = ceil_div(p.k, kBlock);
    if ((p.m > 1 && (p.a_stride < p.k || p.a_scale_stride < blocks)) ||
        (p.n > 1 && (p.w_stride < p.k || p.w_scale_stride < blocks)) || (p.m > 1 && p.c_stride < p.n))
        return fail(TKH_E_SHAPE, "a row stride is shorter than its row");
    DeviceScope scope(p.device);
    if (scope.status() != TKH_OK) return scope.status();
    if (p.out_dtype == TKH_BF16) return matmul_as<__hip_bfloat16>(p, stream);
    return matmul_as<__half>(p, stream);
}
