// One token a row by temperature, top-k, top-p and min-p from a given random
// number.
//
// A token's weight 2^((x - max) * log2(e) / T) is taken as a whole number of
// 2^-40, so every sum is exact and no result depends on the order in which
// lanes, waves or workgroups add: a row gives the same token in any batch.
// Tokens are compared by a 32-bit key that orders as the logits do; 0 is a
// token that the row may not draw.
//
// What is asked of a row is mostly about its largest logits. k_groups reads
// the logits once and keeps the largest of every group of 64 bytes (16 or 32
// tokens). The n-th largest of those is at most the n-th largest logit, so
// k_pick finds it among them and reads again only the groups that reach it:
// for top-k with n = k that is all that a token needs. Without a top-k the
// weight of all tokens counts: k_masses sums it, a wave a run of groups, and
// k_pick then looks among the 1,024 largest for the set that top-p leaves.
// Wider sets are left to k_wide_bins, k_wide_list and k_rest. A top-k of over
// 1,024 and rows of too many equal logits take sample_row, which reads such a
// row as often as it takes.
#include "head_common.h"

#include <math.h>

namespace tkh {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
typedef unsigned long long u64;

__device__ __forceinline__ uint32_t key_of(float x) {
    // -0 orders as 0, NaN and -inf are never drawn
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t k = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return x > -INFINITY ? k : 0u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// One row and what is asked of it.
struct RowParams {
    float step, top_p, min_p, u;
    uint32_t top_k;  // 0: no limit
};

__device__ __forceinline__ RowParams params_of(const tkh_sample& p, int64_t row) {
    RowParams r;
    const float t = p.temperature ? p.temperature[row] : p.temperature_value;
    const int32_t k = p.top_k ? p.top_k[row] : p.top_k_value;
    const bool greedy = !(t > 0.0f);
    r.top_k = greedy ? 1u : k > 0 ? (uint32_t)k : 0u;
    r.step = 1.44269504088896340736f / (greedy ? 1.0f : t);
    r.top_p = p.top_p ? p.top_p[row] : p.top_p_value;
    if (!(r.top_p < 1.0f)) r.top_p = 1.0f;
    r.min_p = p.min_p ? p.min_p[row] : p.min_p_value;
    r.min_p = r.min_p > 0.0f ? fminf(r.min_p, 1.0f) : 0.0f;
    r.u = p.u[row];
    return r;
}

__device__ __forceinline__ float weight_of(float x, float top, float step) {
    // rounded after the difference, the product and the power, as elementary
    // operations on floats are; 0 for the NaN of an overflow times a step of 0
    return x == top ? 1.0f : fmaxf(__builtin_amdgcn_exp2f((x - top) * step), 0.0f);
}
// floor(weight * 2^40) as two halves of 20 bits: a float's product with a
// power of two and its fraction are exact.
struct Halves {
    uint32_t high, low;
};
__device__ __forceinline__ Halves halves_of(float weight) {
    const float f = weight * 0x1p20f;
    return {(uint32_t)f, (uint32_t)(__builtin_amdgcn_fractf(f) * 0x1p20f)};
}
__device__ __forceinline__ u64 mass_of(float weight) {
    const Halves h = halves_of(weight);
    return ((u64)h.high << 20) + h.low;
}

// The first of its tokens that a row has ceil(part of a mass) before.
__device__ __forceinline__ u64 part_of(float top_p, u64 mass) {
    const double part = ceil((double)top_p * (double)mass);
    return part >= 1.0 ? (u64)part : 1;
}
__device__ __forceinline__ u64 target_of(float u, u64 mass) {
    const double at = floor((double)u * (double)mass);
    const u64 t = at > 0.0 ? (u64)at : 0;  // a NaN draws the first
    return t < mass ? t : mass - 1;
}
// ln(mass / total); near one it is taken of what is missing to it.
__device__ __forceinline__ float logprob_of(u64 mass, u64 total) {
    const float rest = (float)(total - mass) / (float)total;
    return rest < 0.5f ? log1pf(-rest) : logf((float)mass / (float)total);
}

template <typename T> struct Row {
    typedef typename Raw<T>::type R;
    static constexpr int kVec = 16 / sizeof(R);
    const R* x;
    const uint32_t* allowed;
    int v;

    __device__ __forceinline__ Row(const tkh_sample& p, int64_t row)
        : x((const R*)p.logits + row * p.logits_stride),
          allowed(p.allowed ? p.allowed + row * p.allowed_stride : nullptr),
          v((int)p.vocab) {}

    __device__ __forceinline__ uint32_t bit(int i) const {
        return allowed ? (allowed[i >> 5] >> (i & 31)) & 1 : 1;
    }
    __device__ __forceinline__ uint32_t key(int i) const {
        if (!bit(i)) return 0;
        return key_of(Num<T>::get(x[i]));
    }

    // The mask bits of the tokens [i, i + kVec), the first in the lowest.
    __device__ __forceinline__ u64 bits(int i) const {
        if (!allowed) return ~0ull;
        return (((u64)allowed[(i + kVec - 1) >> 5] << 32) | allowed[i >> 5]) >> (i & 31);
    }

    // f(index, key) for the tokens [lo, hi), shared among n lanes; 64 or 32
    // bytes of a lane are under way at a time
    template <typename F> __device__ __forceinline__ void each(int lo, int hi, int lane, int n, F f) const {
        constexpr int kDeep = 16 / kVec;
        int i = lo + lane * kVec;
        for (; i + (kDeep - 1) * n * kVec + kVec <= hi; i += kDeep * n * kVec) {
            R a[kDeep][kVec];
            u64 b[kDeep];
#pragma unroll
            for (int q = 0; q < kDeep; ++q) {
                load_pack(a[q], x + i + q * n * kVec);
                b[q] = bits(i + q * n * kVec);
            }
#pragma unroll
            for (int q = 0; q < kDeep; ++q)
#pragma unroll
                for (int j = 0; j < kVec; ++j)
                    f(i + q * n * kVec + j, (b[q] >> j) & 1 ? key_of(Num<T>::get(a[q][j])) : 0u);
        }
        for (; i + kVec <= hi; i += n * kVec) {
            R a[kVec];
            load_pack(a, x + i);
            const u64 b = bits(i);
#pragma unroll
            for (int j = 0; j < kVec; ++j)
                f(i + j, (b >> j) & 1 ? key_of(Num<T>::get(a[j])) : 0u);
        }
        for (int j = 0; j < kVec; ++j)
            if (i + j < hi) f(i + j, key(i + j));
    }
};

// Sums and prefixes over a workgroup.
constexpr int kList = 2048;  // candidates at most
constexpr int kBins = 2048;  // of a fiftieth of an octave of weight
constexpr int kLastBin = 2001;  // beyond 40 octaves nothing has a mass

struct Shared {
    u64 list[kList];  // key << 32 | ~index: larger first, then lower index
    u64 mass[kList];  // of the list's tokens
    u64 bins[kBins];
    u64 parts[256];   // of the vocabulary
    u64 waves[2][kWaves];
    u64 found[2], end[2];
    uint32_t groups[kList];
    uint32_t tops[kWaves];
    uint16_t members[kList];
    uint32_t n[5];    // lengths: groups, list, members of three turns
};

struct Team {
    Shared& m;
    int turn = 0;
};

// The neighbour's value `Ctrl` names, 0 where there is none or the row of 16
// lanes is not in `Rows`.
template <int Ctrl, int Rows> __device__ __forceinline__ u64 from_lane(u64 v) {
    const int lo = __builtin_amdgcn_update_dpp(0, (int)v, Ctrl, Rows, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), Ctrl, Rows, 0xf, false);
    return (u64)(uint32_t)hi << 32 | (uint32_t)lo;
}
// The sum of a wave's lanes up to this one: within rows of 16 by shifts of 1,
// 2, 4 and 8, then the rows' last lanes into the rows behind.
__device__ __forceinline__ u64 scan64(u64 v) {
    v += from_lane<0x111, 0xf>(v);
    v += from_lane<0x112, 0xf>(v);
    v += from_lane<0x114, 0xf>(v);
    v += from_lane<0x118, 0xf>(v);
    v += from_lane<0x142, 0xa>(v);
    v += from_lane<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ u64 add64(u64 v) {
    v = scan64(v);
    return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), 63) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
// The workgroup's total, in every lane, and in `before` what the waves ahead
// of this one have. Every lane adds the sixteen sums up: shorter than a
// second exchange.
__device__ __forceinline__ u64 block_sum(Team& t, u64 v, u64* before = nullptr) {
    Shared& s = t.m;
    v = add64(v);
    // two places in turn, so that one barrier is enough
    u64* waves = s.waves[t.turn & 1];
    ++t.turn;
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    u64 sum = 0, ahead = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w == (int)(threadIdx.x >> 6)) ahead = sum;
        sum += waves[w];
    }
    if (before) *before = ahead;
    return sum;
}

// The first token at which the running sum of value(index, key) over [lo, hi)
// passes `target`, which is below the sum. The range is narrowed to one of
// the waves' sixteen parts until a token a lane is left.
template <typename T, typename F>
__device__ __forceinline__ int find(Team& t, const Row<T>& row, int lo, int hi, u64 target, F value) {
    Shared& s = t.m;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    while (hi - lo > kThreads) {
        const int part = (hi - lo + kWaves - 1) / kWaves;
        const int a = min(hi, lo + wave * part), b = min(hi, a + part);
        u64 mine = 0;
        row.each(a, b, lane, 64, [&](int i, uint32_t key) { mine += value(i, key); });
        block_sum(t, mine);
        const u64* waves = s.waves[(t.turn & 1) ^ 1];
        int w = 0;
        for (; w + 1 < kWaves && waves[w] <= target; ++w) target -= waves[w];
        lo = min(hi, lo + w * part);
        hi = min(hi, lo + part);
    }
    const int i = lo + (int)threadIdx.x;
    const u64 mine = i < hi ? value(i, row.key(i)) : 0;
    u64 before;
    block_sum(t, mine, &before);
    before += scan64(mine) - mine;
    if (mine && before <= target && target < before + mine) s.found[0] = (u64)i;
    __syncthreads();
    const int at = (int)s.found[0];
    __syncthreads();
    return at;
}

// The largest key at which the sum of value(key) over the tokens of at least
// that key reaches `need`, and the sum over larger keys; key 1 where even
// all tokens' does not. Four rounds of 8 bits over the whole row.
template <typename T, typename F>
__device__ __forceinline__ uint32_t reach(Team& t, const Row<T>& row, u64 need, u64* above, F value) {
    Shared& s = t.m;
    uint32_t prefix = 0;
    u64 before = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < 256) s.bins[threadIdx.x] = 0;
        __syncthreads();
        row.each(0, row.v, threadIdx.x, kThreads, [&](int, uint32_t key) {
            if (key && (shift == 24 || key >> (shift + 8) == prefix)) {
                const u64 n = value(key);
                if (n) atomicAdd(&s.bins[(key >> shift) & 255], n);
            }
        });
        __syncthreads();
        if (threadIdx.x == 0) {
            int bin = 255;
            for (; bin > 0 && before + s.bins[bin] < need; --bin) before += s.bins[bin];
            s.found[0] = (u64)bin;
            s.found[1] = before;
        }
        __syncthreads();
        prefix = prefix << 8 | (uint32_t)s.found[0];
        before = s.found[1];
    }
    *above = before;
    return prefix ? prefix : 1;
}

// The general path: a workgroup takes a row and reads it from memory for
// every question that it asks.
template <typename T> __device__ __forceinline__ void sample_row(Shared& s, const tkh_sample& p, int64_t r) {
    __syncthreads();
    Team t{s};
    const Row<T> row(p, r);
    const RowParams q = params_of(p, r);
    uint32_t top_key = 0;
    u64 count = 0;
    row.each(0, row.v, threadIdx.x, kThreads, [&](int, uint32_t key) {
        top_key = max(top_key, key);
        count += key != 0;
    });
#pragma unroll
    for (int d = 32; d; d >>= 1) top_key = max(top_key, __shfl_xor(top_key, d, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.tops[threadIdx.x >> 6] = top_key;
    count = block_sum(t, count);
    for (int w = 0; w < kWaves; ++w) top_key = max(top_key, s.tops[w]);
    if (!top_key) {
        if (threadIdx.x == 0) {
            p.ids[r] = -1;
            if (p.logprob) p.logprob[r] = -INFINITY;
        }
        return;
    }
    const float top = value_of(top_key);
    const auto mass = [&](uint32_t key) {
        return key ? mass_of(weight_of(value_of(key), top, q.step)) : 0ull;
    };

    // what stays: larger keys than `edge`, and the tokens of that key up to
    // the index `last`
    uint32_t edge = 1;
    u64 ties = ~0ull, above = 0;
    if (q.top_k && q.top_k < count) {
        edge = reach(t, row, (u64)q.top_k, &above, [](uint32_t) { return 1ull; });
        ties = q.top_k - above;
    }
    if (q.top_p < 1.0f) {
        u64 mine = 0;
        row.each(0, row.v, threadIdx.x, kThreads, [&](int, uint32_t key) {
            if (key > edge || (key == edge && ties == ~0ull)) mine += mass(key);
        });
        u64 all = block_sum(t, mine);
        if (ties != ~0ull) all += ties * mass(edge);
        const u64 part = part_of(q.top_p, all);
        const uint32_t low = edge;
        const uint32_t at = reach(t, row, part, &above,
                                  [&](uint32_t key) { return key >= low ? mass(key) : 0ull; });
        // top_p < 1, so `part` is at most the sum and the token at which it is
        // reached has a mass
        const u64 one = mass(at), n = (part - above + one - 1) / one;
        ties = at == edge ? min(ties, n) : n;
        edge = at;
    }
    int last = row.v;
    if (ties != ~0ull) {
        u64 mine = 0;
        const uint32_t e = edge;
        row.each(0, row.v, threadIdx.x, kThreads, [&](int, uint32_t key) { mine += key == e; });
        if (block_sum(t, mine) > ties)
            last = find(t, row, 0, row.v, ties - 1, [=](int, uint32_t key) { return (u64)(key == e); });
    }
    const auto kept = [&](int i, uint32_t key) -> u64 {
        if (key < edge || (key == edge && i > last)) return 0;
        const float w = weight_of(value_of(key), top, q.step);
        return w >= q.min_p ? mass_of(w) : 0;
    };
    u64 mine = 0;
    row.each(0, row.v, threadIdx.x, kThreads, [&](int i, uint32_t key) { mine += kept(i, key); });
    const u64 total = block_sum(t, mine);
    const int id = find(t, row, 0, row.v, target_of(q.u, total), kept);
    if (threadIdx.x == 0) {
        p.ids[r] = id;
        if (p.logprob) p.logprob[r] = logprob_of(kept(id, row.key(id)), total);
    }
}

// ---- groups

constexpr int kLoads = 4;  // 16-byte loads a lane: a group of 64 bytes

// A run is what a wave reads at a time, 64 groups: load u of lane l is the
// run's bytes [(64 u + l) * 16, + 16).
template <typename T> __host__ __device__ constexpr int run_tokens() {
    return 64 * kLoads * (16 / (int)sizeof(typename Raw<T>::type));
}

// What k_pick leaves of a row for k_masses and its own second turn.
struct Found {
    uint32_t top;  // largest key, 0: none
    int edge;      // candidates are the tokens of the bins up to this one
    uint32_t n;    // tokens in the row's list of a wide set
    u64 part;      // what top-p wants before a token that it cuts
};
constexpr int kSlices = 8;  // workgroups that share a row with a wide set

struct Work {
    u64* masses;     // [rows, runs]
    u64* bins;       // [rows, kBins] of the rows with a wide set
    u64* lists;      // [rows, kList] of them
    Found* found;    // [rows]
    uint32_t* left;  // how many rows k_pick left, and which
    uint32_t* keys;  // [rows, runs * 64] largest key of each group
    int runs;
};

// A lane's load u of a run: its first token, and how many of them there are.
template <typename T> __device__ __forceinline__ int first_of(int run, int u, int lane) {
    return run * run_tokens<T>() + (u * 64 + lane) * Row<T>::kVec;
}

// f(u, j, value) for a group's tokens within the row, masked ones as -inf
template <typename T, typename F>
__device__ __forceinline__ void group_values(const Row<T>& row, int run, int lane, F f) {
    constexpr int V = Row<T>::kVec;
    typename Row<T>::R a[kLoads][V];
    const bool whole = first_of<T>(run, kLoads - 1, 63) + V <= row.v;
    if (whole && !row.allowed) {
#pragma unroll
        for (int u = 0; u < kLoads; ++u) load_pack(a[u], row.x + first_of<T>(run, u, lane));
#pragma unroll
        for (int u = 0; u < kLoads; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) f(u, j, Num<T>::get(a[u][j]));
        return;
    }
    uint32_t bits[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
        const int first = first_of<T>(run, u, lane);
        if (whole) {
            load_pack(a[u], row.x + first);
            bits[u] = (uint32_t)row.bits(first);
            continue;
        }
        bits[u] = 0;
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (first + j < row.v) {
                a[u][j] = row.x[first + j];
                bits[u] |= row.bit(first + j) << j;
            }
    }
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) f(u, j, (bits[u] >> j) & 1 ? Num<T>::get(a[u][j]) : -INFINITY);
}

// The one pass over all logits: a wave a run, a lane a group, the mask applied.
// Bound by memory: 256 x 128256 bf16 13.0 us (5.0 TB/s), 512 x 200019 floats
// 75 us (5.5 TB/s), one row of 151669 floats 3.3 us (the launch).
template <typename T> __global__ __launch_bounds__(256) void k_groups(const tkh_sample p, const Work w) {
    const int lane = threadIdx.x & 63;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t r = at / w.runs;
    const int run = (int)(at - r * w.runs);
    if (at == 0 && lane == 0) w.left[0] = 0;
    if (r >= p.rows) return;
    const Row<T> row(p, r);
    float top = -INFINITY;  // fmaxf passes over a NaN
    group_values(row, run, lane, [&](int, int, float x) { top = fmaxf(top, x); });
    w.keys[(r * w.runs + run) * 64 + lane] = key_of(top);
}

// The weight of a run's tokens; where nothing is cut by top-p, of those that
// min-p leaves. Whole numbers, so that a row may be shared among any number of
// waves. Bound by the exponential and its split into two integers: 256 x 128256 bf16 19 us (the logits come from the
// last cache, being read a second time).
template <typename T> __global__ __launch_bounds__(256) void k_masses(const tkh_sample p, const Work w) {
    const int lane = threadIdx.x & 63;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t r = at / w.runs;
    const int run = (int)(at - r * w.runs);
    if (r >= p.rows) return;
    const RowParams q = params_of(p, r);
    const Found found = w.found[r];
    if (q.top_k || !found.top) return;
    const float top = value_of(found.top), least = q.top_p < 1.0f ? 0.0f : q.min_p;
    const Row<T> row(p, r);
    // 32 masses at most: their halves' sums stay below 2^26
    Halves sum = {0, 0};
    // a group whose largest weighs nothing is not read again
    const uint32_t key = w.keys[(r * w.runs + run) * 64 + lane];
    if (key && mass_of(weight_of(value_of(key), top, q.step))) {
        const auto add = [&](float weight) {
            const Halves h = halves_of(weight);
            sum.high += h.high;
            sum.low += h.low;
        };
        // a NaN's weight is 0, as -inf's: exp2 leaves a NaN, fmaxf drops it.
        // The largest's own must be 1: weight_of where its difference or the
        // step (a temperature near 0) is infinite
        if (least > 0.0f || top == INFINITY || q.step == INFINITY)
            group_values(row, run, lane, [&](int, int, float x) {
                const float weight = x > -INFINITY ? weight_of(x, top, q.step) : 0.0f;
                add(weight >= least ? weight : 0.0f);
            });
        else
            group_values(row, run, lane, [&](int, int, float x) {
                add(fmaxf(__builtin_amdgcn_exp2f((x - top) * q.step), 0.0f));
            });
    }
    const u64 mine = add64(((u64)sum.high << 20) + sum.low);
    if (lane == 0) w.masses[r * w.runs + run] = mine;
}

// ---- a row's token from its largest logits

// Each lane's first place among the entries that it and the others add to a
// list; one addition a wave.
__device__ __forceinline__ uint32_t places(uint32_t count, uint32_t* counter) {
    const uint32_t upto = (uint32_t)scan64(count);
    uint32_t base = 0;
    if ((threadIdx.x & 63) == 63 && upto) base = atomicAdd(counter, upto);
    return (uint32_t)__builtin_amdgcn_readlane((int)base, 63) + upto - count;
}

// A token's part of the range of weights, from the largest down. Like the
// weight it falls with x, so parts and keys never disagree on an order.
__device__ __forceinline__ int bin_of(float x, float top, float step) {
    return x == top ? 0 : (int)fminf((top - x) * step * 50.0f, kBins - 1.0f);
}

// Where a running sum over the bins reaches `need`: the bin, and what lies
// before it; false if even all of them do not. A lane holds two bins.
__device__ __forceinline__ bool reach_bin(Team& t, u64 need, int* bin, u64* before) {
    Shared& s = t.m;
    const u64 b0 = s.bins[2 * threadIdx.x], b1 = s.bins[2 * threadIdx.x + 1];
    u64 at;
    const u64 all = block_sum(t, b0 + b1, &at);
    at += scan64(b0 + b1) - b0 - b1;
    if (at < need && need <= at + b0 + b1) {
        const bool second = at + b0 < need;
        s.found[0] = 2 * threadIdx.x + second;
        s.found[1] = at + (second ? b0 : 0);
    }
    __syncthreads();
    *bin = (int)s.found[0];
    *before = s.found[1];
    return need <= all;
}

constexpr int kHeld = 13;  // group keys that a lane holds: 200,019 floats' fit

// The row's group keys of a lane; f(i, key) for each of them.
struct Keys {
    const uint32_t* keys;
    int groups;
    uint32_t held[kHeld];

    __device__ __forceinline__ Keys(const uint32_t* keys, int groups) : keys(keys), groups(groups) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int at = threadIdx.x + i * kThreads;
            held[i] = at < groups ? keys[at] : 0;
        }
    }
    template <typename F> __device__ __forceinline__ void each(F f) const {
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (i * kThreads < groups) f((int)threadIdx.x + i * kThreads, held[i]);
#pragma unroll 1
        for (int i = threadIdx.x + kHeld * kThreads; i < groups; i += kThreads) f(i, keys[i]);
    }
};

// The tokens of the bins up to `edge` into the list, and the bins cleared;
// false if the tokens are too many.
template <typename T>
__device__ __forceinline__ bool gather(Team& t, const Row<T>& row, const Keys& keys, float top, float step, int edge) {
    Shared& s = t.m;
    const auto wanted = [&](float x) { return x > -INFINITY && bin_of(x, top, step) <= edge; };
    uint32_t count = 0;
    keys.each([&](int, uint32_t key) { count += key && wanted(value_of(key)); });
    uint32_t at = places(count, &s.n[0]);
    keys.each([&](int i, uint32_t key) {
        if (!key || !wanted(value_of(key))) return;
        if (at < (uint32_t)kList) s.groups[at] = (uint32_t)i;
        ++at;
    });
    s.bins[2 * threadIdx.x] = s.bins[2 * threadIdx.x + 1] = 0;
    __syncthreads();
    const int n = (int)s.n[0];
    if (n > kList) return false;
    constexpr int V = Row<T>::kVec, kAtOnce = 3;
#pragma unroll 1
    for (int base = 0; base < n * kLoads; base += kThreads * kAtOnce) {
        typename Row<T>::R a[kAtOnce][V];
        u64 b[kAtOnce];
        int first[kAtOnce];
#pragma unroll
        for (int c = 0; c < kAtOnce; ++c) {
            const int i = base + c * kThreads + (int)threadIdx.x;
            b[c] = 0;
            if (i >= n * kLoads) continue;
            const int group = (int)s.groups[i / kLoads];
            first[c] = first_of<T>(group >> 6, i % kLoads, group & 63);
            if (first[c] + V <= row.v) {
                load_pack(a[c], row.x + first[c]);
                b[c] = row.bits(first[c]);
            } else {
                for (int j = 0; j < V; ++j)
                    if (first[c] + j < row.v) {
                        a[c][j] = row.x[first[c] + j];
                        b[c] |= (u64)row.bit(first[c] + j) << j;
                    }
            }
        }
        uint32_t want = 0;
#pragma unroll
        for (int c = 0; c < kAtOnce; ++c) {
            if (!__any(b[c] != 0)) continue;  // most of a short list's waves
#pragma unroll
            for (int j = 0; j < V; ++j)
                want |= (uint32_t)(((uint32_t)b[c] >> j & 1) && wanted(Num<T>::get(a[c][j]))) << (c * V + j);
        }
        uint32_t to = places((uint32_t)__popc(want), &s.n[1]);
#pragma unroll
        for (int c = 0; c < kAtOnce; ++c)
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (want >> (c * V + j) & 1) {
                    if (to < (uint32_t)kList)
                        s.list[to] = (u64)key_of(Num<T>::get(a[c][j])) << 32 | (uint32_t)~(first[c] + j);
                    ++to;
                }
    }
    __syncthreads();
    return s.n[1] <= (uint32_t)kList;
}
__device__ __forceinline__ void put(const tkh_sample& p, int64_t r, int id, u64 mass, u64 total) {
    p.ids[r] = id;
    if (p.logprob) p.logprob[r] = id < 0 ? -INFINITY : logprob_of(mass, total);
}

// A token of the list, as the lane holds it that works on it.
struct Entry {
    u64 self;  // 0: none
    u64 mass;
    float weight;
    __device__ __forceinline__ int index() const { return (int)~(uint32_t)self; }
};
__device__ __forceinline__ Entry entry(const Shared& s, int i, int n, float top, float step) {
    Entry e = {0, 0, 0.0f};
    if (i < n) {
        e.self = s.list[i];
        e.weight = weight_of(value_of((uint32_t)(e.self >> 32)), top, step);
        e.mass = mass_of(e.weight);
    }
    return e;
}

// use(load(j)) for j in [0, n), At of the loads under way at a time; past n
// the last again is loaded, and not used.
struct Pair {
    u64 self, mass;
};
template <int At, typename Load, typename Use> __device__ __forceinline__ void each_of(int n, Load load, Use use) {
#pragma unroll 1
    for (int base = 0; base < n; base += At) {
        Pair o[At];
#pragma unroll
        for (int c = 0; c < At; ++c) o[c] = load(min(base + c, n - 1));
#pragma unroll
        for (int c = 0; c < At; ++c)
            if (base + c < n) use(o[c]);
    }
}

// A token out of the first n of the list, n at most kSmall: a lane a token
// counts what comes before it, by value and then by index, going through all
// of them. `part`: the weight that top-p wants before a token that it cuts,
// or 0 to take it of what top-k leaves.
constexpr int kSmall = 128;

__device__ __forceinline__ void pick_small(Team& t, const tkh_sample& p, int64_t r, const RowParams& q, float top,
                                           int n, u64 part) {
    Shared& s = t.m;
    const Entry e = entry(s, (int)threadIdx.x, n, top, q.step);
    if (threadIdx.x < kSmall) {
        s.mass[threadIdx.x] = e.mass;
        if ((int)threadIdx.x >= n) s.list[threadIdx.x] = 0;
    }
    __syncthreads();
    bool stays = e.mass != 0;
    uint32_t rank = 0;
    u64 before = 0;
    if (__any(stays)) {
        each_of<8>((n + 7) / 8 * 8, [&](int j) { return Pair{s.list[j], s.mass[j]}; }, [&](const Pair& o) {
            const bool ahead = o.self > e.self;
            rank += ahead;
            before += ahead ? o.mass : 0;
        });
    }
    stays = stays && (!q.top_k || rank < q.top_k);
    if (q.top_p < 1.0f) {
        if (!part) part = part_of(q.top_p, block_sum(t, stays ? e.mass : 0));
        stays = stays && before < part;
    }
    stays = stays && e.weight >= q.min_p;
    if (threadIdx.x < kSmall) s.bins[threadIdx.x] = stays ? e.mass : 0;
    const u64 total = block_sum(t, stays ? e.mass : 0);
    if (!__any(stays)) return;
    const u64 target = target_of(q.u, total);
    u64 less = 0;
    each_of<8>((n + 7) / 8 * 8, [&](int j) { return Pair{s.list[j], s.bins[j]}; },
               [&](const Pair& o) { less += (uint32_t)o.self > (uint32_t)e.self ? o.mass : 0; });
    if (stays && less <= target && target < less + e.mass) put(p, r, e.index(), e.mass, total);
}

// The 256 parts: the one in which their running sum passes `target`, which is
// below the sum, and what lies before it. Every wave by itself, four to a lane.
__device__ __forceinline__ int part_at(const Shared& s, u64 target, u64* before) {
    const int lane = threadIdx.x & 63;
    u64 four[4], sum = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) sum += four[c] = s.parts[4 * lane + c];
    u64 at = scan64(sum) - sum;
    const u64 here = __ballot(at <= target && target < at + sum);
    int where = 4 * lane;
#pragma unroll
    for (int c = 0; c < 3; ++c)
        if (where == 4 * lane + c && at + four[c] <= target) {
            at += four[c];
            ++where;
        }
    const int from = __ffsll((long long)here) - 1;
    *before = (u64)(uint32_t)__builtin_amdgcn_readlane((int)(at >> 32), from) << 32 |
              (uint32_t)__builtin_amdgcn_readlane((int)at, from);
    return __builtin_amdgcn_readlane(where, from);
}

// The smallest token that stays where each must have less than `need` of a
// value (1 or its mass) before it, `need` being reached within `bin`, before
// which lies `before`. That bin is divided by 256, and the tokens of the part
// in which `need` is reached are put in order, each counting what is before
// it: they are few unless many logits are equal.
template <int Turn, int Entries, typename F>
__device__ __forceinline__ u64 end_in_bin(Team& t, const Entry (&own)[Entries], float top, float step, int bin,
                                          u64 before, u64 need, F value) {
    Shared& s = t.m;
    if (threadIdx.x < 256) s.parts[threadIdx.x] = 0;
    if (threadIdx.x == 0) s.end[Turn] = ~0ull;
    __syncthreads();
    int part[Entries];
#pragma unroll
    for (int c = 0; c < Entries; ++c) {
        part[c] = -1;
        const u64 v = own[c].mass ? value(own[c]) : 0;
        const float x = value_of((uint32_t)(own[c].self >> 32));
        if (!v || bin_of(x, top, step) != bin) continue;
        const float place = x == top ? 0.0f : (top - x) * step * 50.0f;
        part[c] = (int)((place - (float)bin) * 256.0f);
        atomicAdd(&s.parts[part[c]], v);
    }
    __syncthreads();
    u64 ahead_of_part;
    const int where = part_at(s, need - before - 1, &ahead_of_part);
    before += ahead_of_part;
#pragma unroll
    for (int c = 0; c < Entries; ++c)
        if (part[c] == where) s.members[atomicAdd(&s.n[2 + Turn], 1)] = (uint16_t)(c * kThreads + threadIdx.x);
    __syncthreads();
    const int m = (int)s.n[2 + Turn];
#pragma unroll 1
    for (int i = threadIdx.x; i < m; i += kThreads) {
        const u64 me = s.list[s.members[i]];
        u64 ahead = before;
        each_of<4>(m, [&](int j) { return Pair{s.list[s.members[j]], s.mass[s.members[j]]}; },
                   [&](const Pair& o) { ahead += o.self > me ? value(Entry{o.self, o.mass, 0.0f}) : 0; });
        if (ahead < need) atomicMin(&s.end[Turn], me);
    }
    __syncthreads();
    return s.end[Turn];
}

// The same from any number of tokens in the list: where top-k and top-p end
// is found by bins of weight, the draw by parts of the vocabulary. False if
// `part` is more than the tokens weigh and min-p does not end the set either:
// `edge` is the last bin that is all in the list.
__device__ __forceinline__ bool pick_list(Team& t, const tkh_sample& p, int64_t r, const RowParams& q, float top, int n, u64 part, int edge) {
    Shared& s = t.m;
    constexpr int kOwn = kList / kThreads;
    Entry own[kOwn];
#pragma unroll
    for (int c = 0; c < kOwn; ++c) {
        own[c] = entry(s, c * kThreads + (int)threadIdx.x, n, top, q.step);
        s.mass[c * kThreads + threadIdx.x] = own[c].mass;
    }
    const auto fill = [&](auto value) {
#pragma unroll
        for (int c = 0; c < kOwn; ++c) {
            const u64 v = own[c].mass ? value(own[c]) : 0;
            if (v) atomicAdd(&s.bins[bin_of(value_of((uint32_t)(own[c].self >> 32)), top, q.step)], v);
        }
        __syncthreads();
    };
    u64 end = 0, before;
    int bin;
    if (q.top_k && q.top_k < (uint32_t)n) {
        // tokens without a mass are never drawn: they need not be counted
        const auto one = [](const Entry&) -> u64 { return 1; };
        fill(one);
        if (reach_bin(t, q.top_k, &bin, &before))
            end = end_in_bin<0>(t, own, top, q.step, bin, before, q.top_k, one);
        s.bins[2 * threadIdx.x] = s.bins[2 * threadIdx.x + 1] = 0;
        __syncthreads();
    }
    if (q.top_p < 1.0f) {
        const auto left = [&](const Entry& e) -> u64 { return e.self >= end ? e.mass : 0; };
        fill(left);
        if (!part) {
            u64 mine = 0;
#pragma unroll
            for (int c = 0; c < kOwn; ++c) mine += left(own[c]);
            part = part_of(q.top_p, block_sum(t, mine));
        }
        if (reach_bin(t, part, &bin, &before)) {
            end = end_in_bin<1>(t, own, top, q.step, bin, before, part, left);
        } else {
            // what is not in the list lies in bins behind the edge: lighter
            // than half a bin less than it, to any rounding
            const float beyond = __builtin_amdgcn_exp2f(-((float)edge + 0.5f) * 0.02f);
            if (beyond >= q.min_p) return false;
        }
    }
    u64 mine = 0;
#pragma unroll
    for (int c = 0; c < kOwn; ++c) {
        if (own[c].self < end || !(own[c].weight >= q.min_p)) own[c].mass = 0;
        s.mass[c * kThreads + threadIdx.x] = own[c].mass;
        mine += own[c].mass;
    }
    // the weight of each 256th part of the vocabulary, then the tokens of the
    // part in which the running weight passes the target
    int shift = 0;
    while ((p.vocab - 1) >> shift >= 256) ++shift;
    if (threadIdx.x < 256) s.parts[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kOwn; ++c)
        if (own[c].mass) atomicAdd(&s.parts[own[c].index() >> shift], own[c].mass);
    const u64 total = block_sum(t, mine);
    u64 target = target_of(q.u, total), ahead;
    const int where = part_at(s, target, &ahead);
    target -= ahead;
#pragma unroll
    for (int c = 0; c < kOwn; ++c)
        if (own[c].mass && own[c].index() >> shift == where)
            s.members[atomicAdd(&s.n[4], 1)] = (uint16_t)(c * kThreads + threadIdx.x);
    __syncthreads();
    const int m = (int)s.n[4];
#pragma unroll 1
    for (int i = threadIdx.x; i < m; i += kThreads) {
        const u64 me = s.list[s.members[i]], mass = s.mass[s.members[i]];
        u64 less = 0;
        each_of<4>(m, [&](int j) { return Pair{s.list[s.members[j]], s.mass[s.members[j]]}; },
                   [&](const Pair& o) { less += (uint32_t)o.self > (uint32_t)me ? o.mass : 0; });
        if (less <= target && target < less + mass) put(p, r, (int)~(uint32_t)me, mass, total);
    }
    return true;
}

// Draws where each run's weight is known: the run in which the running weight
// passes the target, and the token in it by kept(index, key).
template <typename T, typename F>
__device__ __forceinline__ void draw_run(Team& t, const tkh_sample& p, int64_t r, const Row<T>& row, const u64* masses,
                                         int runs, float u, u64 total, F kept) {
    Shared& s = t.m;
    u64 target = target_of(u, total);
    int run = 0;
#pragma unroll 1
    for (int base = 0; base < runs; base += kThreads) {
        const int i = base + (int)threadIdx.x;
        const u64 own = i < runs ? masses[i] : 0;
        u64 before;
        const u64 sum = block_sum(t, own, &before);
        if (target >= sum) {
            target -= sum;
            continue;
        }
        before += scan64(own) - own;
        if (own && before <= target && target < before + own) {
            s.found[0] = (u64)i;
            s.found[1] = before;
        }
        __syncthreads();
        run = (int)s.found[0];
        target -= s.found[1];
        __syncthreads();
        break;
    }
    const int lo = run * run_tokens<T>(), hi = min(row.v, lo + run_tokens<T>());
    const int id = find(t, row, lo, hi, target, kept);
    if (threadIdx.x == 0) put(p, r, id, kept(id, row.key(id)), total);
}

constexpr int kMostK = 1024, kFirst = 1024;

// A workgroup a row. First turn: the rows with a top-k, and for the others
// what k_masses needs. Second turn: those others. Bound by the length of the
// steps that follow from each other, each ended by a barrier, not by what they
// read or compute. One row of 151669 floats with top-k 50, 15.0 us of which:
// group keys and their largest 2, bins and the bin of the 50th 3, the tokens of
// the groups that reach it 4.5, ranking them 5. The second turn over 256 rows of
// 128256 bf16 with top-p 0.95 takes 25.3 us: 1 for the sums, 16 to gather
// the tokens of 1,024 groups or more, 6 to pick.
template <typename T, bool Second> __global__ __launch_bounds__(kThreads) void k_pick(const tkh_sample p, const Work w) {
    __shared__ Shared s;
    Team t{s};
    const int64_t r = blockIdx.x;
    const RowParams q = params_of(p, r);
    if (Second && q.top_k) return;
    const Row<T> row(p, r);
    const int groups = w.runs * 64;
    if (threadIdx.x < 5) s.n[threadIdx.x] = 0;
    if (!Second) {
        const Keys keys(w.keys + r * groups, groups);
        s.bins[2 * threadIdx.x] = s.bins[2 * threadIdx.x + 1] = 0;
        uint32_t top_key = 0;
        keys.each([&](int, uint32_t key) { top_key = max(top_key, key); });
#pragma unroll
        for (int d = 32; d; d >>= 1) top_key = max(top_key, __shfl_xor(top_key, d, 64));
        if ((threadIdx.x & 63) == 0) s.tops[threadIdx.x >> 6] = top_key;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWaves; ++i) top_key = max(top_key, s.tops[i]);
        if (!top_key || (!q.top_k && q.top_p >= 1.0f)) {
            if (threadIdx.x == 0) {
                if (!top_key) put(p, r, -1, 0, 0);
                w.found[r] = Found{top_key, 0, 0, 0};
            }
            return;
        }
        const float top = value_of(top_key);
        // the bin by which enough groups have their largest: as many tokens
        // at least are in the bins up to it
        keys.each([&](int, uint32_t key) {
            const int bin = key ? bin_of(value_of(key), top, q.step) : kBins;
            if (bin <= kLastBin) atomicAdd(&s.bins[bin], 1ull);
        });
        __syncthreads();
        int edge;
        u64 before;
        if (!reach_bin(t, q.top_k ? q.top_k : kFirst, &edge, &before)) edge = kLastBin;
        if (!q.top_k) {
            if (threadIdx.x == 0) w.found[r] = Found{top_key, edge, 0, 0};
            return;
        }
        if (q.top_k > (uint32_t)kMostK || !gather(t, row, keys, top, q.step, edge))
            sample_row<T>(s, p, r);
        else if (s.n[1] <= (uint32_t)kSmall)
            pick_small(t, p, r, q, top, (int)s.n[1], 0);
        else
            pick_list(t, p, r, q, top, (int)s.n[1], 0, kLastBin);
        return;
    }
    const Found found = w.found[r];
    if (!found.top) return;
    const float top = value_of(found.top);
    u64 mine = 0;
    const u64* masses = w.masses + r * w.runs;
#pragma unroll 1
    for (int i = threadIdx.x; i < w.runs; i += kThreads) mine += masses[i];
    if (q.top_p < 1.0f) {
        const Keys keys(w.keys + r * groups, groups);
        const u64 part = part_of(q.top_p, block_sum(t, mine));
        if (!gather(t, row, keys, top, q.step, found.edge) ||
            !pick_list(t, p, r, q, top, (int)s.n[1], part, found.edge)) {
            w.bins[r * kBins + 2 * threadIdx.x] = w.bins[r * kBins + 2 * threadIdx.x + 1] = 0;
            if (threadIdx.x == 0) {
                w.found[r].part = part;
                w.left[1 + atomicAdd(&w.left[0], 1)] = (uint32_t)r;
            }
        }
        return;
    }
    // nothing is cut but by min-p
    draw_run(t, p, r, row, masses, w.runs, q.u, block_sum(t, mine), [&](int, uint32_t key) -> u64 {
        const float weight = key ? weight_of(value_of(key), top, q.step) : 0.0f;
        return weight >= q.min_p ? mass_of(weight) : 0;
    });
}

// ---- the rows that k_pick left

// The set that top-p leaves of all tokens, where it is wider than the list,
// eight workgroups a row. k_wide_bins takes the weight of each bin; k_wide_list
// lists the tokens of the bin in which the set ends and sums, a run at a time,
// what lies before it; k_rest ends the bin and draws. With
// all of it in one workgroup a row, a call over 256 x 128256 bf16 with top-p
// 0.95 took 93 us instead of 67, one over 512 x 200019 floats with settings of
// each row's own 414 us instead of 356; of the latter's 218 us now, these
// three take 9, 15 and 12. Where no row is left they cost their launches, 1 to
// 4 us each: the host does not know.
template <typename T> __global__ __launch_bounds__(kThreads) void k_wide_bins(const tkh_sample p, const Work w) {
    __shared__ u64 bins[kBins];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slice = blockIdx.x % kSlices;
    const int per = (w.runs + kSlices - 1) / kSlices, last = min(w.runs, (slice + 1) * per);
    for (uint32_t slot = blockIdx.x / kSlices; slot < w.left[0]; slot += gridDim.x / kSlices) {
        const int64_t r = w.left[1 + slot];
        const Found found = w.found[r];
        const RowParams q = params_of(p, r);
        const float top = value_of(found.top);
        const Row<T> row(p, r);
        bins[2 * threadIdx.x] = bins[2 * threadIdx.x + 1] = 0;
        __syncthreads();
#pragma unroll 1
        for (int run = slice * per + wave; run < last; run += kWaves)
            group_values(row, run, lane, [&](int, int, float x) {
                const u64 m = x > -INFINITY ? mass_of(weight_of(x, top, q.step)) : 0;
                if (m) atomicAdd(&bins[bin_of(x, top, q.step)], m);
            });
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 2; ++c)
            if (bins[2 * threadIdx.x + c])
                atomicAdd(&w.bins[r * kBins + 2 * threadIdx.x + c], bins[2 * threadIdx.x + c]);
        __syncthreads();
    }
}

template <typename T> __global__ __launch_bounds__(kThreads) void k_wide_list(const tkh_sample p, const Work w) {
    __shared__ Shared s;
    Team t{s};
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slice = blockIdx.x % kSlices;
    const int per = (w.runs + kSlices - 1) / kSlices, last = min(w.runs, (slice + 1) * per);
    for (uint32_t slot = blockIdx.x / kSlices; slot < w.left[0]; slot += gridDim.x / kSlices) {
        const int64_t r = w.left[1 + slot];
        const Found found = w.found[r];
        const RowParams q = params_of(p, r);
        const float top = value_of(found.top);
        const Row<T> row(p, r);
        s.bins[2 * threadIdx.x] = w.bins[r * kBins + 2 * threadIdx.x];
        s.bins[2 * threadIdx.x + 1] = w.bins[r * kBins + 2 * threadIdx.x + 1];
        int bin;
        u64 above;
        reach_bin(t, found.part, &bin, &above);
#pragma unroll 1
        for (int run = slice * per + wave; run < last; run += kWaves) {
            Halves sum = {0, 0};
            group_values(row, run, lane, [&](int u, int j, float x) {
                if (!(x > -INFINITY)) return;
                const int b = bin_of(x, top, q.step);
                if (b > bin) return;
                if (b == bin) {
                    const uint32_t at = atomicAdd(&w.found[r].n, 1);
                    if (at < (uint32_t)kList)
                        w.lists[r * kList + at] = (u64)key_of(x) << 32 | (uint32_t)~(first_of<T>(run, u, lane) + j);
                } else {
                    const float weight = weight_of(x, top, q.step);
                    const Halves h = halves_of(weight >= q.min_p ? weight : 0.0f);
                    sum.high += h.high;
                    sum.low += h.low;
                }
            });
            const u64 mine = add64(((u64)sum.high << 20) + sum.low);
            if (lane == 0) w.masses[r * w.runs + run] = mine;
        }
        __syncthreads();
    }
}

// False if the bin in which the set ends has too many tokens, or the row too
// many runs.
template <typename T>
__device__ __forceinline__ bool wide_row(Team& t, const tkh_sample& p, int64_t r, const Row<T>& row, const Work& w,
                                         const Found& found) {
    Shared& s = t.m;
    const RowParams q = params_of(p, r);
    const float top = value_of(found.top);
    const int n = (int)found.n;
    if (n > kList || w.runs > kBins) return false;
    s.bins[2 * threadIdx.x] = w.bins[r * kBins + 2 * threadIdx.x];
    s.bins[2 * threadIdx.x + 1] = w.bins[r * kBins + 2 * threadIdx.x + 1];
    if (threadIdx.x < 5) s.n[threadIdx.x] = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) s.list[i] = w.lists[r * kList + i];
    int bin;
    u64 above;
    reach_bin(t, found.part, &bin, &above);
    constexpr int kOwn = kList / kThreads;
    Entry own[kOwn];
#pragma unroll
    for (int c = 0; c < kOwn; ++c) {
        own[c] = entry(s, c * kThreads + (int)threadIdx.x, n, top, q.step);
        s.mass[c * kThreads + threadIdx.x] = own[c].mass;
    }
    u64* const masses = s.bins;  // of runs, from here on
    for (int i = threadIdx.x; i < w.runs; i += kThreads) masses[i] = w.masses[r * w.runs + i];
    const u64 end =
        end_in_bin<0>(t, own, top, q.step, bin, above, found.part, [](const Entry& e) { return e.mass; });
#pragma unroll
    for (int c = 0; c < kOwn; ++c)
        if (own[c].mass && own[c].self >= end && own[c].weight >= q.min_p)
            atomicAdd(&masses[own[c].index() / run_tokens<T>()], own[c].mass);
    __syncthreads();
    u64 mine = 0;
    for (int i = threadIdx.x; i < w.runs; i += kThreads) mine += masses[i];
    draw_run(t, p, r, row, masses, w.runs, q.u, block_sum(t, mine), [&](int i, uint32_t key) -> u64 {
        if (!key || ((u64)key << 32 | (uint32_t)~i) < end) return 0;
        const float weight = weight_of(value_of(key), top, q.step);
        return weight >= q.min_p ? mass_of(weight) : 0;
    });
    return true;
}

template <typename T> __global__ __launch_bounds__(kThreads) void k_rest(const tkh_sample p, const Work w) {
    __shared__ Shared s;
    for (uint32_t slot = blockIdx.x; slot < w.left[0]; slot += gridDim.x) {
        const int64_t r = w.left[1 + slot];
        Team t{s};
        if (!wide_row(t, p, r, Row<T>(p, r), w, w.found[r])) sample_row<T>(s, p, r);
        __syncthreads();
    }
}

static int runs_of(int64_t vocab, int dtype) {
    return (int)ceil_div(vocab, dtype == TKH_F32 ? run_tokens<float>() : run_tokens<__half>());
}

// The parts of the workspace; the bytes that they take.
static uint64_t lay_out(Work* w, void* at, int64_t rows, int runs) {
    w->runs = runs;
    w->masses = (u64*)at;
    w->bins = w->masses + rows * runs;
    w->lists = w->bins + rows * kBins;
    w->found = (Found*)(w->lists + rows * kList);
    w->left = (uint32_t*)(w->found + rows);
    w->keys = w->left + rows + 1;
    return (uint64_t)((char*)(w->keys + rows * runs * 64) - (char*)at);
}

template <typename T> static int sample_rows(const tkh_sample& p, void* stream) {
    Work w;
    lay_out(&w, p.workspace, p.rows, runs_of(p.vocab, p.dtype));
    const dim3 waves((unsigned)ceil_div(p.rows * w.runs, 4)), rows((unsigned)p.rows), threads(kThreads);
    // as many as one turn over the chip holds: each goes on to the next row
    const unsigned few = (unsigned)(p.rows < 32 ? p.rows : 32), many = (unsigned)(p.rows < 256 ? p.rows : 256);
    int status = launch("k_groups", k_groups<T>, waves, dim3(256), 0, stream, p, w);
    if (status == TKH_OK) status = launch("k_pick", k_pick<T, false>, rows, threads, 0, stream, p, w);
    // not where every row has a top-k
    if (p.top_k || !(p.top_k_value > 0 || (!p.temperature && !(p.temperature_value > 0.0f)))) {
        if (status == TKH_OK) status = launch("k_masses", k_masses<T>, waves, dim3(256), 0, stream, p, w);
        if (status == TKH_OK) status = launch("k_pick", k_pick<T, true>, rows, threads, 0, stream, p, w);
        if (p.top_p || p.top_p_value < 1.0f) {
            const dim3 slices(few * kSlices);
            if (status == TKH_OK) status = launch("k_wide_bins", k_wide_bins<T>, slices, threads, 0, stream, p, w);
            if (status == TKH_OK) status = launch("k_wide_list", k_wide_list<T>, slices, threads, 0, stream, p, w);
            if (status == TKH_OK) status = launch("k_rest", k_rest<T>, dim3(many), threads, 0, stream, p, w);
        }
    }
    return status;
}

}  // namespace tkh

extern "C" uint64_t tk_head_sample_workspace(int64_t rows, int64_t vocab, int32_t dtype) {
    using namespace tkh;
    if (rows < 1 || vocab < 1 || vocab > TKH_SAMPLE_MAX_VOCAB) return 0;
    Work w;
    return lay_out(&w, nullptr, rows, runs_of(vocab, dtype));
}

extern "C" int tk_head_sample(const tkh_sample* args, void* stream) {
    using namespace tkh;
    if (!args) return fail(TKH_E_INVALID_ARG, "no arguments");
    const tkh_sample& p = *args;
    if (p.rows < 0 || !fits_launch(p.rows, kThreads) || p.vocab < 1 || p.vocab > TKH_SAMPLE_MAX_VOCAB)
        return fail(TKH_E_SHAPE, "rows %lld, vocab %lld", (long long)p.rows, (long long)p.vocab);
    if (p.dtype < TKH_F32 || p.dtype > TKH_F16) return fail(TKH_E_UNSUPPORTED, "dtype %d", p.dtype);
    if (p.rows == 0) return TKH_OK;
    if (!p.logits || !p.u || !p.ids) return fail(TKH_E_INVALID_ARG, "a null pointer");
    if (p.rows > 1 && p.logits_stride < 0) return fail(TKH_E_SHAPE, "logits stride");
    if (p.allowed && p.allowed_stride && p.allowed_stride < ceil_div(p.vocab, 32))
        return fail(TKH_E_SHAPE, "a mask row has %lld words", (long long)ceil_div(p.vocab, 32));
    if (p.workspace_size < tk_head_sample_workspace(p.rows, p.vocab, p.dtype))
        return fail(TKH_E_CAPACITY, "workspace of %llu bytes", (unsigned long long)p.workspace_size);
    if (!p.workspace || (uintptr_t)p.workspace % 16) return fail(TKH_E_INVALID_ARG, "workspace is not 16-byte aligned");
    if (!fits_launch(ceil_div(p.rows * runs_of(p.vocab, p.dtype), 4), 256))
        return fail(TKH_E_SHAPE, "rows %lld of vocab %lld", (long long)p.rows, (long long)p.vocab);
    DeviceScope scope(p.device);
    if (scope.status() != TKH_OK) return scope.status();
    if (p.dtype == TKH_F32) return sample_rows<float>(p, stream);
    if (p.dtype == TKH_BF16) return sample_rows<__hip_bfloat16>(p, stream);
    return sample_rows<__half>(p, stream);
}
