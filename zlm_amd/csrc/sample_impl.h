// sample_impl.h -- CDNA4 (gfx950) device code of the kernels that draw a token from each
// row of logits by temperature, top-k, top-p and min-p with a given uniform number
// (zlm_sample.hip), and that find what a draw would take a row's tokens by (zlm_verify.hip).
//
// The tokens in order of probability (the lower index first among equals) are
// x_1 >= x_2 >= ..; every filter keeps a prefix of that order, and the draw takes
// the first token whose cumulative weight exceeds u times that of the prefix.  So
// each step asks where a cumulative count or weight is reached, and no sort of the
// row is needed.  Two launches:
//   hist  a histogram by value of each 8192 logits, and the slice's largest tokens
//   pick  a workgroup a row joins the histograms: they answer to within a bin.  The
//         tokens of the bins in question are mostly among the slices' largest; else the
//         workgroup looks the row through for them, once
//
// Weights.  y = 16 x / T in 64 bits; bin floor(y), 1/16 of a temperature wide, on a
// grid that does not depend on the row's maximum, so the slices of a row need no
// pass for it.  A token's weight relative to its bin's upper edge, in (0.939, 1],
// is held as an integer of 2^-34: the sums of a bin are exact in any order, a
// bin's sum times e^(-bin/16) in 64 bits.  512 bins reach e^-32 below the largest:
// what lies under that has no weight (all of 2^20 such tokens are 1.3e-8 of it,
// less than the step of u).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sample_args.h"

// y, its bin and the distance between them come from one rounded product: where
// logits are large, an fma of it would be another number.
#pragma clang fp contract(off)

namespace {

using Args = zlm::SampleArgs;
using zlm::SampleSlice;
constexpr uint32_t kWave = 64, kThreads = 512;  // of a row's workgroup
constexpr uint32_t kSlice = zlm::kSampleSlice, kBins = zlm::kSampleBins, kSlices = zlm::kSampleSlices;
constexpr uint32_t kShort = zlm::kSampleShort;
// Tokens that are looked at one by one, in LDS: as many as leave a CU one workgroup, or (the
// cuts of rows without their draws) two.  Where a flat row has more of them in question each cut
// reads it again; two workgroups a CU are worth that as soon as rows are many: verification of
// 226 rows of 128256 144 us, 156 with a list of 12288, of standard deviation 0.3 and top-k 2000
// 127 and 138, top-p 0.9 171 and 187, top-k 20000 171 and 188; of 5 rows of 151936 34 and 34, flat
// ones 34 and 35, 68 and 62, 66 and 59.
#ifdef ZLM_SAMPLE_FEW
constexpr uint32_t kList = 4096;
#else
constexpr uint32_t kList = 12288;
#endif
constexpr double kUnit = 17179869184.0;  // 2^34: the weight at a bin's edge
constexpr int kCountShift = 50;          // a bin's count above its weights: 8192 x 2^34 is 2^47

// Logits as ordered integers; 0 for those that are never drawn (-inf, NaN).
__device__ __forceinline__ uint32_t key_of(float x) {
    if (!(x > -INFINITY)) return 0;
    x = __builtin_fminf(x, 3.402823466e38f) + 0.0f;  // infinity counts as the largest number, -0 as 0
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// The weight of a token that lies f = y - floor(y) above its bin's lower edge,
// e^((f - 1) / 16) in units of 2^-34: a polynomial of degree 5 through the
// Chebyshev nodes of [0, 1], good to 4e-14, a 1400th of the unit.  Its
// coefficients stay in scalar registers.
struct Weight {
    double c[6];
    __device__ Weight() {
        const double k[6] = {0.939413062813436,     0.05871331642866946,   0.0018347911054814223,
                             3.822495502710707e-05, 5.969942951840798e-07, 7.703050641794107e-09};
#pragma unroll
        for (int i = 0; i < 6; i++) {
            c[i] = k[i] * kUnit;
            asm("" : "+s"(c[i]));
        }
    }
    __device__ __forceinline__ uint64_t operator()(double f) const {
        return __builtin_bit_cast(uint64_t, raised(f)) & 0xfffffffffffffull;
    }
    // With a count of one above it: 2^52's exponent goes and 2^50 comes in one addition.
    __device__ __forceinline__ uint64_t counted(double f) const {
        return __builtin_bit_cast(uint64_t, raised(f)) + ((1ull << kCountShift) - (0x433ull << 52));
    }
    __device__ __forceinline__ double units(double f) const { return raised(f) - 4503599627370496.0; }  // the integer itself

private:
    __device__ __forceinline__ double raised(double f) const {
        double r = __builtin_fma(c[5], f, c[4]);
        r = __builtin_fma(r, f, c[3]);
        r = __builtin_fma(r, f, c[2]);
        r = __builtin_fma(r, f, c[1]);
        return __builtin_fma(r, f, c[0]) + 4503599627370496.0;  // + 2^52: the integer in the low bits
    }
};

__device__ __forceinline__ double rate_of(const Args& a, uint32_t row) {  // 16 / T; 0: greedy
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    return t > 0.0f ? 16.0 / static_cast<double>(__builtin_fminf(t, 3.402823466e38f)) : 0.0;
}

// Another lane's value by a DPP control; 0 where the control has no source or the
// row is not in kRows.
template <int kCtrl, int kRows = 0xf>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, kRows, 0xf, false));
}
template <int kCtrl, int kRows = 0xf>
__device__ __forceinline__ uint64_t dpp(uint64_t v) {
    return static_cast<uint64_t>(dpp<kCtrl, kRows>(static_cast<uint32_t>(v >> 32))) << 32 | dpp<kCtrl, kRows>(static_cast<uint32_t>(v));
}
template <int kCtrl, int kRows = 0xf>
__device__ __forceinline__ double dpp(double v) {
    return __builtin_bit_cast(double, dpp<kCtrl, kRows>(__builtin_bit_cast(uint64_t, v)));
}

// Inclusive sums over the wave: within rows of 16, then row 0's and 2's last to
// rows 1 and 3, then the lower half's last to the upper.
template <class T>
__device__ __forceinline__ T wave_scan(T v) {
    v += dpp<0x111>(v);
    v += dpp<0x112>(v);
    v += dpp<0x114>(v);
    v += dpp<0x118>(v);
    v += dpp<0x142, 0xa>(v);
    return v + dpp<0x143, 0xc>(v);
}

// The largest of the wave (0 if none is larger), in every lane.
template <class T>
__device__ __forceinline__ T wave_max(T v) {
    const auto more = [&](T w) { v = w > v ? w : v; };
    more(dpp<0x111>(v));
    more(dpp<0x112>(v));
    more(dpp<0x114>(v));
    more(dpp<0x118>(v));
    more(dpp<0x142, 0xa>(v));
    more(dpp<0x143, 0xc>(v));
    return v;
}
template <class T>
__device__ __forceinline__ T last_lane(T v);
template <>
__device__ __forceinline__ uint32_t last_lane(uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}
template <>
__device__ __forceinline__ uint64_t last_lane(uint64_t v) {
    return static_cast<uint64_t>(last_lane(static_cast<uint32_t>(v >> 32))) << 32 | last_lane(static_cast<uint32_t>(v));
}

// The smallest key of a bin whose lower edge is at y = edge: the border is known to
// a rounding, the wave's lanes try the 64 keys around it.
__device__ __forceinline__ uint32_t key_at(double edge, double rate) {
    const double e = __builtin_fmax(__builtin_fmin(edge / rate, 3.402823466e38), -3.402823466e38);
    const uint32_t k = key_of(static_cast<float>(e)) - 31;
    const uint64_t in = __ballot(static_cast<double>(value_of(k + (threadIdx.x & (kWave - 1)))) * rate >= edge);
    return k + (in ? __builtin_ctzll(in) : kWave);
}

// One slice of a row: its largest logit, the histogram below it, and the short list
// of the tokens that most draws are decided among.  256 threads hold the slice in
// registers: eight workgroups a CU are at different steps of it, and all of a
// slice's loads are in flight at once.  Where there are too few slices for that,
// 1024 threads a slice finish it sooner.
template <uint32_t kHistThreads>
__device__ __forceinline__ void slice_hist(const Args& a, uint32_t row) {
    constexpr uint32_t kHistPer = kSlice / kHistThreads, kHistWaves = kHistThreads / kWave;
    const Weight weight;
    constexpr uint32_t kCopies = 4;  // neighbouring lanes count apart: equal bins of a wave's lanes collide less
    __shared__ __attribute__((aligned(16))) unsigned long long hist[kBins][kCopies];
    __shared__ uint32_t max_of[kHistWaves];
    __shared__ uint32_t ends[kHistWaves], at_of[kHistWaves], n_short, n_bins;
    const uint32_t tid = threadIdx.x, s = blockIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
    const float* from = a.logits + row * a.stride;
    const double rate = rate_of(a, row);
    float x[kHistPer];
    if ((s + 1) * kSlice <= a.vocab) {
#pragma unroll
        for (uint32_t j = 0; j < kHistPer; j++) x[j] = from[s * kSlice + j * kHistThreads + tid];
    } else {
#pragma unroll
        for (uint32_t j = 0; j < kHistPer; j++) {
            const uint32_t i = s * kSlice + j * kHistThreads + tid;
            x[j] = i < a.vocab ? from[i] : -INFINITY;
        }
    }
    float mx = -INFINITY;
#pragma unroll
    for (uint32_t j = 0; j < kHistPer; j++) mx = __builtin_fmaxf(mx, x[j]);
    if (__ballot(mx > 3.402823466e38f)) {  // a NaN stays one: no comparison below holds for it
#pragma unroll
        for (uint32_t j = 0; j < kHistPer; j++) x[j] = x[j] > 3.402823466e38f ? 3.402823466e38f : x[j];
        mx = __builtin_fminf(mx, 3.402823466e38f);
    }
    const uint32_t wave_key = last_lane(wave_max(key_of(mx)));
    if (lane == 0) max_of[wid] = wave_key;
    for (uint32_t i = tid; i < kBins * kCopies; i += kHistThreads) hist[0][i] = 0;
    if (tid == 0) n_short = n_bins = 0;
    __syncthreads();
    uint32_t best_key = 0;
#pragma unroll
    for (uint32_t w = 0; w < kHistWaves; w++) best_key = max(best_key, max_of[w]);
    mx = value_of(best_key);
    const size_t at = static_cast<size_t>(row) * a.slices + s;
    const uint64_t best = static_cast<uint64_t>(best_key) << 32;
    if (best == 0 || rate == 0.0) {
        uint32_t first = 0xffffffffu;  // of the largest, for a greedy row
#pragma unroll
        for (uint32_t j = kHistPer; j-- > 0;)
            if (best && x[j] == mx) first = s * kSlice + j * kHistThreads + tid;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) first = min(first, static_cast<uint32_t>(__shfl_xor(first, o)));
        if (lane == 0) at_of[wid] = first;
        __syncthreads();
        if (tid == 0) {
            for (uint32_t w = 0; w < kHistWaves; w++) first = min(first, at_of[w]);
            a.info[at] = {best ? best | static_cast<uint32_t>(~first) : 0, 0, 0};
        }
        return;
    }
    const double top = __builtin_floor(static_cast<double>(mx) * rate);
#pragma unroll
    for (uint32_t j = 0; j < kHistPer; j++) {
        const double y = static_cast<double>(x[j]) * rate, b = __builtin_floor(y);
        const double d = top - b;
        if (d < static_cast<double>(kBins)) atomicAdd(&hist[static_cast<uint32_t>(d)][tid % kCopies], static_cast<unsigned long long>(weight.counted(y - b)));
    }
    __syncthreads();
    // the bins that the short list has room for: two a thread
    uint32_t c0 = 0, c1 = 0;
    if (tid < kBins / 2) {
        ulonglong2 h = {0, 0};
#pragma unroll
        for (uint32_t i = 0; i < kCopies; i++) {
            h.x += hist[2 * tid][i];
            h.y += hist[2 * tid + 1][i];
        }
        reinterpret_cast<ulonglong2*>(a.hist + at * kBins)[tid] = h;
        c0 = static_cast<uint32_t>(h.x >> kCountShift);
        c1 = static_cast<uint32_t>(h.y >> kCountShift);
    }
    uint32_t c = wave_scan(c0 + c1);
    if (lane == kWave - 1) ends[wid] = c;
    __syncthreads();
    for (uint32_t w = 0; w < wid; w++) c += ends[w];
    const bool two = tid < kBins / 2;
    const uint32_t fits = __builtin_popcountll(__ballot(two && c - c1 <= kShort)) + __builtin_popcountll(__ballot(two && c <= kShort));
    if (lane == 0 && fits) atomicAdd(&n_bins, fits);
    __syncthreads();
    const uint32_t bins = n_bins;
    if (bins) {
        const float least = value_of(key_at(top - static_cast<double>(bins - 1), rate));
#pragma unroll
        for (uint32_t j = 0; j < kHistPer; j++)
            if (x[j] >= least) {
                const uint32_t to = atomicAdd(&n_short, 1u);
                if (to < kShort)
                    a.shorts[at * kShort + to] =
                        static_cast<uint64_t>(key_of(x[j])) << 32 | static_cast<uint32_t>(~(s * kSlice + j * kHistThreads + tid));
            }
    }
    __syncthreads();
    if (tid == 0) a.info[at] = {best, n_short <= kShort ? bins : 0, n_short};
}

constexpr uint32_t kRuns = 4;   // top-k's bin, top-p's, min-p's, the draw's
constexpr uint32_t kFinal = 64;  // tokens that a wave decides among

struct Shared {
    uint64_t list[kList];   // the tokens of the flagged bins, in no order: key, ~index
    double weight[kBins];   // cumulative, all bins up to and with this one
    uint32_t count[kBins];
    double scale[kBins];    // e^(-bin/16) in units of the weights
    // sums by range of tokens
    uint32_t sub_count[kThreads];
    unsigned long long sub_weight[kThreads];
    uint64_t last[kFinal];
    uint32_t flags[kBins / 32];
    float lo[kRuns], hi[kRuns];  // the flagged bins' runs, by value
    uint64_t best[kSlices];
    uint32_t shift[kSlices];  // a slice's top bin below the row's (kBins: no tokens with weight)
    uint32_t bins[kSlices], n_short[kSlices];
    // what the waves of a scan or search hand on: two sets, used in turn, so that a
    // wave may start the next while others read the last
    uint64_t part_w[2][kThreads / kWave];
    uint32_t part_c[2][kThreads / kWave], part_i[2][kThreads / kWave];
    uint32_t n, step_n, step_count;
    uint64_t step_weight;
};

// Inclusive sums over the workgroup in thread order.  `turn` alternates.
__device__ __forceinline__ uint32_t block_scan(Shared& sm, uint32_t& turn, uint32_t c) {
    const uint32_t wid = threadIdx.x / kWave;
    turn ^= 1;
    c = wave_scan(c);
    if ((threadIdx.x & (kWave - 1)) == kWave - 1) sm.part_c[turn][wid] = c;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kThreads / kWave; i++) c += i < wid ? sm.part_c[turn][i] : 0;
    return c;
}
template <class T>  // double or uint64_t
__device__ __forceinline__ T block_scan(Shared& sm, uint32_t& turn, T w) {
    const uint32_t wid = threadIdx.x / kWave;
    turn ^= 1;
    w = wave_scan(w);
    if ((threadIdx.x & (kWave - 1)) == kWave - 1) sm.part_w[turn][wid] = __builtin_bit_cast(uint64_t, w);
    __syncthreads();
    T before = 0;
#pragma unroll
    for (uint32_t i = 0; i < kThreads / kWave; i++) before += i < wid ? __builtin_bit_cast(T, sm.part_w[turn][i]) : T(0);
    return before + w;
}

constexpr uint32_t kNone = 0xffffffffu;

// The index `i` of the first thread that says yes (i does not fall with the thread), or kNone.
__device__ __forceinline__ uint32_t first_of(Shared& sm, uint32_t& turn, bool yes, uint32_t i) {
    turn ^= 1;
    const uint64_t m = __ballot(yes);
    const uint32_t own = m ? __builtin_amdgcn_readlane(i, __builtin_ctzll(m)) : kNone;
    if ((threadIdx.x & (kWave - 1)) == 0) sm.part_i[turn][threadIdx.x / kWave] = own;
    __syncthreads();
    uint32_t first = kNone;
#pragma unroll
    for (uint32_t w = 0; w < kThreads / kWave; w++) first = min(first, sm.part_i[turn][w]);
    return first;
}

// What a search looks for.
enum Mode { kCount, kAtLeast, kMore, kKey };  // kKey: the tokens from a key on
struct Goal {
    Mode mode;
    double w;      // kAtLeast, kMore: the cumulative weight
    uint32_t n;    // kCount: how many tokens; kKey: the smallest key
    uint32_t b0 = 0, b1 = kBins - 1;  // the bins in question for it, whose tokens are listed
    __device__ bool reached(uint32_t count, double weight) const {
        return mode == kCount ? count >= n : mode == kAtLeast ? weight >= w : weight > w;
    }
};
// A token in the order, and the cumulative weight with it.
struct Found {
    uint64_t token;  // key, ~index
    double weight;
};

class Row {
public:
    // What pick reads of the row at its start, all in one latency: the histograms and
    // short lists of the first slices, as many as registers hold.
    static constexpr uint32_t kAhead = kList < 12288 ? 24 : 32, kSide = kThreads / kShort;
    struct Ahead {
        uint64_t hist[kAhead], shorts[kAhead / kSide];
    };
    __device__ __forceinline__ static void read_ahead(const Args& a, uint32_t row, uint32_t s0, Ahead& h) {
        const uint64_t* hist = a.hist + static_cast<size_t>(row) * a.slices * kBins;
        const uint64_t* shorts = a.shorts + static_cast<size_t>(row) * a.slices * kShort;
        constexpr uint32_t kStep = 8;  // slices, as far as there are any
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k += kStep) {
            if (s0 + k < a.slices) {
#pragma unroll
                for (uint32_t j = k; j < k + kStep; j++)
                    h.hist[j] = hist[static_cast<size_t>(min(s0 + j, a.slices - 1)) * kBins + threadIdx.x];
#pragma unroll
                for (uint32_t j = k / kSide; j < (k + kStep) / kSide; j++)
                    h.shorts[j] = shorts[static_cast<size_t>(min(s0 + kSide * j + threadIdx.x / kShort, a.slices - 1)) * kShort +
                                         threadIdx.x % kShort];
            } else {
#pragma unroll
                for (uint32_t j = k; j < k + kStep; j++) h.hist[j] = 0;
#pragma unroll
                for (uint32_t j = k / kSide; j < (k + kStep) / kSide; j++) h.shorts[j] = 0;
            }
        }
    }

    __device__ __forceinline__ Row(const Args& a, Shared& sm, uint32_t row, double rate, uint64_t best)
        : a_(a), sm_(sm), row_(row), rate_(rate), x_(a.logits + row * a.stride), tid_(threadIdx.x), best_(best),
          top_(edge_of(static_cast<uint32_t>(best >> 32))) {
        static_assert(kThreads == kBins, "a bin a thread");
        sm_.scale[tid_] = exp(static_cast<double>(tid_) * -0.0625) / kUnit;
        if (tid_ < kBins / 32) sm_.flags[tid_] = 0;
        if (tid_ == 0) sm_.n = 0;
        if (tid_ < a_.slices) {
            const uint64_t b = sm_.best[tid_];
            sm_.shift[tid_] =
                b ? static_cast<uint32_t>(__builtin_fmin(top_ - edge_of(static_cast<uint32_t>(b >> 32)), 1.0 * kBins)) : kBins;
        }
        __syncthreads();
    }

    // The slices' histograms as the row's: cumulative counts and weights by bin.
    __device__ __forceinline__ void join(Ahead& h) {
        // eight slices at a time through LDS (the list's room), to their places on the row's grid
        static_assert(8 * kBins <= kList, "room for eight histograms");
        uint32_t count = 0;
        uint64_t weight = 0;
        for (uint32_t s0 = 0; s0 < a_.slices; s0 += kAhead) {
            if (s0) read_ahead(a_, row_, s0, h);
#pragma unroll
            for (uint32_t j0 = 0; j0 < kAhead; j0 += 8) {
                if (s0 + j0 >= a_.slices) break;
                __syncthreads();
#pragma unroll
                for (uint32_t j = 0; j < 8; j++) sm_.list[j * kBins + tid_] = h.hist[j0 + j];
                __syncthreads();
#pragma unroll
                for (uint32_t j = 0; j < 8; j++) {
                    const uint32_t s = s0 + j0 + j, shift = sm_.shift[min(s, a_.slices - 1)];
                    const bool has = s < a_.slices && tid_ >= shift;
                    const uint64_t x = sm_.list[j * kBins + (has ? tid_ - shift : 0)];
                    count += has ? static_cast<uint32_t>(x >> kCountShift) : 0;
                    weight += has ? x & ((1ull << kCountShift) - 1) : 0;
                }
            }
        }
        own_ = count;
        const uint32_t c = block_scan(sm_, turn_, count);
        const double w = block_scan(sm_, turn_, static_cast<double>(weight) * sm_.scale[tid_]);
        sm_.count[tid_] = c;
        sm_.weight[tid_] = w;
        __syncthreads();
    }

    __device__ __forceinline__ double weight_to(uint32_t end) const { return end ? sm_.weight[end - 1] : 0.0; }  // bins under `end`
    __device__ __forceinline__ uint32_t count_to(uint32_t end) const { return end ? sm_.count[end - 1] : 0; }

    // The smallest and the largest key of a bin.
    __device__ __forceinline__ uint32_t first_key(uint32_t bin) const { return key_at(top_ - static_cast<double>(bin), rate_); }
    __device__ __forceinline__ uint32_t last_key(uint32_t bin) const {
        return bin ? first_key(bin - 1) - 1 : static_cast<uint32_t>(best_ >> 32);
    }

    __device__ __forceinline__ uint32_t bin_of(uint32_t key) const {  // kBins: below them
        const double d = top_ - edge_of(key);
        return d < 1.0 * kBins ? static_cast<uint32_t>(__builtin_fmax(d, 0.0)) : kBins;
    }

    // The first bin with tokens by whose end the goal is reached; where none is (a rounding:
    // no goal is past the row's weight), the last bin with tokens.
    __device__ __forceinline__ uint32_t bin_for(const Goal& g) {
        const uint32_t b = first_of(sm_, turn_, own_ && g.reached(sm_.count[tid_], sm_.weight[tid_]), tid_);
        return b != kNone ? b : kBins - 1 - first_of(sm_, turn_, sm_.count[kBins - 1 - tid_] != count_to(kBins - 1 - tid_), tid_);
    }

    // Bins b0 .. b1 are in question.
    __device__ __forceinline__ void flag(uint32_t b0, uint32_t b1) {
        if (tid_ >= b0 && tid_ <= b1) atomicOr(&sm_.flags[tid_ / 32], 1u << tid_ % 32);
    }
    // Those of a goal between two weights are: b[0] .. b[1].  Light bins behind heavy ones add
    // less than a rounding, so the second weight may be a rounding below the first.
    __device__ __forceinline__ void bins_for(Mode mode, double w0, double w1, uint32_t b[2]) {
        b[0] = bin_for({mode, w0, 0});
        b[1] = max(bin_for({mode, w1, 0}), b[0]);
        flag(b[0], b[1]);
    }
    __device__ __forceinline__ bool flagged(uint32_t bin) const { return sm_.flags[bin / 32] >> bin % 32 & 1; }

    // The number of the flagged bins' tokens.
    __device__ __forceinline__ uint32_t in_question() {
        __syncthreads();
        const uint32_t c = block_scan(sm_, turn_, flagged(tid_) ? own_ : 0);
        if (tid_ == kThreads - 1) sm_.step_n = c;
        __syncthreads();
        return sm_.step_n;
    }

    __device__ __forceinline__ void put(uint64_t token) {
        const uint32_t at = atomicAdd(&sm_.n, 1u);
        if (at < kList) sm_.list[at] = token;
    }

    // Lists the flagged bins' tokens from the slices' short lists; false where one of
    // these ends before the last of the bins.
    __device__ __forceinline__ bool list_shorts(Ahead& h) {
        const uint32_t lane = tid_ & (kWave - 1), bits = lane < kBins / 32 ? sm_.flags[lane] : 0;
        const uint32_t last = last_lane(wave_max(bits ? 32 * lane + 31 - __builtin_clz(bits) : 0u));
        const bool open = tid_ < a_.slices && sm_.shift[tid_] <= last && last - sm_.shift[tid_] >= sm_.bins[tid_];
        if (first_of(sm_, turn_, open, tid_) != kNone) return false;
        const uint32_t least = first_key(last);
        for (uint32_t s0 = 0; s0 < a_.slices; s0 += kAhead) {
            if (a_.slices > kAhead) read_ahead(a_, row_, s0, h);
#pragma unroll
            for (uint32_t j = 0; j < kAhead / kSide; j++) {
                const uint32_t s = s0 + kSide * j + tid_ / kShort, key = static_cast<uint32_t>(h.shorts[j] >> 32);
                const bool has = s < a_.slices && tid_ % kShort < sm_.n_short[min(s, a_.slices - 1)];
                if (!has || key < least) continue;
                const uint32_t b = bin_of(key);
                if (b < kBins && flagged(b)) put(h.shorts[j]);
            }
        }
        __syncthreads();
        n_ = min(sm_.n, kList);
        return true;
    }

    // Lists the flagged bins' tokens from the row itself.  Four logits a load, 16 loads
    // in flight; a logit in no run costs two comparisons a run and a bit.
    __device__ __forceinline__ void list_row() {
        uint32_t runs = 0, prev = 0;
        for (uint32_t w = 0; w < kBins / 32; w++) {
            // runs begin where a bin is flagged and the one before is not
            const uint32_t bits = sm_.flags[w], begins = bits & ~(bits << 1 | prev >> 31);
            prev = bits;
            for (uint32_t m = begins; m; m &= m - 1) {
                const uint32_t b0 = 32 * w + __builtin_ctz(m);
                uint32_t b1 = b0;
                while (b1 + 1 < kBins && flagged(b1 + 1)) b1++;
                const uint32_t hi = last_key(b0), lo = first_key(b1);
                if (tid_ == 0 && runs < kRuns) {
                    sm_.lo[runs] = value_of(lo);
                    sm_.hi[runs] = hi >= key_of(3.402823466e38f) ? INFINITY : value_of(hi);
                }
                runs++;
            }
        }
        runs = min(runs, kRuns);
        __syncthreads();
        typedef float v4 __attribute__((ext_vector_type(4), aligned(4)));
        constexpr uint32_t kLoads = 16;
        const uint32_t n4 = a_.vocab / 4;
        for (uint32_t c = 0; c < n4; c += kThreads * kLoads) {
            v4 x[kLoads];
#pragma unroll
            for (uint32_t j = 0; j < kLoads; j++)
                x[j] = *reinterpret_cast<const v4*>(x_ + 4 * static_cast<size_t>(min(c + j * kThreads + tid_, n4 - 1)));
            uint32_t hit[2] = {0, 0};
            for (uint32_t r = 0; r < runs; r++) {
                const float lo = sm_.lo[r], hi = sm_.hi[r];
#pragma unroll
                for (uint32_t j = 0; j < kLoads; j++)
#pragma unroll
                    for (uint32_t e = 0; e < 4; e++)
                        hit[j / 8] |= x[j][e] >= lo && x[j][e] <= hi ? 1u << (4 * (j % 8) + e) : 0u;
            }
#pragma unroll
            for (uint32_t h = 0; h < 2; h++)
                for (uint32_t m = hit[h]; m; m &= m - 1) {
                    const uint32_t bit = __builtin_ctz(m), v = c + (8 * h + bit / 4) * kThreads + tid_;
                    if (v < n4) put(static_cast<uint32_t>(~(4 * v + bit % 4)));
                }
        }
        const uint32_t i = 4 * n4 + tid_;  // up to three more
        if (i < a_.vocab) {
            bool in = false;
            for (uint32_t r = 0; r < runs; r++) in = in || (x_[i] >= sm_.lo[r] && x_[i] <= sm_.hi[r]);
            if (in) put(static_cast<uint32_t>(~i));
        }
        __syncthreads();
        n_ = min(sm_.n, kList);
        // the keys of those found, all at once
        for (uint32_t k = tid_; k < n_; k += kThreads)
            sm_.list[k] |= static_cast<uint64_t>(key_of(x_[static_cast<uint32_t>(~static_cast<uint32_t>(sm_.list[k]))])) << 32;
        __syncthreads();
    }

    // f(token) for the listed tokens, or for those of the row with keys lo .. hi.
    template <class F>
    __device__ __forceinline__ void each(bool listed, uint32_t lo, uint32_t hi, const F& f) {
        if (listed) {
            for (uint32_t i = tid_; i < n_; i += kThreads) f(sm_.list[i]);
            return;
        }
        // Four logits a load, 16 loads in flight: a row is one CU's to read.  Where some of
        // a thread's are in question it puts 16 of them into LDS (the list's room), so that
        // f stands here once.
        static_assert(16 * kThreads * sizeof(float) <= sizeof(sm_.list), "room for 16 logits a thread");
        float* const mine = reinterpret_cast<float*>(sm_.list) + tid_;
        const float least = value_of(lo), most = hi >= key_of(3.402823466e38f) ? INFINITY : value_of(hi);
        const auto token = [&](float x, uint32_t i) { f(static_cast<uint64_t>(key_of(x)) << 32 | static_cast<uint32_t>(~i)); };
        typedef float v4 __attribute__((ext_vector_type(4), aligned(4)));
        constexpr uint32_t kLoads = 16;
        const uint32_t n4 = a_.vocab / 4;
        for (uint32_t c = tid_; c < n4; c += kThreads * kLoads) {
            v4 x[kLoads];
#pragma unroll
            for (uint32_t j = 0; j < kLoads; j++)
                x[j] = *reinterpret_cast<const v4*>(x_ + 4 * static_cast<size_t>(min(c + j * kThreads, n4 - 1)));
#pragma unroll
            for (uint32_t j0 = 0; j0 < kLoads; j0 += 4) {
                uint32_t hit = 0;
#pragma unroll
                for (uint32_t e = 0; e < 16; e++)
                    hit |= x[j0 + e / 4][e % 4] >= least && x[j0 + e / 4][e % 4] <= most ? 1u << e : 0u;
                if (!hit) continue;
#pragma unroll
                for (uint32_t e = 0; e < 16; e++) mine[e * kThreads] = x[j0 + e / 4][e % 4];
                for (uint32_t m = hit; m; m &= m - 1) {
                    const uint32_t e = __builtin_ctz(m), v = c + (j0 + e / 4) * kThreads;
                    if (v < n4) token(mine[e * kThreads], 4 * v + e % 4);
                }
            }
        }
        const uint32_t i = 4 * n4 + tid_;  // up to three more
        if (i < a_.vocab && x_[i] >= least && x_[i] <= most) token(x_[i], i);
    }

    // Where a goal is reached.  Its bin's tokens, among those listed or in the row, are
    // counted and weighed in 512 equal ranges of (key, ~index); so again those of the
    // range in which it is reached, until they are few; a wave decides among these.  In
    // a bin the weights are whole numbers, so every sum here is exact.  A goal is formed from
    // sums in another order than the bins' ends and may lie a rounding past those of its
    // bins in question: the nearest of these has the neighbouring token then.
    __device__ __forceinline__ Found find(const Goal& g, bool listed) {
        const uint32_t b = g.mode == kKey ? bin_of(g.n) : min(max(bin_for(g), g.b0), g.b1);
        if (b >= kBins) return {0, weight_to(kBins)};  // a key under all that has weight
        const double base = weight_to(b), scale = sm_.scale[b];
        const uint32_t before = count_to(b);
        if (g.mode == kKey && !flagged(b)) {
            // min-p's border in a bin that is in no question: another filter cuts before it
            return {static_cast<uint64_t>(g.n) << 32, base};
        }
        uint64_t lo = static_cast<uint64_t>(first_key(b)) << 32, hi = static_cast<uint64_t>(last_key(b)) << 32 | 0xffffffffu;
        uint32_t count = 0;   // of the bin's tokens above hi
        uint64_t weight = 0;  // theirs
        uint32_t n = sm_.count[b] - before;
        if (g.mode == kKey) {
            // the weight of the bin's tokens from the key on
            lo = static_cast<uint64_t>(g.n) << 32;
            uint64_t w = 0;
            each(listed, lo >> 32, hi >> 32, [&](uint64_t t) {
                if (t >= lo && t <= hi) w += weight_of(t);
            });
            w = block_scan(sm_, turn_, w);
            __syncthreads();
            if (tid_ == kThreads - 1) sm_.step_weight = w;
            __syncthreads();
            return {lo, base + static_cast<double>(sm_.step_weight) * scale};
        }
        while (n > kFinal) {
            const uint32_t sh = max(64 - __builtin_clzll(hi - lo | 511), 9) - 9;  // (hi - lo) >> sh < 512
            __syncthreads();
            sm_.sub_count[tid_] = 0;
            sm_.sub_weight[tid_] = 0;
            __syncthreads();
            each(listed, lo >> 32, hi >> 32, [&](uint64_t t) {
                if (t < lo || t > hi) return;
                const uint32_t at = static_cast<uint32_t>((hi - t) >> sh);
                atomicAdd(&sm_.sub_count[at], 1u);
                atomicAdd(&sm_.sub_weight[at], static_cast<unsigned long long>(weight_of(t)));
            });
            __syncthreads();
            const uint32_t own = sm_.sub_count[tid_];
            const uint64_t own_w = sm_.sub_weight[tid_];
            const uint32_t c = count + block_scan(sm_, turn_, own);
            const uint64_t w = weight + block_scan(sm_, turn_, own_w);
            uint32_t at = first_of(sm_, turn_, own && g.reached(before + c, base + static_cast<double>(w) * scale), tid_);
            if (at == kNone) {  // missed by a rounding: the last token
                const uint32_t from_end = first_of(sm_, turn_, sm_.sub_count[kThreads - 1 - tid_] != 0, tid_);
                if (from_end == kNone) break;  // no token: the logits are not those that were counted
                at = kThreads - 1 - from_end;
            }
            if (tid_ == at) {
                sm_.step_n = own;
                sm_.step_count = c - own;
                sm_.step_weight = w - own_w;
            }
            __syncthreads();
            n = sm_.step_n;
            count = sm_.step_count;
            weight = sm_.step_weight;
            hi -= static_cast<uint64_t>(at) << sh;
            const uint64_t width = (1ull << sh) - 1;
            if (hi - lo > width) lo = hi - width;
        }
        __syncthreads();
        if (tid_ == 0) sm_.step_n = 0;
        __syncthreads();
        each(listed, lo >> 32, hi >> 32, [&](uint64_t t) {
            if (t < lo || t > hi) return;
            const uint32_t at = atomicAdd(&sm_.step_n, 1u);
            if (at < kFinal) sm_.last[at] = t;
        });
        __syncthreads();
        n = min(sm_.step_n, kFinal);
        const uint32_t lane = tid_ & (kWave - 1);
        const uint64_t own = lane < n ? sm_.last[lane] : 0, own_w = lane < n ? weight_of(own) : 0;
        uint32_t c = count;
        uint64_t w = weight;
        for (uint32_t j = 0; j < n; j++) {  // lane j's token before this one, or itself
            const uint64_t t = lane_of(own, j), tw = lane_of(own_w, j);
            if (t >= own) {
                c++;
                w += tw;
            }
        }
        const bool yes = lane < n && g.reached(before + c, base + static_cast<double>(w) * scale);
        // the largest that reaches it; where none does (a rounding), the smallest of all
        const uint64_t most = last_lane(wave_max(yes ? own : 0)), least = ~last_lane(wave_max(lane < n ? ~own : 0));
        const uint64_t token = most ? most : least;
        const uint64_t at = __ballot(own == token && lane < n);
        const uint64_t sum = lane_of(w, at ? __builtin_ctzll(at) : 0);
        __syncthreads();
        if (n == 0) return {0, base};
        return {token, base + static_cast<double>(sum) * scale};
    }

    // A token's weight as the sums hold it.
    __device__ __forceinline__ double weight_at(uint64_t token) const {
        return static_cast<double>(weight_of(token)) * sm_.scale[min(bin_of(static_cast<uint32_t>(token >> 32)), kBins - 1)];
    }

private:
    __device__ __forceinline__ double edge_of(uint32_t key) const {
        return __builtin_floor(static_cast<double>(value_of(key)) * rate_);
    }
    __device__ __forceinline__ uint64_t weight_of(uint64_t token) const {  // in its bin's units
        const double y = static_cast<double>(value_of(static_cast<uint32_t>(token >> 32))) * rate_;
        return weight_(y - __builtin_floor(y));
    }
    __device__ __forceinline__ static uint64_t lane_of(uint64_t v, uint32_t lane) {
        return static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane))) << 32 |
               static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
    }

    const Args a_;
    Shared& sm_;
    uint32_t row_;
    double rate_;
    const float* x_;
    uint32_t tid_;
    uint64_t best_;
    double top_;
    const Weight weight_;
    uint32_t turn_ = 0, n_ = 0, own_ = 0;  // n_: tokens listed; own_: the tokens of bin tid_
};

// The smallest key that min-p keeps: e^((x - max) / T) >= p (p in (0, 1]).  The
// border is known to some 2^-52 of its terms and of T; between those the wave's lanes try
// 64 keys at a time (near 0 there can be many).
__device__ __forceinline__ uint32_t min_p_key(float top, double rate, double p) {
    const double r = rate * 0.0625, m = top, d = log(p) / r;
    const double e = m + d, slack = 1e-14 * (__builtin_fabs(m) + __builtin_fabs(d) + 1.0 / r);
    const double most = 3.402823466e38;
    const uint32_t last = key_of(top);
    uint32_t lo = max(key_of(static_cast<float>(__builtin_fmax(e - slack, -most))), 2u) - 1;
    uint32_t hi = min(key_of(static_cast<float>(__builtin_fmax(__builtin_fmin(e + slack, most), -most))) + 1, last);
    lo = min(max(lo, key_of(-3.402823466e38f)), hi);
    const uint32_t lane = threadIdx.x & (kWave - 1);
    if (hi < last && exp((static_cast<double>(value_of(hi)) - m) * r) < p) hi = last;
    while (lo < hi) {  // hi is kept; keys under lo are not
        const uint32_t step = (hi - lo + kWave - 1) / kWave, k = min(lo + lane * step, hi);
        const uint64_t kept = __ballot(exp((static_cast<double>(value_of(k)) - m) * r) >= p);
        const uint32_t i = kept ? __builtin_ctzll(kept) : kWave;
        const uint32_t from = i ? min(lo + (i - 1) * step + 1, hi) : lo;
        if (i < kWave) hi = min(lo + i * step, hi);
        lo = min(from, hi);
    }
    return hi;
}

// The filters of a row, and their parameters as loaded.
struct Filters {
    bool by_k, by_p, by_min;
    uint32_t k, min_key;
    double p, u;
};
struct Params {
    int32_t k;
    float p, min_p, u;
};

template <bool kDraw>
__device__ __forceinline__ Params params_of(const Args& a, uint32_t row) {
    return {a.top_k ? a.top_k[row] : 0, a.top_p ? a.top_p[row] : 1.0f, a.min_p ? a.min_p[row] : 0.0f, kDraw ? a.u[row] : 0.0f};
}

__device__ __forceinline__ Filters filters_of(const Params& p, double rate, uint64_t best) {
    Filters f;
    f.k = static_cast<uint32_t>(p.k);
    f.p = p.p;
    f.by_k = p.k > 0;
    f.by_p = p.p < 1.0f;
    f.by_min = p.min_p > 0.0f;
    f.min_key = f.by_min ? min_p_key(value_of(static_cast<uint32_t>(best >> 32)), rate, __builtin_fminf(p.min_p, 1.0f)) : 1;
    // u in [0, 1): what lies outside counts as the nearest that does not
    f.u = __builtin_fminf(__builtin_fmaxf(p.u, 0.0f), 0x1.fffffep-1f);
    return f;
}

// A row's slices into LDS; its largest token.
__device__ __forceinline__ uint64_t row_info(const Args& a, Shared& sm, uint32_t row) {
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1);
    if (tid < a.slices) {
        const SampleSlice s = a.info[static_cast<size_t>(row) * a.slices + tid];
        sm.best[tid] = s.best;
        sm.bins[tid] = s.bins;
        sm.n_short[tid] = s.n;
    }
    __syncthreads();
    uint64_t best = lane < a.slices ? sm.best[lane] : 0;
    if (lane + kWave < a.slices && sm.best[lane + kWave] > best) best = sm.best[lane + kWave];
    return last_lane(wave_max(best));
}

// A row's draw, or (kDraw false) what it would draw from, for thread 0, where it is true.
template <bool kDraw>
__device__ __forceinline__ bool pick(const Args& a, uint32_t row, zlm::SampleCut& to) {
    __shared__ Shared sm;
    const uint32_t tid = threadIdx.x;
    const Params params = params_of<kDraw>(a, row);
    const double rate = rate_of(a, row);
    Row::Ahead ahead;
    if (rate != 0.0) Row::read_ahead(a, row, 0, ahead);
    const uint64_t best = row_info(a, sm, row);
    if (best == 0 || rate == 0.0) {  // nothing to draw; temperature 0: the largest
        if (!kDraw) {
            to = {0, best, 0.0, 0.0, 0.0};
        } else if (tid == 0) {
            a.token[row] = best ? static_cast<int32_t>(~static_cast<uint32_t>(best)) : -1;
            if (a.prob) a.prob[row] = best ? 1.0f : 0.0f;
        }
        return tid == 0;
    }
    const Filters f = filters_of(params, rate, best);
    Row r(a, sm, row, rate, best);
    r.join(ahead);
    const double total = r.weight_to(kBins);
    const bool by_k = f.by_k && f.k < r.count_to(kBins);
    // The bins in question.  A cut falls within a bin, so the weight that is left after
    // it lies between two bins' ends, and the next goal in the bins that these make.
    double w0 = total, w1 = total;
    uint32_t k_bin = 0, p_bins[2] = {0, 0};
    if (by_k) {
        k_bin = r.bin_for({kCount, 0.0, f.k});
        r.flag(k_bin, k_bin);
        w0 = r.weight_to(k_bin);
        w1 = r.weight_to(k_bin + 1);
    }
    if (f.by_p) {
        r.bins_for(kAtLeast, w0 * f.p, w1 * f.p, p_bins);
        w0 = r.weight_to(p_bins[0]);
        w1 = __builtin_fmin(w1, r.weight_to(p_bins[1] + 1));
    }
    if (f.by_min) {
        const uint32_t b = r.bin_of(f.min_key);
        if (b < kBins && r.weight_to(b) < w1) {
            r.flag(b, b);
            w0 = __builtin_fmin(w0, r.weight_to(b));
            w1 = __builtin_fmin(w1, r.weight_to(b + 1));
        }
    }
    uint32_t u_bins[2] = {0, 0};
    if constexpr (kDraw) {
        r.bins_for(kMore, w0 * f.u, w1 * f.u, u_bins);
    } else if (!by_k && !f.by_p && !f.by_min) {  // all that have weight
        to = {0, best, total, rate, 0.0};
        return tid == 0;
    }
    const bool listed = r.in_question() <= kList;
    if (listed && !r.list_shorts(ahead)) r.list_row();
    // the filters in turn, then the draw
    Found cut = {0, total};  // the last token kept, and the weight of all that are
    double p_weight = total;
    for (int step = 0; step < (kDraw ? 4 : 3); step++) {
        Goal g = {kMore, cut.weight * f.u, 0, u_bins[0], u_bins[1]};  // the draw
        if (step == 0) {
            if (!by_k) continue;
            g = {kCount, 0.0, f.k, k_bin, k_bin};
        } else if (step == 1) {
            p_weight = cut.weight * f.p;  // top-p is of what top-k left
            if (!f.by_min || f.min_key <= cut.token >> 32) continue;
            g = {kKey, 0.0, f.min_key};
        } else if (step == 2) {
            if (!f.by_p || p_weight >= cut.weight) continue;
            g = {kAtLeast, p_weight, 0, p_bins[0], p_bins[1]};
        }
        const Found t = r.find(g, listed);
        if (step < 3) {
            if (t.token > cut.token) cut = t;
        } else if (tid == 0) {
            a.token[row] = static_cast<int32_t>(~static_cast<uint32_t>(t.token));
            if (a.prob) a.prob[row] = t.token ? static_cast<float>(r.weight_at(t.token) / cut.weight) : 0.0f;
        }
    }
    if constexpr (!kDraw) to = {cut.token, best, cut.weight, rate, 0.0};
    return tid == 0;
}

}  // namespace

