// zlm_sample.hip -- CDNA4 (gfx950) kernels that draw a token from each row of
// logits by temperature, top-k, top-p and min-p with a given uniform number.
// Built as a device-only code object (hipcc --genco) and loaded by the host
// library.
//
// The tokens in order of probability (the lower index first among equals) are
// x_1 >= x_2 >= ..; every filter keeps a prefix of that order, and the draw takes
// the first token whose cumulative weight exceeds u times that of the prefix.  So
// each step asks where a cumulative count or weight is reached, and no sort of the
// row is needed: a histogram by value answers to within a bin, and only the bin in
// question is looked at token by token.
//
// Weights.  y = 16 x / T in 64 bits; bin floor(y), 1/16 of a temperature wide, on a
// grid that does not depend on the row's maximum, so the slices of a row need no
// pass for it.  A token's weight relative to its bin's upper edge, in (0.939, 1],
// is held as an integer of 2^-34: the sums of a bin are exact in any order, a
// bin's sum times e^(-bin/16) in 64 bits.  512 bins reach e^-32 below the largest:
// what lies under that has no weight (all of 2^20 such tokens are 1.3e-8 of it,
// less than the step of u).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sample_args.h"

// y, its bin and the distance between them come from one rounded product: where
// logits are large, an fma of it would be another number.
#pragma clang fp contract(off)

namespace {

using Args = zlm::SampleArgs;
using zlm::SampleSlice;
constexpr uint32_t kWave = 64, kThreads = 1024;
constexpr uint32_t kSlice = zlm::kSampleSlice, kBins = zlm::kSampleBins, kSlices = zlm::kSampleSlices;
constexpr uint32_t kShort = zlm::kSampleShort;
constexpr uint32_t kPer = kSlice / kThreads;
constexpr uint32_t kList = 4096;  // tokens that are looked at one by one
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

// e^z, z in [-1/16, 0]: the series to z^6 (the rest is under 8e-13, a fiftieth of
// the unit that weights are held in).
__device__ __forceinline__ double exp_small(double z) {
    double r = 1.0 / 720;
    r = __builtin_fma(r, z, 1.0 / 120);
    r = __builtin_fma(r, z, 1.0 / 24);
    r = __builtin_fma(r, z, 1.0 / 6);
    r = __builtin_fma(r, z, 0.5);
    r = __builtin_fma(r, z, 1.0);
    return __builtin_fma(r, z, 1.0);
}

// The weight of y in its bin, in units of 2^-34.
__device__ __forceinline__ uint64_t weight_of(double y, double bin) {
    const double e = exp_small((y - (bin + 1.0)) * 0.0625);
    const double d = __builtin_fma(e, kUnit, 4503599627370496.0);  // + 2^52: the integer in the low bits
    return __builtin_bit_cast(uint64_t, d) & 0xfffffffffffffull;
}

__device__ __forceinline__ double rate_of(const Args& a, uint32_t row) {  // 16 / T; 0: greedy
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    return t > 0.0f ? 16.0 / static_cast<double>(__builtin_fminf(t, 3.402823466e38f)) : 0.0;
}

__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t w = __shfl_xor(v, o);
        v = w > v ? w : v;
    }
    return v;
}

// One slice of a row: its largest logit, the histogram below it, and the short list
// of the tokens that most draws are decided among.
__device__ __forceinline__ void slice_hist(const Args& a) {
    __shared__ unsigned long long hist[kBins];
    __shared__ uint64_t best_of[kThreads / kWave];
    __shared__ uint32_t ends[kBins / kWave], n_short, n_bins;
    const uint32_t tid = threadIdx.x, s = blockIdx.x, row = blockIdx.y, lane = tid & (kWave - 1), wid = tid / kWave;
    const float* x = a.logits + row * a.stride;
    const double rate = rate_of(a, row);
    uint32_t key[kPer];
    uint64_t best = 0;
#pragma unroll
    for (uint32_t j = 0; j < kPer; j++) {
        const uint32_t i = s * kSlice + j * kThreads + tid;
        key[j] = i < a.vocab ? key_of(x[i]) : 0;
    }
#pragma unroll
    for (uint32_t j = 0; j < kPer; j++) {
        const uint32_t i = s * kSlice + j * kThreads + tid;
        const uint64_t c = key[j] ? static_cast<uint64_t>(key[j]) << 32 | ~i : 0;
        best = c > best ? c : best;
    }
    best = wave_max(best);
    if (lane == 0) best_of[wid] = best;
    if (tid < kBins) hist[tid] = 0;
    if (tid == 0) n_short = n_bins = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kThreads / kWave; w++) best = best_of[w] > best ? best_of[w] : best;
    const size_t at = static_cast<size_t>(row) * a.slices + s;
    if (best == 0 || rate == 0.0) {
        if (tid == 0) a.info[at] = {best, 0, 0};
        return;
    }
    const double top = __builtin_floor(static_cast<double>(value_of(static_cast<uint32_t>(best >> 32))) * rate);
    uint32_t bin[kPer];
#pragma unroll
    for (uint32_t j = 0; j < kPer; j++) {
        const double y = static_cast<double>(value_of(key[j])) * rate, b = __builtin_floor(y);
        const double d = top - b;
        bin[j] = kBins;
        if (key[j] && d < static_cast<double>(kBins)) {
            bin[j] = static_cast<uint32_t>(d);
            atomicAdd(&hist[bin[j]], (1ull << kCountShift) + weight_of(y, b));
        }
    }
    __syncthreads();
    // the bins that the short list has room for
    uint32_t c = 0;
    if (tid < kBins) {
        const uint64_t h = hist[tid];
        a.hist[at * kBins + tid] = h;
        c = static_cast<uint32_t>(h >> kCountShift);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t y = __shfl_up(c, o);
            if (static_cast<int>(lane) >= o) c += y;
        }
        if (lane == kWave - 1) ends[wid] = c;
    }
    __syncthreads();
    if (tid < kBins) {
        for (uint32_t w = 0; w < wid; w++) c += ends[w];
        const uint64_t fits = __ballot(c <= kShort);
        if (lane == 0 && fits) atomicAdd(&n_bins, static_cast<uint32_t>(__builtin_popcountll(fits)));
    }
    __syncthreads();
    const uint32_t bins = n_bins;
#pragma unroll
    for (uint32_t j = 0; j < kPer; j++)
        if (bin[j] < bins)
            a.shorts[at * kShort + atomicAdd(&n_short, 1u)] =
                static_cast<uint64_t>(key[j]) << 32 | ~(s * kSlice + j * kThreads + tid);
    __syncthreads();
    if (tid == 0) a.info[at] = {best, bins, n_short};
}

struct Shared {
    uint64_t list[kList];  // tokens of bins g0 .. g1 (or of a key's range), largest first: key, ~index
    double cum[kList];     // their cumulative weights
    double weight[kBins];  // cumulative, all bins up to and with this one
    uint32_t count[kBins];
    uint64_t best[kSlices];
    uint32_t shift[kSlices];  // a slice's top bin below the row's (kBins: no tokens with weight)
    uint32_t bins[kSlices], n_short[kSlices];
    uint32_t need[kSlices];  // the slices to look through
    uint32_t n_need;
    uint32_t sub_count[kThreads];
    unsigned long long sub_weight[kThreads];
    double part_w[kThreads / kWave];
    uint32_t part_c[kThreads / kWave];
    uint32_t n, at, lo, hi;
    double base;
};

// Inclusive sums over the workgroup in thread order.
__device__ __forceinline__ void block_scan(Shared& sm, uint32_t& c, double& w) {
    const uint32_t lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t cc = __shfl_up(c, o);
        const double ww = __shfl_up(w, o);
        if (static_cast<int>(lane) >= o) {
            c += cc;
            w += ww;
        }
    }
    __syncthreads();
    if (lane == kWave - 1) {
        sm.part_c[wid] = c;
        sm.part_w[wid] = w;
    }
    __syncthreads();
    uint32_t bc = 0;
    double bw = 0.0;
    for (uint32_t i = 0; i < wid; i++) {
        bc += sm.part_c[i];
        bw += sm.part_w[i];
    }
    c += bc;
    w = bw + w;
}

// The first thread of those that say yes, or kThreads.
__device__ __forceinline__ uint32_t first_of(Shared& sm, bool yes) {
    __syncthreads();
    if (threadIdx.x == 0) sm.at = kThreads;
    __syncthreads();
    const uint64_t m = __ballot(yes);
    if (m && (threadIdx.x & (kWave - 1)) == 0) atomicMin(&sm.at, threadIdx.x + __builtin_ctzll(m));
    __syncthreads();
    return sm.at;
}

// What a search looks for.
enum Mode { kCount, kAtLeast, kMore, kKey };
struct Goal {
    Mode mode;
    double w;      // kAtLeast, kMore: the cumulative weight
    uint32_t n;    // kCount: how many tokens; kKey: the smallest key
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
    __device__ Row(const Args& a, Shared& sm, uint32_t row, double rate)
        : a_(a), sm_(sm), row_(row), rate_(rate), x_(a.logits + row * a.stride), tid_(threadIdx.x) {}

    // The slices' histograms as the row's: cumulative counts and weights by bin.
    __device__ __forceinline__ void join(uint64_t best) {
        best_ = best;
        top_ = edge_of(static_cast<uint32_t>(best >> 32));
        if (tid_ < a_.slices) {
            const uint64_t b = sm_.best[tid_];
            sm_.shift[tid_] = b ? static_cast<uint32_t>(__builtin_fmin(top_ - edge_of(static_cast<uint32_t>(b >> 32)), 1.0 * kBins)) : kBins;
        }
        __syncthreads();
        // the lower half of the threads takes the even slices, the upper the odd ones
        const uint32_t bin = tid_ % kBins;
        uint32_t c = 0;
        uint64_t w = 0;
        const uint64_t* hist = a_.hist + static_cast<size_t>(row_) * a_.slices * kBins;
#pragma unroll 4
        for (uint32_t s = tid_ / kBins; s < a_.slices; s += kThreads / kBins) {
            const uint32_t shift = sm_.shift[s];
            const uint64_t h = bin >= shift ? hist[static_cast<size_t>(s) * kBins + bin - shift] : 0;
            c += static_cast<uint32_t>(h >> kCountShift);
            w += h & ((1ull << kCountShift) - 1);
        }
        if (tid_ >= kBins) {
            sm_.sub_count[bin] = c;
            sm_.sub_weight[bin] = w;
        }
        __syncthreads();
        double ww = 0.0;
        if (tid_ < kBins) {
            c += sm_.sub_count[bin];
            ww = static_cast<double>(w + sm_.sub_weight[bin]) * scale_of(bin);
        } else {
            c = 0;
        }
        block_scan(sm_, c, ww);
        if (tid_ < kBins) {
            sm_.count[tid_] = c;
            sm_.weight[tid_] = ww;
        }
        __syncthreads();
    }

    __device__ __forceinline__ double total() const { return sm_.weight[kBins - 1]; }
    __device__ __forceinline__ uint32_t tokens() const { return sm_.count[kBins - 1]; }
    __device__ __forceinline__ uint32_t count_to(uint32_t bin) const { return sm_.count[bin]; }

    // The smallest and the largest key of a bin: the border is known to a rounding,
    // the wave's lanes try the 64 keys around it.
    __device__ __forceinline__ uint32_t first_key(uint32_t bin) const {
        const double edge = top_ - static_cast<double>(bin);
        const double e = __builtin_fmax(__builtin_fmin(edge / rate_, 3.402823466e38), -3.402823466e38);
        const uint32_t k = key_of(static_cast<float>(e)) - 31 + (tid_ & (kWave - 1));
        const uint64_t in = __ballot(static_cast<double>(value_of(k)) * rate_ >= edge);
        return key_of(static_cast<float>(e)) - 31 + (in ? __builtin_ctzll(in) : kWave);
    }
    __device__ __forceinline__ uint32_t last_key(uint32_t bin) const {
        return bin ? first_key(bin - 1) - 1 : static_cast<uint32_t>(best_ >> 32);
    }

    __device__ __forceinline__ uint32_t bin_of(uint32_t key) const {  // kBins: below them
        const double d = top_ - edge_of(key);
        return d < 1.0 * kBins ? static_cast<uint32_t>(__builtin_fmax(d, 0.0)) : kBins;
    }

    // The first bin by whose end the goal is reached (kBins: none).
    __device__ __forceinline__ uint32_t bin_for(const Goal& g) {
        if (g.mode == kKey) return bin_of(g.n);
        const uint32_t b = first_of(sm_, tid_ < kBins && g.reached(sm_.count[tid_ % kBins], sm_.weight[tid_ % kBins]));
        return b < kBins ? b : kBins;
    }

    // The list: tokens of bins g0 .. g1 with keys lo .. hi, sorted, with cumulative
    // weights from `base`.  The caller knows that there are at most kList.
    __device__ __forceinline__ void gather(uint32_t g0, uint32_t g1, uint32_t lo, uint32_t hi, double base) {
        __syncthreads();
        if (tid_ == 0) sm_.n = 0;
        mark(g0, g1, true);
        const auto take = [&](uint32_t key, uint32_t i) {
            if (key < lo || key > hi) return;
            const uint32_t at = atomicAdd(&sm_.n, 1u);
            if (at < kList) sm_.list[at] = static_cast<uint64_t>(key) << 32 | ~i;
        };
        // short lists, four slices at a time
        const uint64_t* shorts = a_.shorts + static_cast<size_t>(row_) * a_.slices * kShort;
#pragma unroll 4
        for (uint32_t s = tid_ / kShort; s < a_.slices; s += kThreads / kShort) {
            const uint32_t shift = sm_.shift[s];
            if (shift > g1 || g1 - shift >= sm_.bins[s] || tid_ % kShort >= sm_.n_short[s]) continue;
            const uint64_t t = shorts[static_cast<size_t>(s) * kShort + tid_ % kShort];
            take(static_cast<uint32_t>(t >> 32), ~static_cast<uint32_t>(t));
        }
        each_needed([&](uint32_t key, uint32_t i) { take(key, i); });
        __syncthreads();
        n_ = min(sm_.n, kList);
        uint32_t len = 64;
        while (len < n_) len *= 2;
        for (uint32_t i = n_ + tid_; i < len; i += kThreads) sm_.list[i] = 0;
        sort(len);
        // cumulative weights, a run of tokens a thread
        const uint32_t per = (n_ + kThreads - 1) / kThreads;
        double w[kList / kThreads], sum = 0.0;
#pragma unroll
        for (uint32_t j = 0; j < kList / kThreads; j++) {
            const uint32_t i = tid_ * per + j;
            w[j] = j < per && i < n_ ? weight_at(static_cast<uint32_t>(sm_.list[i] >> 32)) : 0.0;
            sum += w[j];
        }
        uint32_t none = 0;
        double run = sum;
        block_scan(sm_, none, run);
        run = base + (run - sum);
#pragma unroll
        for (uint32_t j = 0; j < kList / kThreads; j++) {
            const uint32_t i = tid_ * per + j;
            run += w[j];
            if (j < per && i < n_) sm_.cum[i] = run;
        }
        g0_ = g0;
        g1_ = g1;
        __syncthreads();
    }

    __device__ __forceinline__ Found find(const Goal& g) {
        uint32_t b = bin_for(g);
        if (b >= kBins) {  // all that has weight (a goal missed by a rounding, or a key under all)
            return {0, total()};
        }
        const uint32_t before = b ? sm_.count[b - 1] : 0;
        const double base = b ? sm_.weight[b - 1] : 0.0;
        if (b < g0_ || b > g1_) {
            if (sm_.count[b] - before > kList) return refine(g, b, before, base);
            gather(b, b, first_key(b), last_key(b), base);
        }
        return in_list(g, g0_ ? sm_.count[g0_ - 1] : 0, g0_ ? sm_.weight[g0_ - 1] : 0.0);
    }

    __device__ __forceinline__ double weight_at(uint32_t key) const {
        const double y = static_cast<double>(value_of(key)) * rate_, b = __builtin_floor(y);
        return static_cast<double>(weight_of(y, b)) * scale_of(static_cast<uint32_t>(top_ - b));
    }

private:
    __device__ __forceinline__ static double scale_of(uint32_t bin) { return exp(static_cast<double>(bin) * -0.0625) / kUnit; }

    __device__ __forceinline__ double edge_of(uint32_t key) const {
        return __builtin_floor(static_cast<double>(value_of(key)) * rate_);
    }

    // Which slices have tokens in bins g0 .. g1 (more than one bin: may have), but not
    // (with `beyond`) all of them in their short lists.
    __device__ __forceinline__ void mark(uint32_t g0, uint32_t g1, bool beyond) {
        if (tid_ == 0) sm_.n_need = 0;
        __syncthreads();
        if (tid_ < a_.slices) {
            const uint32_t shift = sm_.shift[tid_];
            bool need = shift <= g1 && !(beyond && g1 - shift < sm_.bins[tid_]);
            if (need && g0 == g1)
                need = (a_.hist[(static_cast<size_t>(row_) * a_.slices + tid_) * kBins + g0 - shift] >> kCountShift) != 0;
            if (need) sm_.need[atomicAdd(&sm_.n_need, 1u)] = tid_;
        }
        __syncthreads();
    }

    // f(key, index) for every logit of the needed slices (key 0: not to be drawn), four
    // slices' loads in flight at once.
    template <class F>
    __device__ __forceinline__ void each_needed(const F& f) const {
        constexpr uint32_t kAtOnce = 4;
        const uint32_t n = sm_.n_need;
        for (uint32_t b = 0; b < n; b += kAtOnce) {
            float x[kAtOnce][kPer];
            uint32_t i0[kAtOnce];
#pragma unroll
            for (uint32_t g = 0; g < kAtOnce; g++) {
                i0[g] = b + g < n ? sm_.need[b + g] * kSlice + tid_ : a_.vocab;
#pragma unroll
                for (uint32_t j = 0; j < kPer; j++)
                    x[g][j] = i0[g] + j * kThreads < a_.vocab ? x_[i0[g] + j * kThreads] : -INFINITY;
            }
#pragma unroll
            for (uint32_t g = 0; g < kAtOnce; g++)
#pragma unroll
                for (uint32_t j = 0; j < kPer; j++) f(key_of(x[g][j]), i0[g] + j * kThreads);
        }
    }

    __device__ __forceinline__ void sort(uint32_t len) {  // largest first; len a power of two
        for (uint32_t size = 2; size <= len; size *= 2)
            for (uint32_t step = size / 2; step > 0; step /= 2) {
                __syncthreads();
                for (uint32_t t = tid_; t < len / 2; t += kThreads) {
                    const uint32_t i = 2 * t - (t & (step - 1)), j = i + step;
                    const uint64_t p = sm_.list[i], q = sm_.list[j];
                    if ((p < q) == ((i & size) == 0)) {
                        sm_.list[i] = q;
                        sm_.list[j] = p;
                    }
                }
            }
        __syncthreads();
    }

    // The goal in the list, whose tokens come after `before` others with weight `base`.
    __device__ __forceinline__ Found in_list(const Goal& g, uint32_t before, double base) {
        __syncthreads();
        if (tid_ == 0) sm_.lo = n_;
        __syncthreads();
        for (uint32_t i = tid_; i < n_; i += kThreads) {
            const bool yes = g.mode == kKey ? static_cast<uint32_t>(sm_.list[i] >> 32) < g.n
                                            : g.reached(before + i + 1, sm_.cum[i]);
            if (yes) atomicMin(&sm_.lo, i);
        }
        __syncthreads();
        uint32_t i = sm_.lo;
        if (g.mode == kKey) {  // i: the first that is too small
            if (i == 0) return {static_cast<uint64_t>(g.n) << 32, base};
            return {static_cast<uint64_t>(g.n) << 32, sm_.cum[i - 1]};
        }
        if (i >= n_) i = n_ - 1;
        return {sm_.list[i], sm_.cum[i]};
    }

    // A goal in a bin of more than kList tokens: histograms of ever narrower ranges
    // of keys, until the list holds one, or one key is left: then its tokens count
    // in order of their index.
    __device__ __forceinline__ Found refine(const Goal& g, uint32_t b, uint32_t before, double base) {
        const double scale = scale_of(b);
        mark(b, b, false);
        uint32_t lo = first_key(b), hi = last_key(b);
        if (g.mode == kKey && g.n > hi) return {static_cast<uint64_t>(g.n) << 32, base};
        for (;;) {
            uint32_t sh = 0;
            while (((hi - lo) >> sh) >= kThreads) sh++;
            __syncthreads();
            sm_.sub_count[tid_] = 0;
            sm_.sub_weight[tid_] = 0;
            __syncthreads();
            each_needed([&](uint32_t key, uint32_t) {
                if (key < lo || key > hi) return;
                const double y = static_cast<double>(value_of(key)) * rate_;
                atomicAdd(&sm_.sub_count[(hi - key) >> sh], 1u);
                atomicAdd(&sm_.sub_weight[(hi - key) >> sh], static_cast<unsigned long long>(weight_of(y, __builtin_floor(y))));
            });
            __syncthreads();
            const uint32_t own = sm_.sub_count[tid_];
            const double own_w = static_cast<double>(sm_.sub_weight[tid_]);
            uint32_t c = own;
            double w = own_w;  // whole numbers under 2^54, sums exact to 2^53
            block_scan(sm_, c, w);
            uint32_t at;
            if (g.mode == kKey) at = g.n > lo ? (hi - g.n) >> sh : (hi - lo) >> sh;
            else at = first_of(sm_, own && g.reached(before + c, base + w * scale));
            if (at == kThreads) at = (hi - lo) >> sh;
            __syncthreads();
            if (tid_ == at) {
                sm_.n = own;
                sm_.lo = before + c - own;
                sm_.base = base + (w - own_w) * scale;
            }
            __syncthreads();
            const uint32_t n = sm_.n;
            before = sm_.lo;
            base = sm_.base;
            hi -= at << sh;
            lo = max(lo, hi - ((1u << sh) - 1));
            if (n <= kList) {
                gather(b, b, lo, hi, base);
                g0_ = 1;  // the list is no whole bin's
                g1_ = 0;
                return in_list(g, before, base);
            }
            if (sh == 0) return in_ties(g, b, lo, n, before, base);
        }
    }

    // A goal among n tokens of one key.
    __device__ __forceinline__ Found in_ties(const Goal& g, uint32_t b, uint32_t key, uint32_t n, uint32_t before, double base) {
        const double w = weight_at(key);
        uint32_t t = n;  // how many of them the goal takes
        if (g.mode == kKey) return {static_cast<uint64_t>(g.n) << 32, base + (key >= g.n ? n * w : 0.0)};
        if (g.mode == kCount) {
            t = g.n - before;
        } else {
            t = static_cast<uint32_t>(__builtin_fmin(__builtin_fmax((g.w - base) / w - 2.0, 0.0), 1.0 * n - 1)) + 1;
            while (t < n && !g.reached(0, base + t * w)) t++;
        }
        t = min(max(t, 1u), n);
        // the t-th in order of index
        uint32_t left = t, at = 0;
        for (uint32_t s = 0; s < a_.slices; s++) {
            if (sm_.shift[s] > b) continue;
            for (uint32_t j = 0; j < kPer; j++) {
                const uint32_t i = s * kSlice + j * kThreads + tid_;
                const bool yes = i < a_.vocab && key_of(x_[i]) == key;
                uint32_t c = yes;
                double none = 0.0;
                block_scan(sm_, c, none);
                const uint32_t hit = first_of(sm_, yes && c == left);
                if (hit < kThreads) {
                    at = s * kSlice + j * kThreads + hit;
                    return {static_cast<uint64_t>(key) << 32 | ~at, base + t * w};
                }
                __syncthreads();
                if (tid_ == kThreads - 1) sm_.lo = c;
                __syncthreads();
                left -= sm_.lo;
            }
        }
        return {static_cast<uint64_t>(key) << 32 | ~at, base + t * w};
    }

    const Args& a_;
    Shared& sm_;
    uint32_t row_;
    double rate_;
    const float* x_;
    uint32_t tid_;
    double top_ = 0.0;
    uint64_t best_ = 0;
    uint32_t n_ = 0, g0_ = 1, g1_ = 0;  // the list's tokens and bins
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

__device__ __forceinline__ void pick(const Args& a) {
    __shared__ Shared sm;
    const uint32_t tid = threadIdx.x, row = blockIdx.x;
    const double rate = rate_of(a, row);
    if (tid < a.slices) {
        const SampleSlice s = a.info[static_cast<size_t>(row) * a.slices + tid];
        sm.best[tid] = s.best;
        sm.bins[tid] = s.bins;
        sm.n_short[tid] = s.n;
    }
    __syncthreads();
    const uint32_t lane = tid & (kWave - 1);
    uint64_t best = lane < a.slices ? sm.best[lane] : 0;
    if (lane + kWave < a.slices && sm.best[lane + kWave] > best) best = sm.best[lane + kWave];
    best = wave_max(best);
    if (best == 0 || rate == 0.0) {  // nothing to draw; temperature 0: the largest
        if (tid == 0) {
            a.token[row] = best ? static_cast<int32_t>(~static_cast<uint32_t>(best)) : -1;
            if (a.prob) a.prob[row] = best ? 1.0f : 0.0f;
        }
        return;
    }
    Row r(a, sm, row, rate);
    r.join(best);
    const int32_t k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f, mp = a.min_p ? a.min_p[row] : 0.0f;
    const bool by_k = k > 0 && static_cast<uint32_t>(k) < r.tokens(), by_p = p < 1.0f, by_min = mp > 0.0f;
    const uint32_t min_key =
        by_min ? min_p_key(value_of(static_cast<uint32_t>(best >> 32)), rate, __builtin_fmin(mp, 1.0f)) : 1;
    // the bins that any filter may leave: where they hold few tokens, all of these are listed at once
    uint32_t last = kBins;
    if (by_k) last = min(last, r.bin_for({kCount, 0.0, static_cast<uint32_t>(k)}));
    if (by_p) last = min(last, r.bin_for({kAtLeast, r.total() * p, 0}));
    if (by_min) last = min(last, r.bin_of(min_key));
    last = min(last, kBins - 1);
    if (r.count_to(last) <= kList) r.gather(0, last, r.first_key(last), r.last_key(0), 0.0);
    // u in [0, 1): what lies outside counts as the nearest that does not
    const double u = __builtin_fminf(__builtin_fmaxf(a.u[row], 0.0f), 0x1.fffffep-1f);
    Found cut = {0, r.total()};  // the last token kept, and the weight of all that are
    double p_weight = cut.weight;
    for (int step = 0; step < 4; step++) {
        Goal g = {kMore, cut.weight * u, 0};  // the draw
        if (step == 0) {
            if (!by_k) continue;
            g = {kCount, 0.0, static_cast<uint32_t>(k)};
        } else if (step == 1) {
            p_weight = cut.weight * p;  // top-p is of what top-k left
            if (!by_min || min_key <= cut.token >> 32) continue;
            g = {kKey, 0.0, min_key};
        } else if (step == 2) {
            if (!by_p || p_weight >= cut.weight) continue;
            g = {kAtLeast, p_weight, 0};
        }
        const Found f = r.find(g);
        if (step < 3) {
            if (f.token > cut.token) cut = f;
        } else if (tid == 0) {
            a.token[row] = static_cast<int32_t>(~static_cast<uint32_t>(f.token));
            if (a.prob)
                a.prob[row] = static_cast<float>(r.weight_at(static_cast<uint32_t>(f.token >> 32)) / cut.weight);
        }
    }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(1024) zlm_sample_hist(Args a) { slice_hist(a); }
extern "C" __global__ void __launch_bounds__(1024) zlm_sample_pick(Args a) { pick(a); }
