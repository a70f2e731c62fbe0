// zlm_verify.hip -- CDNA4 (gfx950) kernels that verify drafted tokens against a target's
// logits with given uniform numbers, so that what comes out has the target's distribution.
// Built as a device-only code object (hipcc --genco) and loaded by the host library.
//
// With p and q what the sampler draws a row's tokens by from the target's and from the
// draft's logits (temperature, top-k, top-p, min-p; sample_impl.h), a sequence's drafted
// tokens d are accepted one after another while u q(d) < p(d).  The first that is not makes
// way for a token drawn from max(p - q, 0), in order of index; where all are, one more is
// drawn from the last row's p.  Three launches:
//   hist  the sampler's histograms of all rows, target's and draft's
//   cuts  the sampler's search of all rows: what is kept of each, and its weight
//   draw  a workgroup for each 8192 tokens of a sequence: it decides which row ends the
//         drafts (a few loads), and sums up its part of what is drawn from; the last of a
//         sequence's to be done adds up the parts and looks the token up in its part
#include "sample_impl.h"

namespace {

using VArgs = zlm::VerifyArgs;
using Cut = zlm::SampleCut;
using Sum = zlm::VerifySum;
constexpr uint32_t kDrawThreads = 512, kDrawPer = kSlice / kDrawThreads;

// Whether a draw may look at row r: 0 no, 1 a sequence's last (the draft has none there), 2 yes.
__device__ __forceinline__ uint32_t use_of(const VArgs& v, uint32_t r) {
    const uint32_t lane = threadIdx.x & (kWave - 1);
    bool last = false, in = false;
    for (uint32_t b = 0; b < v.n_seqs; b += kWave) {
        const uint32_t s = min(b + lane, v.n_seqs - 1);
        const int64_t from = v.q_start[s], to = v.q_start[s + 1];
        const bool has = from >= 0 && from <= r && r < to;
        last = last || __any(has && (to == r + 1 || r + 1 == v.n_rows));
        in = in || __any(has);
    }
    return last ? 1 : in ? 2 : 0;
}

// The row that a workgroup of the first two launches works on; false: none.
__device__ __forceinline__ bool row_of(const VArgs& v, uint32_t i, bool& draft, uint32_t& row) {
    draft = i >= v.target.rows;
    row = draft ? i - v.target.rows : i;
    return use_of(v, v.first + row) > (draft ? 1u : 0u);
}

template <uint32_t kHistThreads>
__device__ __forceinline__ void hist(const VArgs& v) {
    bool draft;
    uint32_t row;
    if (!row_of(v, blockIdx.y, draft, row)) return;
    slice_hist<kHistThreads>(draft ? v.draft : v.target, row);
}

__device__ __forceinline__ void cuts(const VArgs& v) {
    if (v.first == 0 && blockIdx.x == 0)  // for the launch after this
        for (uint32_t s = threadIdx.x; s < v.n_seqs; s += kThreads) v.counts[s] = 0;
    bool draft;
    uint32_t row;
    if (!row_of(v, blockIdx.x, draft, row)) return;
    pick<false>(draft ? v.draft : v.target, row, v.cuts + (draft ? v.n_rows : 0) + v.first + row);
}

// A row's tokens by their shares.
struct Share {
    Cut cut;
    double top, inv;
    const double* scale;  // e^(-bin/16) in units of the weights
    __device__ __forceinline__ Share(const Cut& c, const double* scales) : cut(c), scale(scales) {
        top = __builtin_floor(static_cast<double>(value_of(static_cast<uint32_t>(c.best >> 32))) * c.rate);
        inv = c.weight > 0.0 ? 1.0 / c.weight : 0.0;
    }
    // (weight: a Weight, whose coefficients stay where they are)
    __device__ __forceinline__ double operator()(float x, uint32_t i, const Weight& weight) const {
        const uint64_t token = static_cast<uint64_t>(key_of(x)) << 32 | static_cast<uint32_t>(~i);
        if (cut.rate == 0.0) return token == cut.best && token >> 32 ? 1.0 : 0.0;
        if (token >> 32 == 0 || token < cut.token) return 0.0;
        const double y = static_cast<double>(value_of(static_cast<uint32_t>(token >> 32))) * cut.rate, b = __builtin_floor(y);
        const double d = top - b;
        if (!(d < 1.0 * kBins)) return 0.0;
        return static_cast<double>(weight(y - b)) * scale[static_cast<uint32_t>(__builtin_fmax(d, 0.0))] * inv;
    }
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

__device__ __forceinline__ void put(double* p, double v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double get(const double* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

struct DrawShared {
    double scale[kBins];
    double part[2][kDrawThreads / kWave];
    uint32_t stop, last, at;
    double goal;
};

// A thread's tokens, kDrawPer in a row: what is drawn from, and the target's shares.
struct Rows {
    const float *p, *q;  // q null: none, or a certain token
    Share ps, qs;
    uint32_t certain;    // that token, or none
};

__device__ __forceinline__ void weigh(const VArgs& v, const Rows& r, const Weight& weight, uint32_t i0, double (&rest)[kDrawPer],
                                      double (&all)[kDrawPer]) {
    const uint32_t vocab = v.target.vocab;
    float x[kDrawPer], y[kDrawPer];
    typedef float v4 __attribute__((ext_vector_type(4), aligned(4)));
    if (i0 + kDrawPer <= vocab) {
#pragma unroll
        for (uint32_t j = 0; j < kDrawPer; j += 4) {
            const v4 a = *reinterpret_cast<const v4*>(r.p + i0 + j), b = *reinterpret_cast<const v4*>((r.q ? r.q : r.p) + i0 + j);
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                x[j + e] = a[e];
                y[j + e] = b[e];
            }
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < kDrawPer; j++) {
            x[j] = i0 + j < vocab ? r.p[i0 + j] : -INFINITY;
            y[j] = r.q && i0 + j < vocab ? r.q[i0 + j] : -INFINITY;
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < kDrawPer; j++) {
        const double p = r.ps(x[j], i0 + j, weight);
        const double q = r.q ? r.qs(y[j], i0 + j, weight) : i0 + j == r.certain ? 1.0 : 0.0;
        all[j] = p;
        rest[j] = p > q ? p - q : 0.0;
    }
}

__device__ __forceinline__ void draw(const VArgs& v) {
    __shared__ DrawShared sm;
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
    const uint32_t slice = blockIdx.x, s = blockIdx.y, slices = v.target.slices;
    const int32_t from = v.q_start[s], to = min(v.q_start[s + 1], static_cast<int32_t>(v.n_rows));
    if (from < 0 || from >= to) {  // no rows
        if (slice == 0 && tid == 0) v.accepted[s] = 0;
        return;
    }
    const uint32_t row0 = from, n = static_cast<uint32_t>(to - from), vocab = v.target.vocab;
    const Weight weight;
    sm.scale[tid] = exp(static_cast<double>(tid) * -0.0625) / kUnit;
    static_assert(kDrawThreads == kBins, "a bin a thread");
    if (tid == 0) sm.stop = n - 1;
    __syncthreads();
    if (wid == 0) {
        // the first row whose drafted token is not accepted
        for (uint32_t b = 0; b + 1 < n; b += kWave) {
            const uint32_t i = min(b + lane, n - 2), row = row0 + i;
            const int32_t d = v.token[row];
            const bool is = d >= 0 && static_cast<uint32_t>(d) < vocab;
            const uint32_t at = is ? d : 0;
            const Share ps(v.cuts[row], sm.scale);
            const double p = ps(v.target_logits[row * v.target.stride + at], at, weight);
            double q = 1.0;
            if (v.by_logits) {
                const Share qs(v.cuts[v.n_rows + row], sm.scale);
                q = qs(v.draft_logits[row * v.draft.stride + at], at, weight);
            }
            const double u = __builtin_fminf(__builtin_fmaxf(v.u[row], 0.0f), 0x1.fffffep-1f);
            const uint64_t no = __ballot(!(is && u * q < p));
            if (no) {
                if (lane == 0) sm.stop = min(b + static_cast<uint32_t>(__builtin_ctzll(no)), n - 1);
                break;
            }
        }
    }
    __syncthreads();
    const uint32_t stop = sm.stop, row = row0 + stop;
    const Cut cut = v.cuts[row];
    const int32_t d = stop + 1 < n ? v.token[row] : -1;
    const bool drafted = d >= 0 && static_cast<uint32_t>(d) < vocab;
    const bool by_logits = v.by_logits && drafted;
    const Rows r = {v.target_logits + row * v.target.stride, by_logits ? v.draft_logits + row * v.draft.stride : nullptr,
                    Share(cut, sm.scale), Share(by_logits ? v.cuts[v.n_rows + row] : cut, sm.scale),
                    drafted && !by_logits ? static_cast<uint32_t>(d) : kNone};
    double rest[kDrawPer], all[kDrawPer];
    const auto sums_of = [&](uint32_t part, double& own, double& own_all) {
        weigh(v, r, weight, part * kSlice + tid * kDrawPer, rest, all);
        own = own_all = 0.0;
#pragma unroll
        for (uint32_t j = 0; j < kDrawPer; j++) {
            own += rest[j];
            own_all += all[j];
        }
    };
    double own, own_all;
    sums_of(slice, own, own_all);
    const double a = wave_sum(own), b = wave_sum(own_all);
    if (lane == 0) {
        sm.part[0][wid] = a;
        sm.part[1][wid] = b;
    }
    __syncthreads();
    Sum* const sums = v.sums + static_cast<size_t>(s) * slices;
    if (tid == 0) {
        Sum t = {0.0, 0.0};
        for (uint32_t w = 0; w < kDrawThreads / kWave; w++) {
            t.rest += sm.part[0][w];
            t.all += sm.part[1][w];
        }
        put(&sums[slice].rest, t.rest);
        put(&sums[slice].all, t.all);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // they are in memory
        sm.last = __hip_atomic_fetch_add(v.counts + s, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == slices - 1;
    }
    __syncthreads();
    if (!sm.last) return;
    // the part in which the goal is reached; where a rounding leaves none, the last with any weight
    if (wid == 0) {
        static_assert(kSlices <= 2 * kWave, "two parts a lane");
        double w[2], x[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t at = 2 * lane + i;
            w[i] = at < slices ? get(&sums[at].rest) : 0.0;
            x[i] = at < slices ? get(&sums[at].all) : 0.0;
        }
        const bool any = __any(w[0] + w[1] > 0.0);
        if (!any) {  // p is q: what is drawn from is p
            w[0] = x[0];
            w[1] = x[1];
        }
        double run = w[0] + w[1];
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double y = __shfl_up(run, o);
            if (static_cast<int>(lane) >= o) run += y;
        }
        const double total = __shfl(run, 63);
        const double u = __builtin_fminf(__builtin_fmaxf(v.u_draw[s], 0.0f), 0x1.fffffep-1f);
        const double goal = u * total, before = run - (w[0] + w[1]);
        // (ends of the two parts; a lane without weight is none)
        const double mid = before + w[0];
        const uint64_t in0 = __ballot(w[0] > 0.0 && mid > goal), in1 = __ballot(w[1] > 0.0 && run > goal);
        const uint64_t has0 = __ballot(w[0] > 0.0), has1 = __ballot(w[1] > 0.0);
        const uint32_t f0 = in0 ? 2 * __builtin_ctzll(in0) : kNone, f1 = in1 ? 2 * __builtin_ctzll(in1) + 1 : kNone;
        uint32_t at = min(f0, f1);
        if (at == kNone) {
            const uint32_t l0 = has0 ? 2 * (63 - __builtin_clzll(has0)) : kNone, l1 = has1 ? 2 * (63 - __builtin_clzll(has1)) + 1 : kNone;
            at = l0 == kNone ? l1 : l1 == kNone ? l0 : max(l0, l1);
        }
        if (lane == (at == kNone ? 0 : at / 2)) {
            sm.at = at;
            sm.goal = goal - (at % 2 ? mid : before);
            sm.last = any ? 1 : 2;
        }
    }
    __syncthreads();
    const uint32_t part = sm.at;
    int32_t token = -1;
    if (part != kNone) {
        sums_of(part, own, own_all);
        if (sm.last == 2) {
            own = own_all;
#pragma unroll
            for (uint32_t j = 0; j < kDrawPer; j++) rest[j] = all[j];
        }
        double run = own;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double y = __shfl_up(run, o);
            if (static_cast<int>(lane) >= o) run += y;
        }
        const double wave = __shfl(run, 63);
        __syncthreads();  // the sums of before are read
        if (lane == 0) {
            sm.part[0][wid] = wave;
            sm.part[1][wid] = 0.0;
        }
        __syncthreads();
        double before = 0.0;
        for (uint32_t w = 0; w < wid; w++) before += sm.part[0][w];
        const double end = before + run;
        // this thread's first token past the goal, and its last with weight
        double at = end - own;
        uint32_t first = kNone, back = 0;
#pragma unroll
        for (uint32_t j = 0; j < kDrawPer; j++) {
            at += rest[j];
            const uint32_t i = part * kSlice + tid * kDrawPer + j;
            if (rest[j] > 0.0) {
                back = i + 1;
                if (first == kNone && at > sm.goal) first = i;
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            first = min(first, static_cast<uint32_t>(__shfl_xor(first, o)));
            back = max(back, static_cast<uint32_t>(__shfl_xor(back, o)));
        }
        __syncthreads();
        uint32_t* const firsts = reinterpret_cast<uint32_t*>(sm.part[0]);
        uint32_t* const backs = reinterpret_cast<uint32_t*>(sm.part[1]);
        if (lane == 0) {
            firsts[wid] = first;
            backs[wid] = back;
        }
        __syncthreads();
        for (uint32_t w = 0; w < kDrawThreads / kWave; w++) {
            first = min(first, firsts[w]);
            back = max(back, backs[w]);
        }
        token = first != kNone ? static_cast<int32_t>(first) : static_cast<int32_t>(back) - 1;
    }
    for (uint32_t i = tid; i < n; i += kDrawThreads) {
        const int32_t own_token = v.token[row0 + i];
        v.out[row0 + i] = i < stop ? own_token : i == stop ? token : -1;
    }
    if (tid == 0) v.accepted[s] = static_cast<int32_t>(stop);
}

}  // namespace

extern "C" __global__ void __launch_bounds__(256, 8) zlm_verify_hist(VArgs v) { hist<256>(v); }
extern "C" __global__ void __launch_bounds__(1024) zlm_verify_hist_wide(VArgs v) { hist<1024>(v); }
extern "C" __global__ void __launch_bounds__(512) zlm_verify_cuts(VArgs v) { cuts(v); }
extern "C" __global__ void __launch_bounds__(512) zlm_verify_draw(VArgs v) { draw(v); }
