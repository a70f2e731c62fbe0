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
//   draw  a workgroup for each 4096 tokens of a sequence: it decides which row ends the
//         drafts (a few loads), and sums up its part of what is drawn from; the last of a
//         sequence's to be done adds up the parts and looks the token up in its part
#define ZLM_SAMPLE_FEW
#include "sample_impl.h"

namespace {

using VArgs = zlm::VerifyArgs;
using Cut = zlm::SampleCut;
using Sum = zlm::VerifySum;
constexpr uint32_t kPart = zlm::kVerifyPart, kDrawThreads = 512, kVecs = kPart / (4 * kDrawThreads);

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

// A value that all lanes have, in scalar registers.
template <class T>
__device__ __forceinline__ T uniform(T v) {
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
    } else {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<int>(u)), hi = __builtin_amdgcn_readfirstlane(static_cast<int>(u >> 32));
        return __builtin_bit_cast(T, static_cast<uint64_t>(hi) << 32 | lo);
    }
}

// A row's tokens by their shares.
struct Share {
    double top, rate, inv;
    float least;    // the smallest logit that is kept, as far as `last`, the last token of that logit
    uint32_t last;
    __device__ __forceinline__ explicit Share(const Cut& c) {
        // (a cut of 0 keeps all that is no -inf, a row without any has a `best` of 0)
        const uint64_t from = c.rate == 0.0 ? c.best : c.token;
        const float x = c.best == 0 ? INFINITY : from == 0 ? -INFINITY : value_of(static_cast<uint32_t>(from >> 32));
        rate = uniform(c.rate);
        top = uniform(__builtin_floor(static_cast<double>(value_of(static_cast<uint32_t>(c.best >> 32))) * c.rate));
        inv = uniform(c.weight > 0.0 ? 1.0 / c.weight : 0.0);
        least = uniform(x);
        last = uniform(~static_cast<uint32_t>(from));
    }
    // Bin by bin down from the largest; 0 for those past kBins, which have no weight.
    __device__ __forceinline__ double of(float x, uint32_t i, const Weight& weight, const double* scale, bool table) const {
        x = x > 3.402823466e38f ? 3.402823466e38f : x;  // (a NaN stays one, and is not kept)
        if (!(x > least || (x == least && i <= last))) return 0.0;
        if (rate == 0.0) return 1.0;
        const double y = static_cast<double>(x) * rate, b = __builtin_floor(y), d = top - b;
        if (!(d < 1.0 * kBins)) return 0.0;
        const double w = weight.units(y - b);
        const uint32_t bin = static_cast<uint32_t>(__builtin_fmax(d, 0.0));
        return w * (table ? scale[bin] : exp(static_cast<double>(bin) * -0.0625) / kUnit) * inv;
    }
};

__device__ __forceinline__ void cuts(const VArgs& v) {
    if (v.first == 0 && blockIdx.x == 0)  // for the launch after this
        for (uint32_t s = threadIdx.x; s < v.n_seqs; s += kThreads) v.counts[s] = 0;
    bool draft;
    uint32_t row;
    if (!row_of(v, blockIdx.x, draft, row)) return;
    const Args& a = draft ? v.draft : v.target;
    // the drafted token's logit, on its way early
    const int32_t d = v.token[v.first + row];
    const bool is = d >= 0 && static_cast<uint32_t>(d) < a.vocab;
    const float x = a.logits[row * a.stride + (is ? d : 0)];
    Cut* const to = v.cuts + (draft ? v.n_rows : 0) + v.first + row;
    Cut cut;
    if (!pick<false>(a, row, cut)) return;
    const Weight weight;
    cut.drafted = is ? Share(cut).of(x, d, weight, nullptr, false) : 0.0;
    *to = cut;
}

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
    double part[2][kVecs][kDrawThreads / kWave];
    uint32_t firsts[kDrawThreads / kWave], backs[kDrawThreads / kWave];
    uint32_t stop, last, at;
    double goal;
    Cut target, draft;  // of the row that ends the drafts
};

// What a row's draw goes by.
struct Rows {
    const float *p, *q;  // q null: none, or a certain token
    Share ps, qs;
    uint32_t certain;    // that token, or none
};

// f(vector, element, what lies above the draft's share, the target's share) for a thread's
// tokens: four in a row of each 2048 of the part.
template <class F>
__device__ __forceinline__ void weigh(const Rows& r, uint32_t vocab, const Weight& weight, const double* scale, uint32_t part, const F& f) {
    typedef float v4 __attribute__((ext_vector_type(4), aligned(4)));
    float x[kVecs][4], y[kVecs][4];
    const uint32_t i0 = part * kPart + 4 * threadIdx.x;
    if ((part + 1) * kPart <= vocab) {
#pragma unroll
        for (uint32_t j = 0; j < kVecs; j++) {
            const uint32_t i = i0 + 4 * kDrawThreads * j;
            const v4 a = *reinterpret_cast<const v4*>(r.p + i), b = *reinterpret_cast<const v4*>((r.q ? r.q : r.p) + i);
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                x[j][e] = a[e];
                y[j][e] = b[e];
            }
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < kVecs; j++)
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                const uint32_t i = i0 + 4 * kDrawThreads * j + e;
                x[j][e] = i < vocab ? r.p[i] : -INFINITY;
                y[j][e] = r.q && i < vocab ? r.q[i] : -INFINITY;
            }
    }
#pragma unroll
    for (uint32_t j = 0; j < kVecs; j++)
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) {
            const uint32_t i = i0 + 4 * kDrawThreads * j + e;
            const double p = r.ps.of(x[j][e], i, weight, scale, true);
            const double q = r.q ? r.qs.of(y[j][e], i, weight, scale, true) : i == r.certain ? 1.0 : 0.0;
            f(j, e, p > q ? p - q : 0.0, p);
        }
}

__device__ __forceinline__ double wave_run(double v) {  // inclusive sums
    const uint32_t lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (uint32_t o = 1; o < kWave; o <<= 1) {
        const double y = __shfl_up(v, o);
        if (lane >= o) v += y;
    }
    return v;
}

__device__ __forceinline__ double number(float u) {  // in [0, 1)
    return __builtin_fminf(__builtin_fmaxf(u, 0.0f), 0x1.fffffep-1f);
}

__device__ __forceinline__ void draw(const VArgs& v) {
    __shared__ DrawShared sm;
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
    const uint32_t mine = blockIdx.x, s = blockIdx.y, parts = v.parts, vocab = v.target.vocab;
    const int32_t from = v.q_start[s], to = min(v.q_start[s + 1], static_cast<int32_t>(v.n_rows));
    if (from < 0 || from >= to) {  // no rows
        if (mine == 0 && tid == 0) v.accepted[s] = 0;
        return;
    }
    const uint32_t row0 = from, n = static_cast<uint32_t>(to - from);
    const double u_draw = number(v.u_draw[s]);
    const Weight weight;
    sm.scale[tid] = exp(static_cast<double>(tid) * -0.0625) / kUnit;
    static_assert(kDrawThreads == kBins, "a bin a thread");
    if (wid == 0) {
        // the first row whose drafted token is not accepted, or the last
        for (uint32_t b = 0;; b += kWave) {
            const uint32_t i = min(b + lane, n - 1), row = row0 + i;
            const Cut p = v.cuts[row];
            const bool has_q = v.by_logits && i + 1 < n;
            const Cut q = v.cuts[has_q ? v.n_rows + row : row];
            const int32_t d = v.token[row];
            const bool is = d >= 0 && static_cast<uint32_t>(d) < vocab;
            const uint64_t no = __ballot(i + 1 == n || !(is && number(v.u[row]) * (has_q ? q.drafted : 1.0) < p.drafted));
            if (no) {
                if (lane == static_cast<uint32_t>(__builtin_ctzll(no))) {
                    sm.stop = i;
                    sm.target = p;
                    sm.draft = q;
                }
                break;
            }
        }
    }
    __syncthreads();
    const uint32_t stop = sm.stop, row = row0 + stop;
    const int32_t d = stop + 1 < n ? v.token[row] : -1;
    const bool drafted = d >= 0 && static_cast<uint32_t>(d) < vocab;
    const bool by_logits = v.by_logits && drafted;
    const Rows r = {v.target_logits + row * v.target.stride, by_logits ? v.draft_logits + row * v.draft.stride : nullptr,
                    Share(sm.target), Share(by_logits ? sm.draft : sm.target),
                    drafted && !by_logits ? static_cast<uint32_t>(d) : kNone};
    double own = 0.0, own_all = 0.0;
    weigh(r, vocab, weight, sm.scale, mine, [&](uint32_t, uint32_t, double rest, double all) {
        own += rest;
        own_all += all;
    });
    const double a = wave_sum(own), b = wave_sum(own_all);
    if (lane == 0) {
        sm.part[0][0][wid] = a;
        sm.part[1][0][wid] = b;
    }
    __syncthreads();
    Sum* const sums = v.sums + static_cast<size_t>(s) * parts;
    if (tid == 0) {
        Sum t = {0.0, 0.0};
        for (uint32_t w = 0; w < kDrawThreads / kWave; w++) {
            t.rest += sm.part[0][0][w];
            t.all += sm.part[1][0][w];
        }
        put(&sums[mine].rest, t.rest);
        put(&sums[mine].all, t.all);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // they are in memory
        sm.last = __hip_atomic_fetch_add(v.counts + s, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
    }
    __syncthreads();
    if (!sm.last) return;
    // the part in which the goal is reached; where a rounding leaves none, the last with any weight
    if (wid == 0) {
        constexpr uint32_t kEach = kSlice * kSlices / kPart / kWave;  // parts a lane
        double w[kEach], x[kEach];
#pragma unroll
        for (uint32_t i = 0; i < kEach; i++) {
            const uint32_t at = min(kEach * lane + i, parts - 1);
            const bool has = kEach * lane + i < parts;
            const double rest = get(&sums[at].rest), all = get(&sums[at].all);
            w[i] = has ? rest : 0.0;
            x[i] = has ? all : 0.0;
        }
        double sum = 0.0;
#pragma unroll
        for (uint32_t i = 0; i < kEach; i++) sum += w[i];
        const bool any = __any(sum > 0.0);
        if (!any) {  // p is q: what is drawn from is p
            sum = 0.0;
#pragma unroll
            for (uint32_t i = 0; i < kEach; i++) sum += w[i] = x[i];
        }
        const double run = wave_run(sum), goal = u_draw * __shfl(run, 63);
        double at = run - sum, before = 0.0, last_before = 0.0;
        uint32_t first = kNone, back = kNone;
#pragma unroll
        for (uint32_t i = 0; i < kEach; i++) {
            const double end = at + w[i];
            if (w[i] > 0.0) {
                back = kEach * lane + i;
                last_before = at;
                if (first == kNone && end > goal) {
                    first = back;
                    before = at;
                }
            }
            at = end;
        }
        const uint64_t in = __ballot(first != kNone), has = __ballot(back != kNone);
        const uint32_t who = in ? __builtin_ctzll(in) : has ? 63 - __builtin_clzll(has) : 0;
        if (lane == who) {
            sm.at = in ? first : back;
            sm.goal = goal - (in ? before : last_before);
            sm.last = any ? 1 : 2;
        }
    }
    __syncthreads();
    const uint32_t part = sm.at;
    int32_t token = -1;
    if (part != kNone) {
        const bool whole = sm.last == 2;
        double sum[kVecs] = {}, run[kVecs], x[kVecs][4];
        weigh(r, vocab, weight, sm.scale, part, [&](uint32_t j, uint32_t e, double rest, double all) {
            x[j][e] = whole ? all : rest;
            sum[j] += x[j][e];
        });
#pragma unroll
        for (uint32_t j = 0; j < kVecs; j++) {
            run[j] = wave_run(sum[j]);
            if (lane == kWave - 1) sm.part[0][j][wid] = run[j];
        }
        __syncthreads();
        // before each of this thread's vectors
        double at[kVecs], before = 0.0;
#pragma unroll
        for (uint32_t j = 0; j < kVecs; j++) {
            at[j] = before + run[j] - sum[j];
            for (uint32_t w = 0; w < kDrawThreads / kWave; w++) {
                at[j] += w < wid ? sm.part[0][j][w] : 0.0;
                before += sm.part[0][j][w];
            }
        }
        // its first token past the goal, and its last with weight
        uint32_t first = kNone, back = 0;
#pragma unroll
        for (uint32_t j = 0; j < kVecs; j++)
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                const uint32_t i = part * kPart + 4 * kDrawThreads * j + 4 * tid + e;
                at[j] += x[j][e];
                back = x[j][e] > 0.0 ? i + 1 : back;
                first = x[j][e] > 0.0 && at[j] > sm.goal ? min(first, i) : first;
            }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            first = min(first, static_cast<uint32_t>(__shfl_xor(first, o)));
            back = max(back, static_cast<uint32_t>(__shfl_xor(back, o)));
        }
        if (lane == 0) {
            sm.firsts[wid] = first;
            sm.backs[wid] = back;
        }
        __syncthreads();
        for (uint32_t w = 0; w < kDrawThreads / kWave; w++) {
            first = min(first, sm.firsts[w]);
            back = max(back, sm.backs[w]);
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
extern "C" __global__ void __launch_bounds__(512, 4) zlm_verify_cuts(VArgs v) { cuts(v); }
extern "C" __global__ void __launch_bounds__(512, 4) zlm_verify_draw(VArgs v) { draw(v); }
