// The sampler's kernels on the CPU, a workgroup at a time (tests/host_gpu).
#include "zlm_sample.hip"

#undef asm

namespace {
constexpr uint64_t kMost = 5000;  // barriers of a wave: a draw passes some hundreds
}

namespace {
// The arguments of rows of packed logits, with scratch of their own.
struct Call {
    zlm::SampleArgs a = {};
    std::vector<uint64_t> hist, shorts;
    std::vector<zlm::SampleSlice> info;

    Call(const float* logits, uint32_t rows, uint32_t vocab) {
        a.logits = logits;
        a.stride = a.vocab = vocab;
        a.rows = rows;
        a.slices = (vocab + zlm::kSampleSlice - 1) / zlm::kSampleSlice;
        const size_t all = static_cast<size_t>(rows) * a.slices;
        hist.assign(all * zlm::kSampleBins, ~0ull);
        shorts.assign(all * zlm::kSampleShort, ~0ull);
        info.resize(all);
        a.hist = hist.data();
        a.shorts = shorts.data();
        a.info = info.data();
    }
    int count(uint32_t row) {
        for (uint32_t s = 0; s < a.slices; s++)
            if (const int e = host_gpu::run(256, {s, row, 0}, kMost, [&] { zlm_sample_hist(a); })) return e;
        return 0;
    }
};
}  // namespace

// Draws from rows of logits, packed; the search reads those of `later`.  0: done; what
// host_gpu::run gives up for otherwise.
extern "C" int host_sample(const float* logits, const float* later, uint32_t rows, uint32_t vocab, const float* t,
                           const int32_t* k, const float* p, const float* mp, const float* u, int32_t* token,
                           float* prob) {
    Call c(logits, rows, vocab);
    c.a.temperature = t;
    c.a.top_k = k;
    c.a.top_p = p;
    c.a.min_p = mp;
    c.a.u = u;
    c.a.token = token;
    c.a.prob = prob;
    for (uint32_t r = 0; r < rows; r++) {
        if (const int e = c.count(r)) return e;
        zlm::SampleArgs b = c.a;
        b.logits = later;
        if (const int e = host_gpu::run(512, {r, 0, 0}, kMost, [&] { zlm_sample_pick(b); })) return e;
    }
    return 0;
}

// The search of a row at temperature 1 for a goal that lies where bin `bin`, the only one in
// question, ends (past: more weight than that is asked for) or begins (as much).
extern "C" int host_find(const float* logits, uint32_t vocab, uint32_t bin, int past, int32_t* token, double* weight) {
    Call c(logits, 1, vocab);
    if (const int e = c.count(0)) return e;
    return host_gpu::run(512, {0, 0, 0}, kMost, [&] {
        __shared__ Shared sm;
        const double rate = rate_of(c.a, 0);
        Row::Ahead ahead;
        Row::read_ahead(c.a, 0, 0, ahead);
        const uint64_t best = row_info(c.a, sm, 0);
        Row r(c.a, sm, 0, rate, best);
        r.join(ahead);
        r.flag(bin, bin);
        const bool listed = r.in_question() <= kList;
        if (listed && !r.list_shorts(ahead)) r.list_row();
        const Goal g = past ? Goal{kMore, r.weight_to(bin + 1), 0, bin, bin} : Goal{kAtLeast, r.weight_to(bin), 0, bin, bin};
        const Found f = r.find(g, listed);
        if (threadIdx.x == 0) {
            *token = static_cast<int32_t>(~static_cast<uint32_t>(f.token));
            *weight = f.weight - r.weight_to(bin);
        }
    });
}

// The search for weight up to the end of bin `bin`, its bins in question formed from that weight
// and one a rounding above it, in the wrong order.
extern "C" int host_find_between(const float* logits, uint32_t vocab, uint32_t bin, int32_t* token) {
    Call c(logits, 1, vocab);
    if (const int e = c.count(0)) return e;
    return host_gpu::run(512, {0, 0, 0}, kMost, [&] {
        __shared__ Shared sm;
        const double rate = rate_of(c.a, 0);
        Row::Ahead ahead;
        Row::read_ahead(c.a, 0, 0, ahead);
        Row r(c.a, sm, 0, rate, row_info(c.a, sm, 0));
        r.join(ahead);
        const double end = r.weight_to(bin + 1);
        uint32_t b[2];
        r.bins_for(kAtLeast, nextafter(end, INFINITY), end, b);
        const bool listed = r.in_question() <= kList;
        if (listed && !r.list_shorts(ahead)) r.list_row();
        const Found f = r.find({kAtLeast, end, 0, b[0], b[1]}, listed);
        if (threadIdx.x == 0) *token = static_cast<int32_t>(~static_cast<uint32_t>(f.token));
    });
}
