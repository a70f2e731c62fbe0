// sample_args.h -- the argument block of the sampling kernels (zlm_sample.hip),
// shared with the host library that fills it.
#pragma once
#include <stdint.h>

namespace zlm {

constexpr uint32_t kSampleSlice = 8192;  // logits of one histogram
constexpr uint32_t kSampleBins = 512;
constexpr uint32_t kSampleSlices = 128;  // slices of a row: vocabularies up to 2^20

// A slice of a row: the bin (on the row's absolute grid) of its largest logit and
// that logit as (key, ~index); best 0: no logit that may be drawn.
struct SampleSlice {
    double top;
    uint64_t best;
};

struct SampleArgs {
    const float* logits;
    uint64_t stride;  // floats between rows
    uint32_t rows, vocab, slices;
    const float* temperature;  // null: 1
    const int32_t* top_k;      // null: off; so too the next two
    const float* top_p;
    const float* min_p;
    const float* u;
    int32_t* token;
    float* prob;     // or null
    uint64_t* hist;  // rows x slices x kSampleBins
    SampleSlice* info;  // rows x slices
};

}  // namespace zlm
