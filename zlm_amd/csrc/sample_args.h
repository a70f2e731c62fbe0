// sample_args.h -- the argument block of the sampling kernels (zlm_sample.hip),
// shared with the host library that fills it.
#pragma once
#include <stdint.h>

namespace zlm {

constexpr uint32_t kSampleSlice = 8192;  // logits of one histogram
constexpr uint32_t kSampleBins = 512;
constexpr uint32_t kSampleSlices = 128;  // slices of a row: vocabularies up to 2^20
constexpr uint32_t kSampleShort = 256;   // tokens of a slice's short list

// A slice of a row: its largest logit as (key, ~index) (0: no logit that may be
// drawn) and its short list, all tokens of its first `bins` bins.
struct SampleSlice {
    uint64_t best;
    uint32_t bins, n;
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
    float* prob;        // or null
    uint64_t* hist;     // rows x slices x kSampleBins
    uint64_t* shorts;   // rows x slices x kSampleShort
    SampleSlice* info;  // rows x slices
};

}  // namespace zlm
