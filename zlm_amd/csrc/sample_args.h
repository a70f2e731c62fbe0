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

// What a draw takes a row's tokens by: those whose (key, ~index) is at least `token`, by
// their weights' shares of `weight`; rate 0: `best` alone (0: none at all).
struct SampleCut {
    uint64_t token, best;
    double weight, rate;
    double drafted;  // the share of the token drafted after the row (0 for one that is none)
};

constexpr uint32_t kVerifyPart = 4096;  // tokens of a workgroup of the draw

// A part of what a row that ends a sequence's drafts is drawn from: the weight of the
// target's tokens, and what of it lies above the draft's.
struct VerifySum {
    double rest, all;
};

constexpr uint32_t kVerifyRows = 65536;  // of a call

struct VerifyArgs {
    SampleArgs target, draft;  // the rows at hand
    uint32_t first;            // the first of them
    uint32_t n_rows, n_seqs;   // of the call
    uint32_t by_logits;        // the draft has logits; else a drafted token is certain
    const int32_t* q_start;    // n_seqs + 1: the rows of sequence s are [q_start[s], q_start[s + 1])
    const int32_t* token;      // drafted after each row
    const float* u;            // of each row, for its acceptance
    const float* u_draw;       // of each sequence
    int32_t* accepted;
    int32_t* out;
    const float* target_logits;  // of all rows
    const float* draft_logits;
    SampleCut* cuts;    // n_rows of the target, then as many of the draft
    uint32_t parts;     // of a row
    VerifySum* sums;    // n_seqs x parts
    uint32_t* counts;   // of each sequence: parts that are summed up
};

}  // namespace zlm
