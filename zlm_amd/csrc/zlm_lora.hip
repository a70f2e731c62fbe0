// zlm_lora.hip -- CDNA4 (gfx950) kernels of low-rank adapters: each token of a batch has
// one of many pairs A (rank x k), B (rows x rank), or none, and
//     y[t] = res[t] + scale * B (A x[t]).
// Built as a device-only code object (hipcc --genco) and loaded by the host library.
//
// Tokens are taken in tiles with one adapter, so that a tile reads its A and B once: of up to 16
// of few tokens, of up to 32 of many.  Up to 256 tokens every workgroup finds its tile by itself;
// more are grouped by a launch before.  Then two launches: h = A x, k split over waves and
// workgroups, and y = res + scale * B h.
//
// Both products run on v_mfma_f32_16x16x32_bf16 with the tokens in the N dimension.  A
// 32-bit number is the sum of three bf16 (8 bits of its 24 each, cut off, so exactly), an
// f16 of two, and a product is the sum of its parts' products: three instructions for a bf16
// adapter, six for f16, eight for f32 (all but that of both last parts, under 2^-30 of it).  So
// the results have the accuracy of 32-bit products at 5, 2.7 and 2 times the rate of the 32-bit
// matrix instruction.  bf16 has the exponents of 32 bits: nothing is scaled, and what is cut off
// lies under 2^-133.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lora_args.h"

namespace {

using Args = zlm::LoraArgs;
using zlm::LoraTile;
constexpr uint32_t kWave = 64;
constexpr uint32_t kN = 16;  // tokens of a matrix tile

typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

// ---- parts ----

// The upper halves of two words.
__device__ __forceinline__ uint32_t uppers(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302); }

// Eight floats as kN bf16 each that add up to them (to what kN times 8 bits hold).
template <int kN>
__device__ __forceinline__ void to_parts(const float (&x)[8], v8b (&part)[kN]) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = x[i];
#pragma unroll
    for (int p = 0; p < kN; p++) {
        uint32_t u[8];
#pragma unroll
        for (int i = 0; i < 8; i++) u[i] = __builtin_bit_cast(uint32_t, r[i]);
        part[p] = __builtin_bit_cast(v8b, v4u{uppers(u[0], u[1]), uppers(u[2], u[3]), uppers(u[4], u[5]), uppers(u[6], u[7])});
        if (p + 1 < kN) {
#pragma unroll
            for (int i = 0; i < 8; i++) r[i] -= __builtin_bit_cast(float, u[i] & 0xffff0000u);
        }
    }
}

// Eight weights as loaded, and as parts.
struct Bf16 {
    static constexpr int kParts = 1, kVecs = 1, kBytes = 2;
    __device__ __forceinline__ static void parts(const v4u (&w)[1], v8b (&p)[1]) { p[0] = __builtin_bit_cast(v8b, w[0]); }
};
struct F16 {
    static constexpr int kParts = 2, kVecs = 1, kBytes = 2;
    __device__ __forceinline__ static void parts(const v4u (&w)[1], v8b (&p)[2]) {
        const v8h h = __builtin_bit_cast(v8h, w[0]);
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = static_cast<float>(h[i]);
        to_parts(x, p);
    }
};
struct F32 {
    static constexpr int kParts = 3, kVecs = 2, kBytes = 4;
    __device__ __forceinline__ static void parts(const v4u (&w)[2], v8b (&p)[3]) {
        const v4f a = __builtin_bit_cast(v4f, w[0]), b = __builtin_bit_cast(v4f, w[1]);
        const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        to_parts(x, p);
    }
};

template <class W>
__device__ __forceinline__ void load(const uint8_t* p, v4u (&w)[W::kVecs]) {
#pragma unroll
    for (int i = 0; i < W::kVecs; i++) w[i] = reinterpret_cast<const v4u*>(p)[i];
}

// The products of the parts, the small ones first.  A bf16's and an f16's are all there; of
// two numbers of three parts the last ones' is left out.  (Each part that is cut off is under
// 2^-7 of the one before and has its sign: without the two products before that one all results
// would be too small, by up to 2^-21.  They cost f32 about 1% of a call: 2048 tokens of 8
// prompts, k and rows 4096, rank 256 195 and 197 us, 1024 tokens of 40 adapters 181 and 183.)
template <int kN>
__device__ __forceinline__ v4f multiply(const v8b (&w)[kN], const v8b (&x)[3], v4f acc) {
#pragma unroll
    for (int s = kN < 3 ? kN + 1 : 3; s >= 0; s--)
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int j = s - i;
            if (j < 0 || j > 2) continue;
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[i], x[j], acc, 0, 0, 0);
        }
    return acc;
}

// ---- tiles ----

// A tile, and this lane's tokens of it (lane % 16 and 16 on; the tile's first where it has
// fewer).
template <int kNt>
struct Mine {
    uint32_t adapter, rank, n, token[kNt];
    __device__ __forceinline__ bool live(int i) const { return kN * i + (threadIdx.x & (kN - 1)) < n; }
};

__device__ __forceinline__ uint32_t adapter_of(const Args& a, uint32_t t) {
    return min(static_cast<uint32_t>(a.adapter[t]), a.n_adapters);  // n_adapters: none
}

__device__ __forceinline__ uint32_t rank_of(const Args& a, uint32_t adapter) {
    if (adapter >= a.n_adapters) return 0;
    return a.ranks ? min(static_cast<uint32_t>(max(a.ranks[adapter], 0)), a.rank) : a.rank;
}

// What a workgroup finds its tile by: a token of each adapter, and all of that token's
// adapter's; the first of all tiles; its own.
template <uint32_t kTokens>
struct Grouping {
    uint8_t one_of[zlm::kLoraAdapters + 2];
    unsigned long long with[kTokens][kTokens / kWave], begins[kTokens / kWave];
    uint32_t adapter, rank, from, n;
    uint8_t member[kN];
};

// False: there are not so many tiles.  Tokens without an adapter make tiles of their own,
// but where y is res.  Places and tiles follow the tokens' order, so that all workgroups of both
// launches find the same.
//
// Up to 64 tokens, a wave: those of each lane's adapter, and its place among them; those at
// 0, 16, 32 and 48 begin tiles.
__device__ __forceinline__ bool few_tile(const Args& a, uint32_t tile, Mine<1>& m, Grouping<kWave>& sm) {
    const uint32_t lane = threadIdx.x & (kWave - 1), j = lane & (kN - 1);
    const bool has = lane < a.n_tokens;
    const uint32_t own = has ? adapter_of(a, lane) : a.n_adapters + 1;
    const uint32_t rank = rank_of(a, own);
    if (threadIdx.x < kWave) {
        sm.with[lane][0] = 0;
        sm.one_of[own] = static_cast<uint8_t>(lane);
    }
    __syncthreads();
    const uint32_t one = sm.one_of[own];
    if (threadIdx.x < kWave) atomicOr(&sm.with[one][0], 1ull << lane);
    __syncthreads();
    const uint64_t mine = sm.with[one][0], below = (1ull << lane) - 1;
    const uint32_t place = __builtin_popcountll(mine & below);
    const bool left = has && !(a.in_place && own == a.n_adapters);
    uint64_t begins = __ballot(left && place % kN == 0);
    if (tile >= static_cast<uint32_t>(__builtin_popcountll(begins))) return false;
    for (uint32_t i = 0; i < tile; i++) begins &= begins - 1;
    const uint32_t first = __builtin_ctzll(begins);
    m.adapter = __builtin_amdgcn_readlane(own, first);
    m.rank = __builtin_amdgcn_readlane(rank, first);
    const uint32_t from = __builtin_amdgcn_readlane(place, first);
    uint64_t with = __ballot(own == m.adapter && place >= from && place < from + kN);
    m.n = __builtin_popcountll(with);
    m.token[0] = first;
    for (uint32_t i = 0; i < m.n; i++) {
        if (j == i) m.token[0] = __builtin_ctzll(with);
        with &= with - 1;
    }
    return true;
}

// More, the first four waves: the same with a token a thread, the tile's members written
// down by themselves.  k and rows 4096, bf16, by this and grouped by a launch in tiles of 32:
// 65 tokens of 40 adapters of rank 16 12 and 18 us, of rank 256 63 and 65; 256 tokens of one
// of rank 64 16 and 31, of 40 of rank 128 27 and 39, of 200 of rank 256 208 and 207.
__device__ __forceinline__ bool small_tile(const Args& a, uint32_t tile, Mine<1>& m, Grouping<zlm::kLoraOwn>& sm) {
    constexpr uint32_t kTokens = zlm::kLoraOwn, kWords = kTokens / kWave;
    static_assert(kTokens <= 256, "a token in a byte, and a thread");
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
    const bool in = tid < kTokens, has = tid < a.n_tokens;
    const uint32_t own = has ? adapter_of(a, tid) : a.n_adapters + 1;
    const uint32_t rank = rank_of(a, own);
    if (in) {
#pragma unroll
        for (uint32_t i = 0; i < kWords; i++) sm.with[tid][i] = 0;
        sm.one_of[own] = static_cast<uint8_t>(tid);
    }
    if (tid == 0) sm.n = 0;
    __syncthreads();
    const uint32_t one = sm.one_of[own];
    if (in) atomicOr(&sm.with[one][wid], 1ull << lane);
    __syncthreads();
    const uint64_t below = (1ull << lane) - 1;
    uint32_t place = 0, all = 0;
#pragma unroll
    for (uint32_t i = 0; i < kWords; i++) {
        const uint64_t with = sm.with[one][i];
        place += __builtin_popcountll(i < wid ? with : i == wid ? with & below : 0);
        all += __builtin_popcountll(with);
    }
    const bool begins = has && place % kN == 0 && !(a.in_place && own == a.n_adapters);
    const uint64_t mine = __ballot(begins);
    if (in && lane == 0) sm.begins[wid] = mine;
    __syncthreads();
    uint32_t index = __builtin_popcountll(mine & below);
#pragma unroll
    for (uint32_t i = 0; i < kWords; i++) index += i < wid ? __builtin_popcountll(sm.begins[i]) : 0;
    if (begins && index == tile) {
        sm.adapter = own;
        sm.rank = rank;
        sm.from = place;
        sm.n = min(all - place, kN);
    }
    __syncthreads();
    m.n = __builtin_amdgcn_readfirstlane(sm.n);
    if (m.n == 0) return false;  // the workgroup as one
    m.adapter = __builtin_amdgcn_readfirstlane(sm.adapter);
    m.rank = __builtin_amdgcn_readfirstlane(sm.rank);
    const uint32_t at = place - sm.from;
    if (has && own == m.adapter && place >= sm.from && at < m.n) sm.member[at] = static_cast<uint8_t>(tid);
    __syncthreads();
    m.token[0] = sm.member[m.live(0) ? lane & (kN - 1) : 0];
    return true;
}

// As the launch before has grouped them.
template <int kNt>
__device__ __forceinline__ bool grouped_tile(const Args& a, uint32_t tile, Mine<kNt>& m) {
    if (tile >= *a.n_tiles) return false;
    const LoraTile t = a.tile[tile];
    m.adapter = t.adapter;
    m.rank = rank_of(a, t.adapter);
    m.n = t.n;
#pragma unroll
    for (int i = 0; i < kNt; i++) m.token[i] = a.order[t.first + (m.live(i) ? kN * i + (threadIdx.x & (kN - 1)) : 0)];
    return true;
}

__device__ __forceinline__ bool tile_of(const Args& a, uint32_t tile, Mine<1>& m) {
    __shared__ union {
        Grouping<kWave> few;
        Grouping<zlm::kLoraOwn> small;
    } sm;
    if (a.n_tokens <= kWave) return few_tile(a, tile, m, sm.few);
    if (a.n_tokens <= zlm::kLoraOwn) return small_tile(a, tile, m, sm.small);
    return grouped_tile(a, tile, m);
}

__device__ __forceinline__ bool tile_of(const Args& a, uint32_t tile, Mine<2>& m) { return grouped_tile(a, tile, m); }

// The tokens by adapter: counted, their places summed up, then put there (in any order: a
// token's result does not depend on its place).  One workgroup; the first 8192 tokens'
// adapters stay in registers between the two passes.
__device__ __forceinline__ void group(const Args& a) {
    constexpr uint32_t kThreads = 1024, kMost = zlm::kLoraAdapters + 1, kPer = (kMost + kThreads - 1) / kThreads;
    constexpr uint32_t kHold = 8;
    const uint32_t tile = a.per_tile;
    __shared__ uint32_t count[kPer * kThreads], tiles_to[kPer * kThreads];
    __shared__ uint32_t sums[2][kThreads / kWave];
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
    const uint32_t groups = a.n_adapters + (a.in_place ? 0 : 1);
    uint32_t held[kHold];
#pragma unroll
    for (uint32_t i = 0; i < kHold; i++) held[i] = kThreads * i < a.n_tokens ? adapter_of(a, min(kThreads * i + tid, a.n_tokens - 1)) : 0;
    // f(token, its adapter), by all lanes that have a token
    const auto each = [&](const auto& f) {
#pragma unroll
        for (uint32_t i = 0; i < kHold; i++)
            if (kThreads * i + tid < a.n_tokens) f(kThreads * i + tid, held[i]);
        for (uint32_t t = kThreads * kHold + tid; t < a.n_tokens; t += kThreads) f(t, adapter_of(a, t));
    };
    // a place after `count`'s: one atomic for the tokens of a wave that are its first's
    const auto add = [&](uint32_t id) {
        const uint32_t head = __builtin_amdgcn_readfirstlane(id);
        const uint64_t same = __ballot(id == head);
        const uint32_t first = __builtin_ctzll(same);
        uint32_t at = 0;
        if (id != head) at = atomicAdd(&count[id], 1u);
        else if (lane == first) at = atomicAdd(&count[id], static_cast<uint32_t>(__builtin_popcountll(same)));
        const uint32_t base = __builtin_amdgcn_readlane(at, first);
        return id == head ? base + static_cast<uint32_t>(__builtin_popcountll(same & ((1ull << lane) - 1))) : at;
    };
    for (uint32_t i = tid; i <= a.n_adapters + 1; i += kThreads) count[i] = 0;
    __syncthreads();
    each([&](uint32_t, uint32_t id) { add(id); });
    __syncthreads();
    // exclusive sums of tokens and tiles, kPer groups a thread
    const uint32_t per = (groups + kThreads) / kThreads;
    uint32_t n = 0, k = 0, own[kPer];
#pragma unroll
    for (uint32_t i = 0; i < kPer; i++) {
        const uint32_t g = tid * per + i;
        own[i] = i < per && g < groups ? count[g] : 0;
        n += own[i];
        k += (own[i] + tile - 1) / tile;
    }
    uint32_t to_n = n, to_k = k;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_up(to_n, o), y = __shfl_up(to_k, o);
        if (static_cast<int>(lane) >= o) {
            to_n += x;
            to_k += y;
        }
    }
    if (lane == kWave - 1) {
        sums[0][wid] = to_n;
        sums[1][wid] = to_k;
    }
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (uint32_t i = 0; i < kThreads / kWave; i++) {
        to_n += i < wid ? sums[0][i] : 0;
        to_k += i < wid ? sums[1][i] : 0;
        all += sums[1][i];
    }
    to_n -= n;
    to_k -= k;
#pragma unroll
    for (uint32_t i = 0; i < kPer; i++) {
        const uint32_t g = tid * per + i;
        if (i < per && g <= groups) {
            count[g] = to_n;  // from here on the place of the group's next token
            tiles_to[g] = to_k;
        }
        to_n += own[i];
        to_k += (own[i] + tile - 1) / tile;
    }
    __syncthreads();
    for (uint32_t i = tid; i < all; i += kThreads) {
        uint32_t lo = 0, hi = groups;  // the last group that begins at or before tile i
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (tiles_to[mid] <= i) lo = mid;
            else hi = mid;
        }
        const uint32_t at = tile * (i - tiles_to[lo]);
        a.tile[i] = {lo, count[lo] + at, min(count[lo + 1] - count[lo] - at, tile)};
    }
    if (tid == 0) *a.n_tiles = all;
    __syncthreads();
    each([&](uint32_t t, uint32_t id) {
        if (id < groups) a.order[add(id)] = t;
    });
}

// ---- h = A x ----
//
// A workgroup: a tile, a split of k, up to 16 kMt rows of A.  Its waves take k in turn
// (runs of 32, the lane's eight of them together) and add up their sums through LDS.  5000
// tokens of k 4096, rank 64: 30 us by tiles of 32 tokens, three splits and four waves (one
// split 52, eight 32; by tiles of 16, which read A twice as often, 41).
template <class W, int kMt, int kNt>
__device__ __forceinline__ void down(const Args& a) {
    constexpr uint32_t kWaves = zlm::kLoraWaves[kNt - 1];
    constexpr int kStep = kMt * kNt < 4 ? kMt * kNt : 4;
    __shared__ v4f sums[kWaves][kStep][kWave];
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(tid / kWave);
    const uint32_t m = lane & 15, q = lane >> 4, tile = blockIdx.x, split = blockIdx.y;
    Mine<kNt> mine;
    if (!tile_of(a, tile, mine) || mine.adapter >= a.n_adapters) return;
    const uint32_t r = mine.rank, r0 = 16 * kMt * blockIdx.z;
    if (r0 >= r) return;
    const uint32_t chunks = a.k / 32, parts = a.splits * kWaves, part = split * kWaves + wid;
    const uint32_t c0 = static_cast<uint64_t>(chunks) * part / parts, c1 = static_cast<uint64_t>(chunks) * (part + 1) / parts;
    const float* x[kNt];
#pragma unroll
    for (int t = 0; t < kNt; t++) x[t] = a.x + mine.token[t] * a.x_stride + 8 * q;
    const uint8_t* w[kMt];
#pragma unroll
    for (int i = 0; i < kMt; i++) {
        const uint32_t row = min(r0 + 16 * i + m, a.rank - 1);
        w[i] = static_cast<const uint8_t*>(a.a) + ((static_cast<uint64_t>(mine.adapter) * a.rank + row) * a.k + 8 * q) * W::kBytes;
    }
    v4f acc[kNt][kMt];
#pragma unroll
    for (int t = 0; t < kNt; t++)
#pragma unroll
        for (int i = 0; i < kMt; i++) acc[t][i] = v4f{0, 0, 0, 0};
    // runs in flight: as many as registers hold for two waves a SIMD
    constexpr uint32_t kU = kMt * W::kVecs <= 4 ? zlm::kLoraRuns[kNt - 1] : kMt * W::kVecs <= 8 ? 2 : 1;
    for (uint32_t c = c0; c < c1; c += kU) {
        v4f xv[kU][kNt][2];
        v4u wv[kU][kMt][W::kVecs];
#pragma unroll
        for (uint32_t u = 0; u < kU; u++) {
            const uint32_t at = 32 * min(c + u, c1 - 1);
#pragma unroll
            for (int t = 0; t < kNt; t++) {
                xv[u][t][0] = xv[u][t][1] = v4f{0, 0, 0, 0};
                if (mine.live(t)) {
                    xv[u][t][0] = *reinterpret_cast<const v4f*>(x[t] + at);
                    xv[u][t][1] = *reinterpret_cast<const v4f*>(x[t] + at + 4);
                }
            }
#pragma unroll
            for (int i = 0; i < kMt; i++)
                if (r0 + 16 * i < r) load<W>(w[i] + static_cast<size_t>(at) * W::kBytes, wv[u][i]);
        }
#pragma unroll
        for (uint32_t u = 0; u < kU; u++) {
            if (c + u >= c1) break;
            v8b xp[kNt][3];
#pragma unroll
            for (int t = 0; t < kNt; t++) {
                const v4f lo = xv[u][t][0], hi = xv[u][t][1];
                const float f[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                to_parts(f, xp[t]);
            }
#pragma unroll
            for (int i = 0; i < kMt; i++) {
                if (r0 + 16 * i >= r) break;
                v8b wp[W::kParts];
                W::parts(wv[u][i], wp);
#pragma unroll
                for (int t = 0; t < kNt; t++) acc[t][i] = multiply(wp, xp[t], acc[t][i]);
            }
        }
    }
    float* to = a.part + (static_cast<uint64_t>(split) * a.tiles + tile) * (kN * kNt) * a.rank;
#pragma unroll
    for (int i0 = 0; i0 < kMt * kNt; i0 += kStep) {
        if (i0) __syncthreads();
#pragma unroll
        for (int i = 0; i < kStep; i++) sums[wid][i][lane] = acc[(i0 + i) / kMt][(i0 + i) % kMt];
        __syncthreads();
        for (uint32_t i = wid; i < kStep; i += kWaves) {
            v4f s = sums[0][i][lane];
#pragma unroll
            for (uint32_t v = 1; v < kWaves; v++) s += sums[v][i][lane];
            const uint32_t row = r0 + 16 * ((i0 + i) % kMt) + 4 * q, j = kN * ((i0 + i) / kMt) + m;
            if (j >= mine.n || row >= a.rank) continue;
            *reinterpret_cast<v4f*>(to + j * a.rank + row) = s;
        }
    }
}

// ---- y = res + scale B h ----

// h of the lane's tokens as parts, runs c0 .. c0 + kKt of 32 of the rank: the splits' sum.
template <int kKt, int kNt>
__device__ __forceinline__ void load_h(const Args& a, const Mine<kNt>& mine, uint32_t tile, uint32_t c0, v8b (&hp)[kNt][kKt][3]) {
    const uint32_t m = threadIdx.x & 15, q = (threadIdx.x & (kWave - 1)) >> 4, r = mine.rank;
    const uint64_t step = static_cast<uint64_t>(a.tiles) * (kN * kNt) * a.rank;
    constexpr uint32_t kU = kKt * kNt <= 2 ? 4 : kKt * kNt <= 4 ? 2 : 1;  // splits in flight
    v4f sum[kNt][kKt][2];
#pragma unroll
    for (int t = 0; t < kNt; t++)
#pragma unroll
        for (int c = 0; c < kKt; c++) sum[t][c][0] = sum[t][c][1] = v4f{0, 0, 0, 0};
    for (uint32_t s = 0; s < a.splits; s += kU) {
        v4f v[kU][kNt][kKt][2];
#pragma unroll
        for (uint32_t u = 0; u < kU; u++)
#pragma unroll
            for (int t = 0; t < kNt; t++)
#pragma unroll
                for (int c = 0; c < kKt; c++) {
                    const uint32_t k = 32 * (c0 + c) + 8 * q;
                    v[u][t][c][0] = v[u][t][c][1] = v4f{0, 0, 0, 0};
                    if (mine.live(t) && k < r) {
                        const v4f* p = reinterpret_cast<const v4f*>(
                            a.part + min(s + u, a.splits - 1) * step + (static_cast<uint64_t>(tile) * (kN * kNt) + kN * t + m) * a.rank + k);
                        v[u][t][c][0] = p[0];
                        v[u][t][c][1] = p[1];
                    }
                }
#pragma unroll
        for (uint32_t u = 0; u < kU; u++) {
            if (s + u >= a.splits) break;
#pragma unroll
            for (int t = 0; t < kNt; t++)
#pragma unroll
                for (int c = 0; c < kKt; c++) {
                    sum[t][c][0] += v[u][t][c][0];
                    sum[t][c][1] += v[u][t][c][1];
                }
        }
    }
#pragma unroll
    for (int t = 0; t < kNt; t++)
#pragma unroll
        for (int c = 0; c < kKt; c++) {
            const v4f lo = sum[t][c][0], hi = sum[t][c][1];
            float h[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
            for (int i = 0; i < 8; i++) h[i] = 32 * (c0 + c) + 8 * q + i < r ? h[i] : 0.0f;
            to_parts(h, hp[t][c]);
        }
}

// The same by a workgroup of four waves with one tile: each sums a quarter, through LDS.
template <int kKt>
__device__ __forceinline__ void share_h(const Args& a, const Mine<1>& mine, uint32_t tile, v8b (&hp)[1][kKt][3]) {
    constexpr uint32_t kPitch = 32 * kKt + 4, kPer = 8 * kKt, kEach = kN * kPer / 256;  // by four
    __shared__ __attribute__((aligned(16))) float h[kN * kPitch];
    const uint32_t tid = threadIdx.x, m = tid & 15, q = (tid & (kWave - 1)) >> 4, r = mine.rank;
    const uint64_t step = static_cast<uint64_t>(a.tiles) * kN * a.rank;
    v4f sum[kEach];
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) sum[i] = v4f{0, 0, 0, 0};
    constexpr uint32_t kU = kEach <= 2 ? 4 : 2;  // splits in flight
    for (uint32_t s = 0; s < a.splits; s += kU) {
        v4f v[kU][kEach];
#pragma unroll
        for (uint32_t u = 0; u < kU; u++)
#pragma unroll
            for (uint32_t i = 0; i < kEach; i++) {
                const uint32_t at = 256 * i + tid, j = at / kPer, k = 4 * (at % kPer);
                v[u][i] = v4f{0, 0, 0, 0};
                if (s + u < a.splits && j < mine.n && k < r)
                    v[u][i] = *reinterpret_cast<const v4f*>(a.part + (s + u) * step + (static_cast<uint64_t>(tile) * kN + j) * a.rank + k);
            }
#pragma unroll
        for (uint32_t u = 0; u < kU; u++)
#pragma unroll
            for (uint32_t i = 0; i < kEach; i++) sum[i] += v[u][i];
    }
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) {
        const uint32_t at = 256 * i + tid, j = at / kPer, k = 4 * (at % kPer);
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) sum[i][e] = k + e < r ? sum[i][e] : 0.0f;
        *reinterpret_cast<v4f*>(h + j * kPitch + k) = sum[i];
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kKt; c++) {
        const v4f lo = *reinterpret_cast<const v4f*>(h + m * kPitch + 32 * c + 8 * q);
        const v4f hi = *reinterpret_cast<const v4f*>(h + m * kPitch + 32 * c + 8 * q + 4);
        const float f[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        to_parts(f, hp[0][c]);
    }
}

// Sixteen rows of an adapter's B, rows n + m: the lane's eights of runs c0 and on of the rank.
template <class W, int kKt>
__device__ __forceinline__ void load_b(const Args& a, const uint8_t* b, uint32_t n, uint32_t r, uint32_t c0, v4u (&w)[kKt][W::kVecs]) {
    const uint32_t m = threadIdx.x & 15, q = (threadIdx.x & (kWave - 1)) >> 4;
    const uint8_t* p = b + (static_cast<uint64_t>(min(n + m, a.rows - 1)) * a.rank + 32 * c0 + 8 * q) * W::kBytes;
#pragma unroll
    for (int c = 0; c < kKt; c++) {
#pragma unroll
        for (int i = 0; i < W::kVecs; i++) w[c][i] = v4u{0, 0, 0, 0};
        if (32 * (c0 + c) + 8 * q < r) load<W>(p + 32 * c * W::kBytes, w[c]);
    }
}

// Their products with h, added.
template <class W, int kKt, int kNt>
__device__ __forceinline__ void multiply_b(uint32_t r, uint32_t c0, v4u (&w)[kKt][W::kVecs], const v8b (&hp)[kNt][kKt][3], v4f (&acc)[kNt]) {
    const uint32_t q = (threadIdx.x & (kWave - 1)) >> 4;
#pragma unroll
    for (int c = 0; c < kKt; c++) {
        if (32 * (c0 + c) >= r) break;
        if (32 * (c0 + c) + 32 > r) {  // weights behind the adapter's rank: there, but not its own
#pragma unroll
            for (int i = 0; i < 4 * W::kVecs; i++) {
                const uint32_t per = 4 / W::kBytes, first = 32 * (c0 + c) + 8 * q + i * per;
                uint32_t keep = first < r ? ~0u : 0u;
                if (per == 2 && first + 1 >= r) keep &= 0xffffu;
                w[c][i / 4][i % 4] &= keep;
            }
        }
        v8b wp[W::kParts];
        W::parts(w[c], wp);
#pragma unroll
        for (int t = 0; t < kNt; t++) acc[t] = multiply(wp, hp[t][c], acc[t]);
    }
}

// y of few tokens.  A wave: a tile and some rows of y, 32 at a time (two matrix tiles); the
// next 32 rows' B and res are on their way while these are multiplied.  A workgroup's waves have
// one tile: past a rank of 32 they sum h's splits together (256 tokens of one adapter of rank
// 256, k and rows 4096: 22 us, each wave by itself 28).
template <class W, int kKt>
__device__ __forceinline__ void up_few(const Args& a) {
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(tid / kWave);
    const uint32_t q = lane >> 4, tile = blockIdx.y;
    Mine<1> mine;
    if (!tile_of(a, tile, mine)) return;
    const uint32_t n0 = (blockIdx.x * 4 + wid) * a.wave_rows;
    if (kKt == 1 && n0 >= a.rows) return;
    const uint32_t n1 = min(n0 + a.wave_rows, a.rows);
    const bool with = mine.adapter < a.n_adapters;
    const uint32_t r = mine.rank;
    const float scale = with && a.scales ? a.scales[mine.adapter] : 1.0f;
    const uint8_t* b = static_cast<const uint8_t*>(a.b) +
                       (with ? static_cast<uint64_t>(mine.adapter) * a.rows * a.rank * W::kBytes : 0);
    const bool live = mine.live(0);
    const uint64_t at = mine.token[0] * a.y_stride;
    v4u w[2][kKt][W::kVecs];
    v4f was[2];
    const auto load_rows = [&](uint32_t n) {
        const uint32_t col = n + 4 * q;  // and 16 on
#pragma unroll
        for (int e = 0; e < 2; e++) load_b<W, kKt>(a, b, n + 16 * e, r, 0, w[e]);
        was[0] = was[1] = v4f{0, 0, 0, 0};
        if (!a.res || !live) return;
        const float* p = a.res + at + col;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            if (a.vectors) {
                if (col + 16 * e < n1) was[e] = *reinterpret_cast<const v4f*>(p + 16 * e);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (col + 16 * e + i < n1) was[e][i] = p[16 * e + i];
            }
        }
    };
    load_rows(n0);
    v8b hp[1][kKt][3];
    if constexpr (kKt == 1) load_h(a, mine, tile, 0, hp);
    else share_h(a, mine, tile, hp);
    for (uint32_t n = n0; n < n1; n += 32) {
        v4f acc[2][1] = {{v4f{0, 0, 0, 0}}, {v4f{0, 0, 0, 0}}};
#pragma unroll
        for (int e = 0; e < 2; e++) multiply_b<W>(r, 0, w[e], hp, acc[e]);
        v4f o[2];
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[e][i] = r ? __builtin_fmaf(scale, acc[e][0][i], was[e][i]) : was[e][i];
        if (n + 32 < n1) load_rows(n + 32);
        if (!live) continue;
        const uint32_t col = n + 4 * q;
        float* p = a.y + at + col;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            if (a.vectors) {
                if (col + 16 * e < n1) *reinterpret_cast<v4f*>(p + 16 * e) = o[e];
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (col + 16 * e + i < n1) p[16 * e + i] = o[e][i];
            }
        }
    }
}

// y of many tokens: bound by res and y, which meet the products in LDS so that a wave reads and
// writes 512 bytes of a row at a time (64 bytes, straight from the matrix instruction: 150 us
// for 5000 tokens of 12288 rows, rank 64; so 122, of which 100 without the products; a plain
// copy of y 80).  A wave: a tile of 32 tokens (by 16, which read B twice as often: 141) and 128
// rows of y at a time; a workgroup's waves have neighbouring tiles and the same rows of B.  A
// rank past 32 kKt goes in several passes over the span, whose sums wait in LDS: with all of
// its h in registers a rank of 256 took 133 us for 2048 tokens of 4096 rows.
constexpr uint32_t kSpan = 128, kPitch = kSpan + 4;  // (a row of LDS begins 16 bytes past the one before's banks)

template <class W, int kKt>
__device__ __forceinline__ void up_many(const Args& a) {
    constexpr int kNt = 2;
    constexpr uint32_t kTokens = kN * kNt;
    __shared__ __attribute__((aligned(16))) float rows[4][kTokens * kPitch];
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(tid / kWave);
    const uint32_t m = lane & 15, q = lane >> 4, tile = blockIdx.y * 4 + wid;
    Mine<kNt> mine;
    if (!tile_of(a, tile, mine)) return;
    const uint32_t n0 = blockIdx.x * a.wave_rows;
    if (n0 >= a.rows) return;
    const uint32_t n1 = min(n0 + a.wave_rows, a.rows);
    const bool with = mine.adapter < a.n_adapters;
    const uint32_t r = mine.rank;
    const float scale = with && a.scales ? a.scales[mine.adapter] : 1.0f;
    const uint8_t* b = static_cast<const uint8_t*>(a.b) +
                       (with ? static_cast<uint64_t>(mine.adapter) * a.rows * a.rank * W::kBytes : 0);
    float* const mem = rows[wid];
    // matrix tiles of B in flight, and pairs of rows of res
    constexpr uint32_t kAhead = kKt * W::kVecs <= 2 ? 4 : 2, kPairs = 8, kTiles = kSpan / 16;
    const uint32_t passes = max((r + 32 * kKt - 1) / (32 * kKt), 1u);
    v4u w[kAhead][kKt][W::kVecs];
    const uint32_t half = lane >> 5, col0 = 4 * (lane & 31);  // two tokens an instruction
    v4f was[kPairs];
    uint64_t to[kPairs];
    const auto load_res = [&](uint32_t j0, uint32_t n, uint32_t span) {
#pragma unroll
        for (uint32_t j = 0; j < kPairs; j++) {
            const uint32_t at = j0 + 2 * j + half;
            const uint32_t t0 = __shfl(mine.token[0], at & 15), t1 = __shfl(mine.token[1], at & 15);
            to[j] = (at < kN ? t0 : t1) * a.y_stride + n + col0;
            was[j] = v4f{0, 0, 0, 0};
            if (a.res && at < mine.n) {
                if (a.vectors) {
                    if (col0 < span) was[j] = *reinterpret_cast<const v4f*>(a.res + to[j]);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (col0 + i < span) was[j][i] = a.res[to[j] + i];
                }
            }
        }
    };
#pragma unroll
    for (uint32_t i = 0; i < kAhead; i++) load_b<W, kKt>(a, b, n0 + 16 * i, r, 0, w[i]);
    load_res(0, n0, min(kSpan, n1 - n0));
    v8b hp[kNt][kKt][3];
    for (uint32_t n = n0; n < n1; n += kSpan) {
        const uint32_t span = min(kSpan, n1 - n);
        for (uint32_t pass = 0; pass < passes; pass++) {
            const uint32_t c0 = kKt * pass;
            if (passes > 1 || n == n0) load_h(a, mine, tile, c0, hp);
            const bool last = pass + 1 == passes;
            for (uint32_t e0 = 0; e0 < kTiles; e0 += kAhead) {
#pragma unroll
                for (uint32_t i = 0; i < kAhead; i++) {
                    const uint32_t e = e0 + i;
                    v4f acc[kNt];
#pragma unroll
                    for (int t = 0; t < kNt; t++) {
                        acc[t] = v4f{0, 0, 0, 0};
                        if (pass) acc[t] = *reinterpret_cast<const v4f*>(mem + (kN * t + m) * kPitch + 16 * e + 4 * q);
                    }
                    multiply_b<W>(r, c0, w[i], hp, acc);
                    // the next: of this run of the rank, or the next one's first
                    const bool on = e + kAhead < kTiles;
                    load_b<W, kKt>(a, b, (on || !last ? n : n + kSpan) + 16 * (on ? e + kAhead : i), r, on ? c0 : last ? 0 : c0 + kKt, w[i]);
#pragma unroll
                    for (int t = 0; t < kNt; t++) *reinterpret_cast<v4f*>(mem + (kN * t + m) * kPitch + 16 * e + 4 * q) = acc[t];
                }
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // a wave's own: no barrier
        for (uint32_t j0 = 0; j0 < mine.n; j0 += 2 * kPairs) {
            if (j0) load_res(j0, n, span);
#pragma unroll
            for (uint32_t j = 0; j < kPairs; j++) {
                const uint32_t at = j0 + 2 * j + half;
                if (at >= mine.n) continue;
                const v4f d = *reinterpret_cast<const v4f*>(mem + at * kPitch + col0);
                v4f o;
#pragma unroll
                for (int i = 0; i < 4; i++) o[i] = r ? __builtin_fmaf(scale, d[i], was[j][i]) : was[j][i];
                if (a.vectors) {
                    if (col0 < span) *reinterpret_cast<v4f*>(a.y + to[j]) = o;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (col0 + i < span) a.y[to[j] + i] = o[i];
                }
            }
        }
        if (n + kSpan < n1) load_res(0, n + kSpan, min(kSpan, n1 - n - kSpan));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the next rows are written
    }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(1024) zlm_lora_group(Args a) { group(a); }

#define ZLM_LORA_DOWN(NAME, W, kMt, S, kNt)                                                                       \
    extern "C" __global__ void __launch_bounds__(64 * zlm::kLoraWaves[kNt - 1]) zlm_lora_down_##NAME##_##kMt##S(Args a) { \
        down<W, kMt, kNt>(a);                                                                                     \
    }
#define ZLM_LORA_UP_FEW(NAME, W, kKt)                                                                             \
    extern "C" __global__ void __launch_bounds__(256) zlm_lora_up_##NAME##_##kKt##_small(Args a) { up_few<W, kKt>(a); }
#define ZLM_LORA_UP_MANY(NAME, W, kKt)                                                                            \
    extern "C" __global__ void __launch_bounds__(256, 2) zlm_lora_up_##NAME##_##kKt(Args a) { up_many<W, kKt>(a); }
#define ZLM_LORA(NAME, W)                                                                                         \
    ZLM_LORA_DOWN(NAME, W, 1, , 2)                                                                                \
    ZLM_LORA_DOWN(NAME, W, 2, , 2)                                                                                \
    ZLM_LORA_DOWN(NAME, W, 4, , 2)                                                                                \
    ZLM_LORA_DOWN(NAME, W, 8, , 2)                                                                                \
    ZLM_LORA_DOWN(NAME, W, 1, _small, 1)                                                                          \
    ZLM_LORA_DOWN(NAME, W, 2, _small, 1)                                                                          \
    ZLM_LORA_DOWN(NAME, W, 4, _small, 1)                                                                          \
    ZLM_LORA_DOWN(NAME, W, 8, _small, 1)                                                                          \
    ZLM_LORA_UP_MANY(NAME, W, 1)                                                                                  \
    ZLM_LORA_UP_MANY(NAME, W, 2)                                                                                  \
    ZLM_LORA_UP_FEW(NAME, W, 1)                                                                                   \
    ZLM_LORA_UP_FEW(NAME, W, 2)                                                                                   \
    ZLM_LORA_UP_FEW(NAME, W, 4)                                                                                   \
    ZLM_LORA_UP_FEW(NAME, W, 8)
ZLM_LORA(bf16, Bf16)
ZLM_LORA(f16, F16)
ZLM_LORA(f32, F32)
