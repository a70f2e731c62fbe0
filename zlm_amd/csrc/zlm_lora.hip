// zlm_lora.hip -- CDNA4 (gfx950) kernels of low-rank adapters: each token of a batch has
// one of many pairs A (rank x k), B (rows x rank), or none, and
//     y[t] = res[t] + scale * B (A x[t]).
// Built as a device-only code object (hipcc --genco) and loaded by the host library.
//
// Tokens are taken in tiles of up to 16 with one adapter, so that a tile reads its A and B
// once.  Up to 64 tokens every wave finds its tile by itself; more are grouped by a launch
// before.  Then two launches: h = A x, k split over waves and workgroups, and
// y = res + scale * B h.
//
// Both products run on v_mfma_f32_16x16x32_bf16 with the tokens in the N dimension.  A
// 32-bit number is the sum of three bf16 (8 bits of its 24 each, cut off, so exactly), an
// f16 of two, and a product is the sum of its parts' products without those below 2^-24 of
// it: three instructions for a bf16 adapter, six for f16 and f32.  So the results have the
// accuracy of 32-bit products at 10 and 5 times the rate of the 32-bit matrix instruction.
// bf16 has the exponents of 32 bits: nothing is scaled.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "lora_args.h"

namespace {

using Args = zlm::LoraArgs;
using zlm::LoraTile;
constexpr uint32_t kWave = 64, kTile = zlm::kLoraTile, kWaves = zlm::kLoraWaves;

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
// two numbers of three parts those of 2^-24 and below are left out.
template <int kN>
__device__ __forceinline__ v4f multiply(const v8b (&w)[kN], const v8b (&x)[3], v4f acc) {
#pragma unroll
    for (int s = kN + 1; s >= 0; s--)
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int j = s - i;
            if (j < 0 || j > 2 || (kN == 3 && s > 2)) continue;
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[i], x[j], acc, 0, 0, 0);
        }
    return acc;
}

// ---- tiles ----

// A tile, and this lane's token of it (lane % 16; the tile's first where it has fewer).
struct Mine {
    uint32_t adapter, n, token;
    bool live;
};

__device__ __forceinline__ uint32_t adapter_of(const Args& a, uint32_t t) {
    return min(static_cast<uint32_t>(a.adapter[t]), a.n_adapters);  // n_adapters: none
}

// False: there are not so many tiles.  Tokens without an adapter make tiles of their own,
// but where y is res.
template <bool kSmall>
__device__ __forceinline__ bool tile_of(const Args& a, uint32_t tile, Mine& m) {
    const uint32_t lane = threadIdx.x & (kWave - 1), j = lane & (kTile - 1);
    if constexpr (kSmall) {
        const bool has = lane < a.n_tokens;
        const uint32_t own = has ? adapter_of(a, lane) : a.n_adapters;
        uint64_t left = __ballot(has && !(a.in_place && own == a.n_adapters));
        while (left) {
            const uint32_t id = __builtin_amdgcn_readlane(own, __builtin_ctzll(left));
            uint64_t with = __ballot(own == id) & left;
            const uint32_t n = __builtin_popcountll(with), tiles = (n + kTile - 1) / kTile;
            if (tile < tiles) {
                m.adapter = id;
                m.n = min(n - kTile * tile, kTile);
                m.live = j < m.n;
                // the (16 tile + j)-th of them: the lane that so many come before
                const uint32_t before = __builtin_popcountll(with & ((1ull << lane) - 1));
                const bool in = (with >> lane & 1) != 0;
                const uint32_t to = in ? before - kTile * tile : kWave;
                // each of the tile's tokens tells the lane of its place
                m.token = __builtin_ctzll(with);
                for (uint32_t i = 0; i < m.n; i++) {
                    const uint32_t t = __builtin_ctzll(__ballot(to == i));
                    if (j == i) m.token = t;
                }
                return true;
            }
            tile -= tiles;
            left &= ~with;
        }
        return false;
    } else {
        if (tile >= *a.n_tiles) return false;
        const LoraTile t = a.tile[tile];
        m.adapter = t.adapter;
        m.n = t.n;
        m.live = j < t.n;
        m.token = a.order[t.first + (m.live ? j : 0)];
        return true;
    }
}

__device__ __forceinline__ uint32_t rank_of(const Args& a, uint32_t adapter) {
    return a.ranks ? min(static_cast<uint32_t>(max(a.ranks[adapter], 0)), a.rank) : a.rank;
}

// The tokens by adapter: counted, their places summed up, then put there (in any order: a
// token's result does not depend on its place).  One workgroup.
__device__ __forceinline__ void group(const Args& a) {
    constexpr uint32_t kThreads = 1024, kMost = zlm::kLoraAdapters + 1, kPer = (kMost + kThreads - 1) / kThreads;
    __shared__ uint32_t count[kPer * kThreads], tiles_to[kPer * kThreads];
    __shared__ uint32_t sums[2][kThreads / kWave];
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wid = tid / kWave;
    const uint32_t groups = a.n_adapters + (a.in_place ? 0 : 1);
    for (uint32_t i = tid; i < kPer * kThreads; i += kThreads) count[i] = 0;
    __syncthreads();
    for (uint32_t t = tid; t < a.n_tokens; t += kThreads) {
        // one atomic for the tokens of a wave that are its first's
        const uint32_t id = adapter_of(a, t);
        const uint32_t head = __builtin_amdgcn_readfirstlane(id);
        const uint64_t same = __ballot(id == head);
        if (id != head) atomicAdd(&count[id], 1u);
        else if (lane == static_cast<uint32_t>(__builtin_ctzll(same))) atomicAdd(&count[id], static_cast<uint32_t>(__builtin_popcountll(same)));
    }
    __syncthreads();
    // exclusive sums of tokens and tiles, kPer groups a thread
    uint32_t n = 0, k = 0, own[kPer];
#pragma unroll
    for (uint32_t i = 0; i < kPer; i++) {
        const uint32_t g = tid * kPer + i;
        own[i] = g < groups ? count[g] : 0;
        n += own[i];
        k += (own[i] + kTile - 1) / kTile;
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
    for (uint32_t i = 0; i < kThreads / kWave; i++) {
        if (i < wid) {
            to_n += sums[0][i];
            to_k += sums[1][i];
        }
        all += sums[1][i];
    }
    to_n -= n;
    to_k -= k;
#pragma unroll
    for (uint32_t i = 0; i < kPer; i++) {
        const uint32_t g = tid * kPer + i;
        count[g] = to_n;  // from here on the place of the group's next token
        tiles_to[g] = to_k;
        to_n += own[i];
        to_k += (own[i] + kTile - 1) / kTile;
    }
    __syncthreads();
    for (uint32_t i = tid; i < all; i += kThreads) {
        uint32_t lo = 0, hi = groups;  // the last group that begins at or before tile i
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (tiles_to[mid] <= i) lo = mid;
            else hi = mid;
        }
        const uint32_t at = kTile * (i - tiles_to[lo]);
        const uint32_t end = lo + 1 < kPer * kThreads ? count[lo + 1] : 0;
        a.tile[i] = {lo, count[lo] + at, min(end - count[lo] - at, kTile)};
    }
    if (tid == 0) *a.n_tiles = all;
    __syncthreads();
    for (uint32_t t = tid; t < a.n_tokens; t += kThreads) {
        const uint32_t id = adapter_of(a, t);
        if (id >= groups) continue;
        const uint32_t head = __builtin_amdgcn_readfirstlane(id);
        const uint64_t same = __ballot(id == head);
        const uint32_t first = __builtin_ctzll(same);
        uint32_t at = 0;
        if (id != head) at = atomicAdd(&count[id], 1u);
        else if (lane == first) at = atomicAdd(&count[id], static_cast<uint32_t>(__builtin_popcountll(same)));
        const uint32_t base = __builtin_amdgcn_readlane(at, first);
        if (id == head) at = base + __builtin_popcountll(same & ((1ull << lane) - 1));
        a.order[at] = t;
    }
}

// ---- h = A x ----
//
// A workgroup: a tile, a split of k, up to 16 kMt rows of A.  Its waves take k in turn
// (runs of 32, the lane's eight of them together) and add up their sums through LDS.
template <class W, int kMt, bool kSmall>
__device__ __forceinline__ void down(const Args& a) {
    __shared__ v4f sums[kWaves][kMt < 4 ? kMt : 4][kWave];
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(tid / kWave);
    const uint32_t m = lane & 15, q = lane >> 4, tile = blockIdx.x, split = blockIdx.y;
    Mine mine;
    if (!tile_of<kSmall>(a, tile, mine) || mine.adapter >= a.n_adapters) return;
    const uint32_t r = rank_of(a, mine.adapter), r0 = 16 * kMt * blockIdx.z;
    if (r0 >= r) return;
    const uint32_t chunks = a.k / 32, parts = a.splits * kWaves, part = split * kWaves + wid;
    const uint32_t c0 = static_cast<uint64_t>(chunks) * part / parts, c1 = static_cast<uint64_t>(chunks) * (part + 1) / parts;
    const float* x = a.x + mine.token * a.x_stride + 8 * q;
    const uint8_t* w[kMt];
#pragma unroll
    for (int i = 0; i < kMt; i++) {
        const uint32_t row = min(r0 + 16 * i + m, a.rank - 1);
        w[i] = static_cast<const uint8_t*>(a.a) + ((static_cast<uint64_t>(mine.adapter) * a.rank + row) * a.k + 8 * q) * W::kBytes;
    }
    v4f acc[kMt];
#pragma unroll
    for (int i = 0; i < kMt; i++) acc[i] = v4f{0, 0, 0, 0};
    constexpr uint32_t kU = kMt <= 2 ? 4 : 2;  // runs in flight
    for (uint32_t c = c0; c < c1; c += kU) {
        float xv[kU][8];
        v4u wv[kU][kMt][W::kVecs];
#pragma unroll
        for (uint32_t u = 0; u < kU; u++) {
            const uint32_t at = 32 * min(c + u, c1 - 1);
            v4f lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
            if (mine.live) {
                lo = *reinterpret_cast<const v4f*>(x + at);
                hi = *reinterpret_cast<const v4f*>(x + at + 4);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                xv[u][i] = lo[i];
                xv[u][4 + i] = hi[i];
            }
#pragma unroll
            for (int i = 0; i < kMt; i++)
                if (r0 + 16 * i < r) load<W>(w[i] + static_cast<size_t>(at) * W::kBytes, wv[u][i]);
        }
#pragma unroll
        for (uint32_t u = 0; u < kU; u++) {
            if (c + u >= c1) break;
            v8b xp[3];
            to_parts(xv[u], xp);
#pragma unroll
            for (int i = 0; i < kMt; i++) {
                if (r0 + 16 * i >= r) break;
                v8b wp[W::kParts];
                W::parts(wv[u][i], wp);
                acc[i] = multiply(wp, xp, acc[i]);
            }
        }
    }
    float* to = a.part + ((static_cast<uint64_t>(split) * a.tiles + tile) * kTile) * a.rank;
    constexpr int kStep = kMt < 4 ? kMt : 4;
#pragma unroll
    for (int i0 = 0; i0 < kMt; i0 += kStep) {
        if (i0) __syncthreads();
#pragma unroll
        for (int i = 0; i < kStep; i++) sums[wid][i][lane] = acc[i0 + i];
        __syncthreads();
        for (uint32_t i = wid; i < kStep; i += kWaves) {
            v4f s = sums[0][i][lane];
#pragma unroll
            for (uint32_t v = 1; v < kWaves; v++) s += sums[v][i][lane];
            const uint32_t row = r0 + 16 * (i0 + i) + 4 * q;
            if (m < mine.n && row < a.rank) *reinterpret_cast<v4f*>(to + m * a.rank + row) = s;
        }
    }
}

// ---- y = res + scale B h ----
//
// A wave: a tile and kLoraRows rows of y, 32 at a time: two matrix tiles whose rows are
// dealt so that a lane's results are eight values of y in a row.  kKt: runs of 32 of the rank.
template <class W, int kKt, bool kSmall>
__device__ __forceinline__ void up(const Args& a) {
    const uint32_t tid = threadIdx.x, lane = tid & (kWave - 1), wid = __builtin_amdgcn_readfirstlane(tid / kWave);
    const uint32_t m = lane & 15, q = lane >> 4, tile = blockIdx.x;
    Mine mine;
    if (!tile_of<kSmall>(a, tile, mine)) return;
    const uint32_t n0 = (blockIdx.y * 4 + wid) * zlm::kLoraRows;
    if (n0 >= a.rows) return;
    const uint32_t n1 = min(n0 + zlm::kLoraRows, a.rows);
    const bool with = mine.adapter < a.n_adapters;
    const uint32_t r = with ? rank_of(a, mine.adapter) : 0;
    const float scale = with && a.scales ? a.scales[mine.adapter] : 1.0f;
    const uint64_t at = mine.token * a.y_stride;
    v8b hp[kKt][3];
#pragma unroll
    for (int c = 0; c < kKt; c++) {
        float h[8];
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = 0.0f;
        const uint32_t k = 32 * c + 8 * q;
        if (mine.live && k < r) {
            for (uint32_t s = 0; s < a.splits; s++) {
                const float* p = a.part + ((static_cast<uint64_t>(s) * a.tiles + tile) * kTile + m) * a.rank + k;
                const v4f lo = reinterpret_cast<const v4f*>(p)[0], hi = reinterpret_cast<const v4f*>(p)[1];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    h[i] += lo[i];
                    h[4 + i] += hi[i];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = k + i < r ? h[i] : 0.0f;
        to_parts(h, hp[c]);
    }
    const uint8_t* b = static_cast<const uint8_t*>(a.b) +
                       (with ? static_cast<uint64_t>(mine.adapter) * a.rows * a.rank * W::kBytes : 0);
    for (uint32_t n = n0; n < n1; n += 32) {
        v4u wv[2][kKt][W::kVecs];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const uint32_t row = min(n + 8 * (m >> 2) + 4 * e + (m & 3), a.rows - 1);
            const uint8_t* p = b + (static_cast<uint64_t>(row) * a.rank + 8 * q) * W::kBytes;
#pragma unroll
            for (int c = 0; c < kKt; c++) {
                const uint32_t k = 32 * c + 8 * q;
#pragma unroll
                for (int i = 0; i < W::kVecs; i++) wv[e][c][i] = v4u{0, 0, 0, 0};
                if (k < r) load<W>(p + 32 * c * W::kBytes, wv[e][c]);
            }
        }
        const uint32_t col = n + 8 * q;
        float was[8];
#pragma unroll
        for (int i = 0; i < 8; i++) was[i] = 0.0f;
        if (a.res && mine.live) {
            const float* p = a.res + at + col;
            if (a.vectors) {
#pragma unroll
                for (int e = 0; e < 2; e++)
                    if (col + 4 * e < n1) {
                        const v4f v = reinterpret_cast<const v4f*>(p)[e];
#pragma unroll
                        for (int i = 0; i < 4; i++) was[4 * e + i] = v[i];
                    }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (col + i < n1) was[i] = p[i];
            }
        }
        v4f acc[2] = {v4f{0, 0, 0, 0}, v4f{0, 0, 0, 0}};
#pragma unroll
        for (int c = 0; c < kKt; c++) {
            if (32u * c >= r) break;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                if (32u * c + 32 > r) {  // weights behind the adapter's rank: there, but not its own
                    const uint32_t k = 32 * c + 8 * q;
#pragma unroll
                    for (int i = 0; i < 4 * W::kVecs; i++) {
                        const uint32_t per = 4 / W::kBytes, first = k + i * per;
                        uint32_t keep = first < r ? ~0u : 0u;
                        if (per == 2 && first + 1 >= r) keep &= 0xffffu;
                        wv[e][c][i / 4][i % 4] &= keep;
                    }
                }
                v8b wp[W::kParts];
                W::parts(wv[e][c], wp);
                acc[e] = multiply(wp, hp[c], acc[e]);
            }
        }
        if (!mine.live) continue;
        float* p = a.y + at + col;
        v4f o[2];
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[e][i] = r ? __builtin_fmaf(scale, acc[e][i], was[4 * e + i]) : was[4 * e + i];
        if (a.vectors) {
#pragma unroll
            for (int e = 0; e < 2; e++)
                if (col + 4 * e < n1) reinterpret_cast<v4f*>(p)[e] = o[e];
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (col + i < n1) p[i] = o[i / 4][i % 4];
        }
    }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(1024) zlm_lora_group(Args a) { group(a); }

#define ZLM_LORA(NAME, W, S, kSmall)                                                                              \
    extern "C" __global__ void __launch_bounds__(512) zlm_lora_down_##NAME##_1##S(Args a) { down<W, 1, kSmall>(a); } \
    extern "C" __global__ void __launch_bounds__(512) zlm_lora_down_##NAME##_2##S(Args a) { down<W, 2, kSmall>(a); } \
    extern "C" __global__ void __launch_bounds__(512) zlm_lora_down_##NAME##_4##S(Args a) { down<W, 4, kSmall>(a); } \
    extern "C" __global__ void __launch_bounds__(512) zlm_lora_down_##NAME##_8##S(Args a) { down<W, 8, kSmall>(a); } \
    extern "C" __global__ void __launch_bounds__(256) zlm_lora_up_##NAME##_1##S(Args a) { up<W, 1, kSmall>(a); }     \
    extern "C" __global__ void __launch_bounds__(256) zlm_lora_up_##NAME##_2##S(Args a) { up<W, 2, kSmall>(a); }     \
    extern "C" __global__ void __launch_bounds__(256) zlm_lora_up_##NAME##_4##S(Args a) { up<W, 4, kSmall>(a); }     \
    extern "C" __global__ void __launch_bounds__(256) zlm_lora_up_##NAME##_8##S(Args a) { up<W, 8, kSmall>(a); }
ZLM_LORA(bf16, Bf16, , false)
ZLM_LORA(f16, F16, , false)
ZLM_LORA(f32, F32, , false)
ZLM_LORA(bf16, Bf16, _small, true)
ZLM_LORA(f16, F16, _small, true)
ZLM_LORA(f32, F32, _small, true)
