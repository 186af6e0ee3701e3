// What surrounds the attention of a serving step, for gfx950: block tables from an engine's token map, a prefill step's
// index arrays from the requests' lengths, and the next tokens from the logits (include/kushkash_amd_step.h).
#include <algorithm>
#include <cmath>

#include "kush_common.h"
#include "kushkash_amd_step.h"

namespace kush {

// int32 or int64 entry i
__device__ __forceinline__ int64_t wide_at(const void* p, int wide, int64_t i) {
    return wide ? reinterpret_cast<const int64_t*>(p)[i] : reinterpret_cast<const int32_t*>(p)[i];
}

// ------------------------------------------------------------------ block tables
// grid (n_reqs, ceil(pages / 256)), block 256: a page per thread. The map is read once per page, 128 bytes apart, so
// its reads take a cache line each: the bytes moved are 32 times those used.
__global__ __launch_bounds__(256) void block_table_kernel(const int32_t* __restrict__ map, int64_t map_stride,
                                                          int64_t map_rows, int64_t map_cols, const void* __restrict__ req,
                                                          int wide_req, const void* __restrict__ lens, int wide_lens,
                                                          int64_t pages, int32_t* __restrict__ table, int64_t stride,
                                                          int32_t* __restrict__ lens_out, int32_t* __restrict__ slots_out) {
    const int64_t r = blockIdx.x, p = (int64_t)blockIdx.y * 256 + threadIdx.x;
    const int64_t id = wide_at(req, wide_req, r), n = wide_at(lens, wide_lens, r);
    if (p == 0) {
        if (lens_out != nullptr) lens_out[r] = (int32_t)n;
        if (slots_out != nullptr) slots_out[r] = (int32_t)id;
    }
    if (p >= pages) return;
    const int64_t seen = id >= 0 && id < map_rows ? (n < map_cols ? n : map_cols) : 0;
    table[r * stride + p] = p * PAGE < seen ? map[id * map_stride + p * PAGE] >> 5 : 0;
}

// ------------------------------------------------------------------ maps of a prefill step
struct MapArgs {
    const int32_t *new_tokens, *history, *slots, *table;
    int64_t stride, cols;
    int n, window, sinks;
    int64_t jobs, pages, tails, tokens;
    int32_t *q_start, *key_start, *seq_lens, *job_seq, *job_page, *page_blk, *page_dst, *tail_blk, *tail_info, *new_dst;
    int64_t* slot_map;
};

// What one request adds to each array (64 bits: sums of any lengths stay sums, and behind the arrays' ends)
struct MapCounts {
    int64_t tokens, keys, pages, jobs, tails;
    __device__ __forceinline__ MapCounts& operator+=(const MapCounts& o) {
        tokens += o.tokens;
        keys += o.keys;
        pages += o.pages;
        jobs += o.jobs;
        tails += o.tails;
        return *this;
    }
};

__device__ __forceinline__ int pages_left_out(const MapArgs& a, int h) {
    if (a.window == 0) return 0;
    const int first = a.sinks / PAGE + (a.sinks % PAGE != 0);
    return max(0, (h >= a.window ? h - a.window + 1 : 0) / PAGE - first);
}

__device__ __forceinline__ MapCounts counts_of(const MapArgs& a, int t, int h) {
    const int gap = pages_left_out(a, h);
    return MapCounts{t, (int64_t)(h - PAGE * gap) + t, h / PAGE - gap, t > 0 ? (int)(((uint32_t)h + t - 1) / PAGE) - h / PAGE + 1 : 0,
                     h % PAGE != 0};
}

__device__ __forceinline__ int64_t wave_sum(int64_t x) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) x += __shfl_xor(x, m, WAVE);
    return x;
}

// grid (n, parts), block 256: a request's entries, dealt to its `parts` workgroups. Where they begin is the sum over the
// requests before it, which every workgroup forms by itself: a few loads per thread for a few hundred requests, against a
// second launch.
__global__ __launch_bounds__(256) void step_maps_kernel(const MapArgs a) {
    __shared__ MapCounts part[4];
    const int r = blockIdx.x, tid = threadIdx.x;
    MapCounts before{0, 0, 0, 0, 0};
    for (int i = tid; i < r; i += 256) before += counts_of(a, max(0, a.new_tokens[i]), max(0, a.history[i]));
    before = MapCounts{wave_sum(before.tokens), wave_sum(before.keys), wave_sum(before.pages), wave_sum(before.jobs),
                       wave_sum(before.tails)};
    if (tid % WAVE == 0) part[tid / WAVE] = before;
    __syncthreads();
    before = part[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) before += part[w];
    const int t = max(0, a.new_tokens[r]), h = max(0, a.history[r]);
    const MapCounts mine = counts_of(a, t, h);
    const int full = h / PAGE, gap = pages_left_out(a, h), kept = h - PAGE * gap;
    const int first = a.sinks / PAGE + (a.sinks % PAGE != 0);
    const int32_t* const table = a.table + (int64_t)r * a.stride;
    const auto block = [&](uint32_t p) { return p < a.cols ? table[p] : 0; };
    if (tid == 0 && blockIdx.y == 0) {
        a.q_start[r] = (int32_t)before.tokens;
        a.key_start[r] = (int32_t)before.keys;
        a.seq_lens[r] = (int32_t)((uint32_t)h + t);
        if (r == a.n - 1) {
            a.q_start[a.n] = (int32_t)(before.tokens + mine.tokens);
            a.key_start[a.n] = (int32_t)(before.keys + mine.keys);
        }
        if (mine.tails && before.tails < a.tails) {
            a.tail_blk[before.tails] = block(full);
            int32_t* const info = a.tail_info + 3 * before.tails;
            info[0] = (int32_t)(before.keys + PAGE * mine.pages);
            info[1] = h % PAGE;
            info[2] = a.slots[r];
        }
    }
    const auto room = [](int64_t n, int64_t first, int64_t size) { return (int)max((int64_t)0, min(n, size - first)); };
    const int jobs = room(mine.jobs, before.jobs, a.jobs), pages = room(mine.pages, before.pages, a.pages),
              tokens = room(t, before.tokens, a.tokens), key = (int)before.keys;
    const int i0 = (int)blockIdx.y * 256 + tid, step = (int)gridDim.y * 256;
    for (int i = i0; i < jobs; i += step) {
        a.job_seq[before.jobs + i] = r;
        a.job_page[before.jobs + i] = full + i;
    }
    for (int i = i0; i < pages; i += step) {
        a.page_blk[before.pages + i] = block(i < first ? i : i + gap);
        a.page_dst[before.pages + i] = key + PAGE * i;
    }
    for (int i = i0; i < tokens; i += step) {
        const uint32_t at = (uint32_t)h + i;
        a.new_dst[before.tokens + i] = key + kept + i;
        a.slot_map[before.tokens + i] = (int64_t)block(at / PAGE) * PAGE + at % PAGE;
    }
}

// ------------------------------------------------------------------ sampling
// One token per row in four launches (one for a vocabulary of up to TILE tokens); every sum is an integer, so no order of
// workgroups, lanes or atomics changes it.
// A weight w = exp((x - max) / T) is held as a multiple of 2^-bits in 64 bits, one unit at least where w > 0; bits = min(50,
// 63 - log2 vocab), such that the vocabulary's sum fits. Together the weights are off by a unit a token at most: by 2^-25 of
// the largest at 2^19 tokens, half the least random number of 24 bits, and by 2^-15 at 2^24 tokens.
//   1. sample_max     every workgroup a piece of a row: its largest logit and where, its smallest, NaN; the row's bins
//                     cleared for the next launch
//   2. sample_bins    the tokens in BINS classes of equal width below the largest logit (class 0: next to it), their
//                     number and, where top-p asks, their mass: in LDS, the classes that are not empty added to the row's
//   3. sample_pick    the classes that the cuts of top-k and top-p fall into, from the bins; the mass of every tile's
//                     tokens above them; the tokens inside them to the row's list (a few hundred of 150,000, as a rule)
//   4. sample_token   the exact cuts, ties by index: in the list, by classes of its own and a sort of the few tokens next
//                     to the cuts; then the token in the vocabulary's order, in the list where top-k bounds it, else in the
//                     tile that u times the kept mass falls into
// What it has to read is the logits, once; the passes read them three times, the later ones from the caches. One row of
// 152,000 bf16 with top-k 50 and top-p takes 20 us (4, 5, 5 and 6: the launches' own times and the steps of one workgroup
// over the list), 64 fp32 rows 47 (9, 11, 13 and 14: 39 MB, 8 us at the card's copy rate).
// A list of more than LIST tokens is cut by a radix search over the row instead, in one workgroup: thousands of equal logits next
// to a cut, or fewer logits above -inf than top_k, which brings every masked token of the row into the list. Of 152,000 tokens
// 20 allowed, top_k 50: one row 1.8 ms, 64 rows 2.2, with top-p 2.5 and 3.5 (all allowed: 20 and 38 us).
struct SampleArgs {
    const void* logits;
    int64_t stride;
    int vocab, bits, tiles, per;     // tiles of TILE tokens, `per` of them to a workgroup
    const float* uniforms;
    double temperature, top_p, min_p;
    int top_k;
    const float *temperatures, *top_ps, *min_ps;
    const int32_t* top_ks;
    int64_t* out;
    // scratch, per row: parts [pieces], bins [BINS] mass and count, tile sums [tiles], the list's length, the list
    struct SamplePart* parts;
    uint64_t *mass, *sums;
    uint32_t *count, *length;
    uint2* list;
    int index_bits;                  // of a token's index
    int64_t row0;                    // the first row of this launch (its scratch is row 0's)
};

// A piece of a row
struct SamplePart {
    float most, least;               // least: the smallest above -inf
    int at;                          // the first index of most
    int nan;
};

constexpr int BINS = 1024, TILE = 4096, LIST = 8192, PIECE_THREADS = 256;
// top_k up to here: the list takes every token down to the class of top-k's cut, so that neither the bins nor the tiles need
// masses. With top-p, this way and with masses: 64 rows of 152,000 with top_k 2,100 57 us and 69, 4,000 66 and 70;
// one row, whose list one workgroup draws from, 2,100 38 and 35, 4,000 46 and 37
constexpr int SMALL_K = 2048;
constexpr float SPAN = 64.0f;        // logits (in units of max(1, T)) that the bins cover at most

// logits in an order of their own: larger logit, larger key; -0 and 0 alike
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }

// a b + c, c the same in every lane and kept in scalar registers (the compiler's own form copies it for every use)
__device__ __forceinline__ double fma_const(double a, double b, double c) {
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
    return r;
}

// 2^t for t <= 0: e^z, |z| <= ln 2 / 2, by its Taylor polynomial of degree 12 (2e-16 off), times a power of two
__device__ __forceinline__ double exp2_64(double t) {
    const double n = __builtin_rint(t), z = (t - n) * 0.693147180559945309417;       // 2^f = e^z
    constexpr double inv[13] = {1.0,          1.0,           1.0 / 2,        1.0 / 6,          1.0 / 24,
                                1.0 / 120,    1.0 / 720,     1.0 / 5040,     1.0 / 40320,      1.0 / 362880,
                                1.0 / 3628800, 1.0 / 39916800, 1.0 / 479001600};
    double p = inv[12];
#pragma unroll
    for (int i = 11; i >= 3; --i) p = fma_const(p, z, inv[i]);
#pragma unroll
    for (int i = 2; i >= 0; --i) p = __builtin_fma(p, z, inv[i]);
    return t < -1100.0 ? 0.0 : __builtin_ldexp(p, (int)n);
}

// What a row is drawn with, and where its weights and bins are counted from
struct SampleRow {
    double c, top_p, min_p;          // c = log2 e / T
    float most, scale;               // scale: bins per logit
    int top_k, at;                   // top_k 0: off; at: the first of the order
    bool none, greedy, by_mass, bin_mass, small_k;      // bin_mass: top-p is cut by the row's bins' masses
    int bits;
    __device__ __forceinline__ double weight(float x) const { return exp2_64(x == most ? 0.0 : ((double)x - (double)most) * c); }
    // w >= 0 in multiples of 2^-bits, at least one where w is above 0
    __device__ __forceinline__ uint64_t fixed(double w) const {
        const double big = __builtin_fma(w, __builtin_ldexp(1.0, bits), 4503599627370496.0);       // + 2^52
        const uint64_t m = __builtin_bit_cast(uint64_t, big) & 0xFFFFFFFFFFFFFull;
        return w > 0.0 ? (m ? m : 1) : 0;
    }
    // the class of a logit: as d = most - x grows, never smaller
    __device__ __forceinline__ int bin(float x) const { return bin(x, scale); }
    __device__ __forceinline__ int bin(float x, float s) const {
        const float d = x == most ? 0.0f : (most - x) * s;
        return d < (float)(BINS - 1) ? (int)d : BINS - 1;
    }
};

// x is 16 bytes of a row's logits; elements past the vocabulary read as -inf
template <typename T>
struct Chunk {
    static constexpr int E = 16 / sizeof(T);
    float x[E];
    __device__ __forceinline__ void load(const T* row, int i, int vocab) {
        if (i + E <= vocab) {
            T v[E];
            __builtin_memcpy(v, row + i, sizeof(v));
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = to_f32(v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = i + e < vocab ? to_f32(row[i + e]) : -__builtin_inff();
        }
    }
};

// A thread's chunks of a tile
template <typename T, int THREADS>
struct TileChunks {
    static constexpr int E = Chunk<T>::E, N = TILE / (THREADS * E);
    static_assert(N * THREADS * E == TILE, "whole chunks");
    Chunk<T> c[N];
    __device__ __forceinline__ static int first(int tile, int j) { return tile * TILE + (j * THREADS + (int)threadIdx.x) * E; }
    __device__ __forceinline__ void load(const T* row, int tile, int vocab) {
#pragma unroll
        for (int j = 0; j < N; ++j) c[j].load(row, first(tile, j), vocab);
    }
    // fn(index, value) of each
    template <typename Fn>
    __device__ __forceinline__ void each(int tile, Fn&& fn) const {
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) fn(first(tile, j) + e, c[j].x[e]);
    }
};

__device__ __forceinline__ SamplePart merge_parts(SamplePart a, const SamplePart& b) {
    if (b.most > a.most || (b.most == a.most && b.at < a.at)) {
        a.most = b.most;
        a.at = b.at;
    }
    a.least = __builtin_fminf(a.least, b.least);
    a.nan |= b.nan;
    return a;
}
// op over the wave's lanes, in all of them, on the VALU
template <typename Op>
__device__ __forceinline__ float wave_all(float x, Op&& op) {
    x = op(x, lane_xor<1>(x));
    x = op(x, lane_xor<2>(x));
    x = op(x, lane_xor<4>(x));
    x = op(x, lane_xor<8>(x));
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ SamplePart wave_part(SamplePart p) {
    const auto larger = [](float u, float v) { return __builtin_fmaxf(u, v); };
    const auto smaller = [](float u, float v) { return __builtin_fminf(u, v); };
    SamplePart r;
    r.most = wave_all(p.most, larger);
    r.least = wave_all(p.least, smaller);
    const auto first = [](float u, float v) { return __int_as_float(min(__float_as_int(u), __float_as_int(v))); };
    r.at = __float_as_int(wave_all(__int_as_float(p.most == r.most ? p.at : 0x7fffffff), first));
    r.nan = __any(p.nan);
    return r;
}
// a logit, the indexes ascending within a thread
__device__ __forceinline__ void merge_logit(SamplePart& p, int i, float x) {
    p.nan |= x != x;
    p.least = x > -__builtin_inff() ? __builtin_fminf(p.least, x) : p.least;
    if (x > p.most) {
        p.most = x;
        p.at = i;
    }
}
constexpr SamplePart NO_PART{-__builtin_inff(), __builtin_inff(), 0x7fffffff, 0};

template <typename T>
__global__ __launch_bounds__(PIECE_THREADS) void sample_max(const SampleArgs a) {
    __shared__ SamplePart ws[PIECE_THREADS / WAVE];
    const int64_t s = blockIdx.y, r = a.row0 + s;
    const int piece = blockIdx.x, pieces = gridDim.x, tid = threadIdx.x;
    const T* const row = reinterpret_cast<const T*>(a.logits) + r * a.stride;
    for (int i = piece * PIECE_THREADS + tid; i < BINS; i += pieces * PIECE_THREADS) {
        a.mass[s * BINS + i] = 0;
        a.count[s * BINS + i] = 0;
    }
    if (piece == 0 && tid == 0) a.length[s] = 0;
    SamplePart p = NO_PART;
    const int end = min(a.tiles, (piece + 1) * a.per);
    for (int t = piece * a.per; t < end; ++t) {
        TileChunks<T, PIECE_THREADS> now;
        now.load(row, t, a.vocab);
        now.each(t, [&](int i, float x) { merge_logit(p, i, x); });
    }
    p = wave_part(p);
    if (tid % WAVE == 0) ws[tid / WAVE] = p;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < PIECE_THREADS / WAVE; ++w) p = merge_parts(p, ws[w]);
        a.parts[s * pieces + piece] = p;
    }
}

// A row's settings and its parts put together, by every wave for itself (the same in all lanes)
__device__ __forceinline__ SampleRow sample_row(const SampleArgs& a, int64_t r, const SamplePart& p) {
    const double temp = a.temperatures ? (double)a.temperatures[r] : a.temperature;
    SampleRow x;
    x.top_p = a.top_ps ? (double)a.top_ps[r] : a.top_p;
    x.min_p = a.min_ps ? (double)a.min_ps[r] : a.min_p;
    const int k = a.top_ks ? a.top_ks[r] : a.top_k;
    x.top_k = k > 0 && k < a.vocab ? k : 0;
    x.by_mass = x.top_p < 1.0;
    x.small_k = x.top_k && x.top_k <= SMALL_K;
    x.bin_mass = x.by_mass && !x.small_k;
    x.none = p.nan || p.most == -__builtin_inff();
    x.greedy = !(temp > 0.0);
    x.most = p.most;
    x.at = p.at;
    x.bits = a.bits;
    x.c = 1.44269504088896340736 / temp;
    // the row's own span, so that a flat row has bins as well, but no more than what matters: SPAN logits for a count,
    // SPAN temperatures for a mass alone
    const float unit = x.top_k ? __builtin_fmaxf(1.0f, (float)temp) : (float)temp;
    const float span = __builtin_fminf(p.most - p.least, SPAN * unit);
    x.scale = span > 0.0f && span < __builtin_inff() ? __builtin_fminf((BINS - 1) / span, 1e30f) : 1.0f;
    return x;
}

__device__ __forceinline__ SampleRow sample_row(const SampleArgs& a, int64_t s, int pieces) {
    SamplePart p = NO_PART;
    for (int i = threadIdx.x % WAVE; i < pieces; i += WAVE) p = merge_parts(p, a.parts[s * pieces + i]);
    return sample_row(a, a.row0 + s, wave_part(p));
}

template <typename T>
__global__ __launch_bounds__(PIECE_THREADS) void sample_bins(const SampleArgs a) {
    __shared__ uint64_t mass[BINS];
    __shared__ uint32_t count[BINS];
    const int64_t s = blockIdx.y, r = a.row0 + s;
    const int piece = blockIdx.x, tid = threadIdx.x, end = min(a.tiles, (piece + 1) * a.per);
    const T* const row = reinterpret_cast<const T*>(a.logits) + r * a.stride;
    const SampleRow x = sample_row(a, s, gridDim.x);
    if (x.none || x.greedy || (!x.top_k && !x.by_mass)) return;
    for (int i = tid; i < BINS; i += PIECE_THREADS) {
        mass[i] = 0;
        count[i] = 0;
    }
    __syncthreads();
    for (int t = piece * a.per; t < end; ++t) {
        TileChunks<T, PIECE_THREADS> now;
        now.load(row, t, a.vocab);
        now.each(t, [&](int i, float v) {
            if (i >= a.vocab) return;
            const int b = x.bin(v);
            atomicAdd(&count[b], 1u);
            if (x.bin_mass) atomicAdd((unsigned long long*)&mass[b], (unsigned long long)x.fixed(x.weight(v)));
        });
    }
    __syncthreads();
    for (int i = tid; i < BINS; i += PIECE_THREADS)
        if (count[i]) {
            atomicAdd(&a.count[s * BINS + i], count[i]);
            if (x.bin_mass) atomicAdd((unsigned long long*)&a.mass[s * BINS + i], (unsigned long long)mass[i]);
        }
}

template <int THREADS, typename X>
__device__ __forceinline__ X block_scan(X x, X* part, X& all) {             // inclusive, in thread order
    const int lane = threadIdx.x % WAVE, w = threadIdx.x / WAVE;
#pragma unroll
    for (int d = 1; d < WAVE; d <<= 1) {
        const X o = __shfl_up(x, d, WAVE);
        if (lane >= d) x += o;
    }
    __syncthreads();
    if (lane == WAVE - 1) part[w] = x;
    __syncthreads();
    all = 0;
#pragma unroll
    for (int i = 0; i < THREADS / WAVE; ++i) {
        if (i < w) x += part[i];
        all += part[i];
    }
    return x;
}

// The classes that the cuts fall into: everything below lo is kept (after the other cuts), lo .. hi and k are looked at
// token by token, all else is dropped. before_lo, before_k: mass below those classes; above_k: tokens below k, in_k: in it.
// all: the row's mass
struct SampleCuts {
    int lo, hi, k;
    uint64_t before_lo, before_k, all;
    uint32_t above_k, in_k;
};

// top-p's limit for a mass of `total` (at least half a unit: the first token is kept)
__device__ __forceinline__ double mass_limit(const SampleRow& x, uint64_t total) {
    return __builtin_fmax(x.top_p * (double)total, 0.5);
}

// What random number u leaves before its token of a kept mass of `all` (at least 1): the token's own mass passes it. 1 and more
// leave all but the last unit, so the last kept token; NaN counts as 0. In integers: from 2^53 on a double of all - 1 is all.
__device__ __forceinline__ uint64_t mass_before(float u, uint64_t all) {
    const double part = (double)__builtin_fmaxf(u, 0.0f) * (double)all;
    return u >= 1.0f ? all - 1 : min((uint64_t)part, all - 1);
}

// From the number and (masses) the mass of the tokens in each class; below: without masses all classes down to k are looked at
template <int THREADS>
__device__ __forceinline__ SampleCuts sample_cuts(const SampleRow& x, const uint32_t* count, const uint64_t* mass, bool masses,
                                                  bool below) {
    __shared__ uint64_t part[THREADS / WAVE];
    __shared__ SampleCuts cuts;
    constexpr int N = BINS / THREADS;
    const int tid = threadIdx.x;
    uint32_t c[N], cs = 0, c_all;
    uint64_t m[N], ms = 0, m_all = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        c[i] = count[tid * N + i];
        m[i] = masses ? mass[tid * N + i] : 0;
        cs += c[i];
        ms += m[i];
    }
    if (tid == 0) cuts = SampleCuts{BINS, BINS, BINS, 0, 0, 0, 0, 0};
    const uint32_t c1 = block_scan<THREADS>(cs, reinterpret_cast<uint32_t*>(part), c_all);
    const uint64_t m1 = masses ? block_scan<THREADS>(ms, part, m_all) : 0;
    if (x.top_k) {
        uint32_t cb = c1 - cs;
        uint64_t mb = m1 - ms;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (cb < (uint32_t)x.top_k && cb + c[i] >= (uint32_t)x.top_k) {
                cuts.k = tid * N + i;
                cuts.above_k = cb;
                cuts.in_k = c[i];
                cuts.before_k = mb;
            }
            cb += c[i];
            mb += m[i];
        }
    }
    __syncthreads();
    const SampleCuts now = cuts;
    __syncthreads();
    if (tid == 0) cuts.all = m_all;
    if (!masses) {
        if (tid == 0) {
            cuts.lo = below ? 0 : now.k;
            cuts.hi = now.k;
        }
    } else {
        // the kept mass lies between what is below k and what k adds: so does top-p's cut
        uint64_t mb = m1 - ms;
        const double low = mass_limit(x, x.top_k ? now.before_k : m_all);
        double high = low;
        if (x.top_k) high = mass_limit(x, now.before_k + mass[now.k]);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint64_t me = mb + m[i];
            if ((double)mb < low && !((double)me < low)) {
                cuts.lo = tid * N + i;
                cuts.before_lo = mb;
            }
            if ((double)mb < high && !((double)me < high)) cuts.hi = tid * N + i;
            mb = me;
        }
    }
    __syncthreads();
    return cuts;
}

// Tokens of the list that a workgroup gathers in LDS before it takes places in the row's: a tile may hold TILE of them, and
// a place of its own for each wave's tokens costs a trip to memory and back (102 us at 64 rows of 600 tokens each; 19 so)
constexpr int GATHER = TILE + 1024;

template <typename T>
__global__ __launch_bounds__(PIECE_THREADS) void sample_pick(const SampleArgs a) {
    __shared__ uint2 gather[GATHER];
    __shared__ unsigned long long sum;
    __shared__ uint32_t held, place;
    const int64_t s = blockIdx.y, r = a.row0 + s;
    const int piece = blockIdx.x, tid = threadIdx.x, lane = tid % WAVE;
    const int end = min(a.tiles, (piece + 1) * a.per);
    const T* const row = reinterpret_cast<const T*>(a.logits) + r * a.stride;
    const SampleRow x = sample_row(a, s, gridDim.x);
    if (x.none || x.greedy) return;
    SampleCuts cut{BINS, BINS, BINS, 0, 0, 0, 0, 0};
    if (x.top_k || x.by_mass)
        cut = sample_cuts<PIECE_THREADS>(x, a.count + s * BINS, a.mass + s * BINS, x.bin_mass, x.small_k);
    if (tid == 0) {
        held = 0;
        sum = 0;
    }
    __syncthreads();
    // the list holds all that is kept, and LDS the list: no sums, one flush (64 rows of 152,000 with top-k 50: 34 us, 37 by the
    // loop below; 400 rows 121, 140)
    if (x.small_k && cut.above_k + cut.in_k <= GATHER) {
        for (int t = piece * a.per; t < end; ++t) {
            TileChunks<T, PIECE_THREADS> now;
            now.load(row, t, a.vocab);
            now.each(t, [&](int i, float v) {
                if (i < a.vocab && x.bin(v) <= cut.k) gather[atomicAdd(&held, 1u)] = uint2{(uint32_t)i, order_key(v)};
            });
        }
        __syncthreads();
        const uint32_t n = held;
        if (n == 0) return;
        if (tid == 0) place = atomicAdd(&a.length[s], n);
        __syncthreads();
        for (uint32_t i = tid; i < n; i += PIECE_THREADS)
            if (place + i < LIST) a.list[s * LIST + place + i] = gather[i];
        return;
    }
    for (int t = piece * a.per; t < end; ++t) {
        uint64_t mine = 0;
        TileChunks<T, PIECE_THREADS> now;
        now.load(row, t, a.vocab);
        now.each(t, [&](int i, float v) {
            if (i >= a.vocab) return;
            const int b = x.bin(v);
            if (b < cut.lo) {
                const double w = x.weight(v);
                if (w >= x.min_p || i == x.at) mine += x.fixed(w);
            } else if (b <= cut.hi || b == cut.k) {
                gather[atomicAdd(&held, 1u)] = uint2{(uint32_t)i, order_key(v)};
            }
        });
        if (cut.lo > 0) {
#pragma unroll
            for (int m = 32; m >= 1; m >>= 1) mine += __shfl_xor(mine, m, WAVE);
            if (lane == 0 && mine) atomicAdd(&sum, (unsigned long long)mine);
        }
        __syncthreads();
        const uint32_t n = held;
        const bool flush = n > 0 && (n > GATHER - TILE || t + 1 == end);
        __syncthreads();
        if (tid == 0) {
            a.sums[s * a.tiles + t] = sum;
            sum = 0;
            if (flush) {
                place = atomicAdd(&a.length[s], n);
                held = 0;
            }
        }
        __syncthreads();
        if (flush) {
            for (uint32_t i = tid; i < n; i += PIECE_THREADS)
                if (place + i < LIST) a.list[s * LIST + place + i] = gather[i];
            __syncthreads();
        }
    }
}

constexpr int TOKEN_THREADS = 256, MAX_TILES = (1 << 24) / TILE;

// The order as one number, larger first: the key, then the smaller index
__device__ __forceinline__ uint64_t order_of(uint32_t key, uint32_t index) { return ((uint64_t)key << 32) | (uint32_t)~index; }

// The tokens of L [n], by their orders, sorted, the largest first (bitonic; the places behind them up to the power of two
// hold 0, below every token). Up to a distance of 64 a wave's pairs lie in 128 places of its own, and its LDS operations
// stay in order: no barrier.
__device__ __forceinline__ void sort_orders(uint64_t* L, int size) {
    bool apart = true;
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            if (apart || j > 64) __syncthreads();
            asm volatile("" ::: "memory");
            apart = j > 64;
            for (int i = threadIdx.x; i < size / 2; i += TOKEN_THREADS) {
                const int p = ((i & ~(j - 1)) << 1) | (i & (j - 1)), q = p | j;
                const uint64_t u = L[p], v = L[q];
                if ((u < v) == ((p & k) == 0)) {
                    L[p] = v;
                    L[q] = u;
                }
            }
        }
    __syncthreads();
}

constexpr int BORDER = 1024;                             // tokens next to the cuts that are sorted by themselves

// LDS of the kernels that draw from a list
struct DrawSpace {
    unsigned long long mass[BINS];
    uint32_t count[BINS];
    uint64_t border[BORDER];
    uint64_t part[TOKEN_THREADS / WAVE];
    uint64_t passed;
    int at;
};

// top-k's and top-p's cuts within L, `m` tokens sorted (largest first) that hold all of the classes that `cut` looks at, by
// classes of width 1 / scale; masses: cut knows the masses below its classes (else L starts at the row's first token).
// add(order, w, mass) for every token that is kept (weights: where they are
// asked for). The order of the last one that is kept.
template <typename Add>
__device__ __forceinline__ uint64_t cut_sorted(const SampleRow& x, const uint64_t* L, int m, const SampleCuts& cut, float scale,
                                               bool masses, bool weights, DrawSpace& sp, Add&& add) {
    const int tid = threadIdx.x;
    const auto logit = [](uint64_t order) { return key_logit((uint32_t)(order >> 32)); };
    // of class k, the first top_k - above_k tokens
    int k_first = m;
    if (x.top_k) {
        if (tid == 0) sp.at = m;
        __syncthreads();
        for (int i = tid; i < m; i += TOKEN_THREADS)
            if (x.bin(logit(L[i]), scale) == cut.k && (i == 0 || x.bin(logit(L[i - 1]), scale) != cut.k)) sp.at = i;
        __syncthreads();
        k_first = sp.at;
    }
    const int keep = x.top_k ? k_first + (x.top_k - (int)cut.above_k) : m;
    double limit = 0.0;
    if (x.by_mass) {
        uint64_t total = cut.all;
        if (x.top_k) {                                       // what top-k keeps: below its class, and its own tokens
            uint64_t sum = 0;
            for (int i = (masses ? k_first : 0) + tid; i < keep; i += TOKEN_THREADS) sum += x.fixed(x.weight(logit(L[i])));
            block_scan<TOKEN_THREADS>(sum, sp.part, total);
            total += masses ? cut.before_k : 0;
        }
        limit = mass_limit(x, total);
    }
    uint64_t before = cut.before_lo;
    int kept = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < keep; i0 += TOKEN_THREADS) {
        const int i = i0 + tid;
        double w = 0.0;
        uint64_t mine = 0, all = 0;
        bool in = i < keep;
        if (in && (x.by_mass || weights)) {
            w = x.weight(logit(L[i]));
            mine = x.fixed(w);
        }
        if (x.by_mass) {
            const uint64_t run = before + block_scan<TOKEN_THREADS>(mine, sp.part, all) - mine;
            before += all;
            in = in && (double)run < limit;
        }
        if (in) add(L[i], w, mine);
        const int now = __syncthreads_count(in);
        kept += now;
        if (now < TOKEN_THREADS) break;
    }
    const uint64_t least = kept > 0 ? L[kept - 1] : ~0ull;
    __syncthreads();
    return least;
}

// draw_from_list's answer for n <= WAVE (what top-k 50 leaves of a row, as a rule): a token per lane, its place in the order
// and the mass before it, there and in the vocabulary, counted over the list, a part of it per wave (one row of
// 152,000: this kernel 13 us by draw_from_list, 7 so; lists of 150 tokens in 256 lanes took 17 and stay there)
__device__ __forceinline__ void draw_counted(const SampleArgs& a, int64_t r, const SampleRow& x, const uint64_t* list, int n,
                                             DrawSpace& sp) {
    constexpr int WAVES = TOKEN_THREADS / WAVE, PART = WAVE / WAVES;
    static_assert(BINS >= (WAVES + 1) * WAVE, "masses and parts");
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    const uint64_t mine = lane < n ? list[lane] : 0;
    const uint32_t index = ~(uint32_t)mine;
    const double w = lane < n ? x.weight(key_logit((uint32_t)(mine >> 32))) : 0.0;
    uint64_t mass = x.fixed(w);
    bool in = lane < n;
    // the sum of term(token, its mass) over the list, the same in all waves
    const auto count = [&](auto&& term) -> uint64_t {
        __syncthreads();
        if (wave == 0) sp.mass[lane] = mass;
        __syncthreads();
        uint64_t part = 0;
#pragma unroll
        for (int j = wave * PART; j < wave * PART + PART; ++j)
            if (j < n) part += term(list[j], (uint64_t)sp.mass[j]);
        sp.mass[(wave + 1) * WAVE + lane] = part;
        __syncthreads();
        uint64_t sum = 0;
#pragma unroll
        for (int i = 1; i <= WAVES; ++i) sum += sp.mass[i * WAVE + lane];
        return sum;
    };
    const auto over_lanes = [](uint64_t v) {
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, WAVE);
        return v;
    };
    if (x.top_k) {
        const uint64_t place = count([&](uint64_t o, uint64_t) -> uint64_t { return o > mine; });
        in = in && (int)place < x.top_k;
    }
    if (x.by_mass) {
        const uint64_t before = count([&](uint64_t o, uint64_t m) { return o > mine ? m : 0; });
        const double limit = mass_limit(x, over_lanes(in ? mass : 0));
        in = in && (double)before < limit;
    }
    if (!in || !(w >= x.min_p || (int)index == x.at)) mass = 0;
    const uint64_t run = count([&](uint64_t o, uint64_t m) { return (uint32_t)o > (uint32_t)mine ? m : 0; });   // (the index's complement)
    const uint64_t all = over_lanes(mass);
    const uint64_t want = mass_before(a.uniforms[r], all);
    if (wave == 0 && mass && run <= want && run + mass > want) a.out[r] = index;
}

// The token of row r from a list [n, filled up with 0 to a power of two] that holds all that may be kept. The list's tokens are
// put into BINS classes (`fine` of them per logit), which leave a handful to sort next to the cuts; then the running sum
// in the vocabulary's order, 10 bits of the tokens' indexes a pass.
__device__ __forceinline__ void draw_from_list(const SampleArgs& a, int64_t r, const SampleRow& x, uint64_t* list, int n, float fine,
                                               DrawSpace& sp) {
    const int tid = threadIdx.x;
    const auto logit = [](uint64_t order) { return key_logit((uint32_t)(order >> 32)); };
    int lo = BINS;                                           // all is kept
    uint64_t least = ~0ull;
    if (x.top_k || x.by_mass) {
        for (int i = tid; i < BINS; i += TOKEN_THREADS) {
            sp.mass[i] = 0;
            sp.count[i] = 0;
        }
        if (tid == 0) sp.at = 0;
        __syncthreads();
        for (int i = tid; i < n; i += TOKEN_THREADS) {
            const float v = logit(list[i]);
            const int b = x.bin(v, fine);
            atomicAdd(&sp.count[b], 1u);
            if (x.by_mass) atomicAdd(&sp.mass[b], (unsigned long long)x.fixed(x.weight(v)));
        }
        __syncthreads();
        SampleCuts cut = sample_cuts<TOKEN_THREADS>(x, sp.count, reinterpret_cast<uint64_t*>(sp.mass), x.by_mass, false);
        for (int i = tid; i < n; i += TOKEN_THREADS) {
            const int b = x.bin(logit(list[i]), fine);
            if (b >= cut.lo && (b <= cut.hi || b == cut.k)) {
                const int at = atomicAdd(&sp.at, 1);
                if (at < BORDER) sp.border[at] = list[i];
            }
        }
        __syncthreads();
        int m = sp.at;
        __syncthreads();
        uint64_t* L = sp.border;
        lo = cut.lo;
        if (m > BORDER) {                                    // (equal logits by the thousands: the list as a whole)
            L = list;
            m = n;
            lo = 0;
            cut.before_lo = 0;
        }
        int size = 2;
        while (size < m) size <<= 1;
        if (L != list)
            for (int i = m + tid; i < size; i += TOKEN_THREADS) L[i] = 0;
        sort_orders(L, size);
        least = cut_sorted(x, L, m, cut, fine, x.by_mass, false, sp, [](uint64_t, double, uint64_t) {});
    }
    const auto mass_of = [&](uint64_t order) -> uint64_t {
        const float v = logit(order);
        if (!(x.bin(v, fine) < lo || order >= least)) return 0;
        const double w = x.weight(v);
        return w >= x.min_p || (int)~(uint32_t)order == x.at ? x.fixed(w) : 0;
    };
    uint64_t want = 0, passed = 0;
    uint32_t prefix = 0;
    constexpr int BITS = 10, N = BINS / TOKEN_THREADS;
    static_assert(BINS == 1 << BITS, "a bin for each value of the digit");
#pragma unroll 1
    for (int top = a.index_bits; top > 0; top -= BITS) {
        const int shift = top > BITS ? top - BITS : 0;
        for (int i = tid; i < BINS; i += TOKEN_THREADS) sp.mass[i] = 0;
        if (tid == 0) sp.at = 0;
        __syncthreads();
        for (int i = tid; i < n; i += TOKEN_THREADS) {
            const uint32_t at = ~(uint32_t)list[i];
            if ((at >> top) != prefix) continue;
            const uint64_t v = mass_of(list[i]);
            if (v) atomicAdd(&sp.mass[(at >> shift) & ((1u << (top - shift)) - 1)], (unsigned long long)v);
        }
        __syncthreads();
        uint64_t v[N], sum = 0, all;
#pragma unroll
        for (int i = 0; i < N; ++i) sum += v[i] = sp.mass[tid * N + i];
        uint64_t at = passed + block_scan<TOKEN_THREADS>(sum, sp.part, all) - sum;
        if (top == a.index_bits) want = mass_before(a.uniforms[r], all);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (v[i] && at <= want && at + v[i] > want) {
                sp.at = tid * N + i;
                sp.passed = at;
            }
            at += v[i];
        }
        __syncthreads();
        prefix = (prefix << (top - shift)) | (uint32_t)sp.at;
        passed = sp.passed;
        __syncthreads();
    }
    if (tid == 0) a.out[r] = prefix;
}

// grid rows: vocabularies of one tile, the row in LDS as its own list (1 - 64 rows: 6 - 22 us, four launches 18 - 35;
// 1,024 rows 11 - 44, four launches 52 - 95)
template <typename T>
__global__ __launch_bounds__(TOKEN_THREADS) void sample_small(const SampleArgs a) {
    __shared__ uint64_t list[TILE];
    __shared__ DrawSpace sp;
    __shared__ SamplePart ws[TOKEN_THREADS / WAVE];
    const int64_t r = a.row0 + blockIdx.x;
    const int tid = threadIdx.x;
    const T* const row = reinterpret_cast<const T*>(a.logits) + r * a.stride;
    SamplePart p = NO_PART;
    int size = 2;
    while (size < a.vocab) size <<= 1;
    TileChunks<T, TOKEN_THREADS> now;
    now.load(row, 0, a.vocab);
    now.each(0, [&](int i, float x) {
        merge_logit(p, i, x);
        if (i < size) list[i] = i < a.vocab ? order_of(order_key(x), i) : 0;
    });
    p = wave_part(p);
    if (tid % WAVE == 0) ws[tid / WAVE] = p;
    __syncthreads();
    p = ws[0];
    for (int w = 1; w < TOKEN_THREADS / WAVE; ++w) p = merge_parts(p, ws[w]);
    const SampleRow x = sample_row(a, r, p);
    if (x.none || x.greedy) {
        if (tid == 0) a.out[r] = x.none ? -1 : x.at;
        return;
    }
    draw_from_list(a, r, x, list, a.vocab, x.scale, sp);
}

// grid rows. What is kept of the row: tokens of classes below `lo`, and those of order `least` or above; w >= min_p.
// Where top-k bounds the list (small_k) the token is drawn from the list alone. Else the list is the tokens of the cuts'
// classes: sorted, added to the tiles' sums, and the token found in its tile.
template <typename T>
__global__ __launch_bounds__(TOKEN_THREADS) void sample_token(const SampleArgs a, int pieces) {
    __shared__ uint64_t list[LIST];
    __shared__ unsigned long long sums[MAX_TILES];
    __shared__ DrawSpace sp;
    uint64_t* const part = sp.part;
    const int64_t s = blockIdx.x, r = a.row0 + s;
    const int tid = threadIdx.x;
    const uint32_t length = a.length[s];
    const SampleRow x = sample_row(a, s, pieces);
    if (x.none || x.greedy) {
        if (tid == 0) a.out[r] = x.none ? -1 : x.at;
        return;
    }
    const T* const row = reinterpret_cast<const T*>(a.logits) + r * a.stride;
    int lo = BINS;                                       // all is kept
    uint64_t least = ~0ull;
    const int n = x.top_k || x.by_mass ? (int)min(length, 0x7fffffffu) : 0;
    if (x.top_k || x.by_mass) {
        int size = 2;
        if (n <= LIST) {
            while (size < n) size <<= 1;
            for (int i = tid; i < size; i += TOKEN_THREADS) {
                const uint2 v = i < n ? a.list[s * LIST + i] : uint2{0, 0};
                list[i] = i < n ? order_of(v.y, v.x) : 0;
            }
        }
        if (x.small_k && n <= WAVE) {
            __syncthreads();
            draw_counted(a, r, x, list, n, sp);
            return;
        }
        const SampleCuts cut = sample_cuts<TOKEN_THREADS>(x, a.count + s * BINS, a.mass + s * BINS, x.bin_mass, x.small_k);
        if (x.small_k && n <= LIST) {
            draw_from_list(a, r, x, list, n, x.scale * ((float)BINS / (float)(cut.k + 1)), sp);
            return;
        }
        lo = cut.lo;
        for (int i = tid; i < a.tiles; i += TOKEN_THREADS) sums[i] = a.sums[s * a.tiles + i];
        if (n <= LIST) {
            sort_orders(list, size);
            least = cut_sorted(x, list, n, cut, x.scale, x.bin_mass, true, sp, [&](uint64_t order, double w, uint64_t mass) {
                const uint32_t at = ~(uint32_t)order;
                if (w >= x.min_p || (int)at == x.at) atomicAdd(&sums[at / TILE], (unsigned long long)mass);
            });
        } else {
            // the token that ends what is kept, by a radix search over the row's orders: 9 bits a pass, from the top,
            // two bins to a thread
            constexpr int SEARCH = 9;
            static_assert((1 << SEARCH) == 2 * TOKEN_THREADS, "two bins to a thread");
            uint64_t* const mass = list;
            uint32_t* const count = reinterpret_cast<uint32_t*>(list + (1 << SEARCH));
            const auto each = [&](auto&& fn) {
                for (int i = tid; i < a.vocab; i += TOKEN_THREADS) fn(i, to_f32(row[i]));
            };
            // of the tokens of order `floor` and above: the `want`-th, or the last with less than `limit` mass before it;
            // kept: the mass up to it
            const auto search = [&](bool by_mass, uint64_t floor, uint32_t want, double limit, uint64_t& kept) -> uint64_t {
                uint64_t prefix = 0, above_mass = 0, above = 0;
                for (int top = 64; top > 0;) {
                    const int width = min(SEARCH, top), shift = top - width, nb = 1 << width;
                    __syncthreads();
                    for (int i = tid; i < (1 << SEARCH); i += TOKEN_THREADS) {
                        mass[i] = 0;
                        count[i] = 0;
                    }
                    __syncthreads();
                    each([&](int i, float v) {
                        const uint64_t o = order_of(order_key(v), i);
                        if (o < floor || (top < 64 && (o >> top) != prefix)) return;
                        const int b = (int)((o >> shift) & (uint64_t)(nb - 1));
                        atomicAdd(&count[b], 1u);
                        atomicAdd((unsigned long long*)&mass[b], (unsigned long long)x.fixed(x.weight(v)));
                    });
                    __syncthreads();
                    const int b1 = nb - 1 - 2 * tid;                       // this thread's bins, the upper first
                    uint64_t c[2], m[2], unused;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        c[j] = b1 - j >= 0 ? count[b1 - j] : 0;
                        m[j] = b1 - j >= 0 ? mass[b1 - j] : 0;
                    }
                    uint64_t cb = above + block_scan<TOKEN_THREADS>(c[0] + c[1], part, unused) - c[0] - c[1];
                    uint64_t mb = above_mass + block_scan<TOKEN_THREADS>(m[0] + m[1], part, unused) - m[0] - m[1];
                    __syncthreads();
                    if (tid == 0) sp.at = 0;
                    __syncthreads();
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const bool here = by_mass ? (double)mb < limit && !((double)(mb + m[j]) < limit)
                                                  : cb < want && cb + c[j] >= want;
                        if (here) {
                            sp.at = b1 - j;
                            sp.passed = mb;
                            part[0] = cb;
                        }
                        cb += c[j];
                        mb += m[j];
                    }
                    __syncthreads();
                    prefix = (prefix << width) | (uint64_t)sp.at;
                    above_mass = sp.passed;
                    above = part[0];
                    kept = above_mass + mass[sp.at];
                    top = shift;
                }
                __syncthreads();
                return prefix;
            };
            uint64_t total = 0;
            least = 0;
            if (x.top_k) least = search(false, 0, (uint32_t)x.top_k, 0.0, total);
            if (x.by_mass) {
                if (!x.top_k) total = cut.all;
                least = search(true, least, 0, mass_limit(x, total), total);
            }
            each([&](int i, float v) {
                if (x.bin(v) < lo || order_of(order_key(v), i) < least) return;
                const double w = x.weight(v);
                if (w >= x.min_p || i == x.at) atomicAdd(&sums[i / TILE], (unsigned long long)x.fixed(w));
            });
        }
    }
    __syncthreads();
    if (!x.top_k && !x.by_mass)
        for (int i = tid; i < a.tiles; i += TOKEN_THREADS) sums[i] = a.sums[s * a.tiles + i];
    __syncthreads();
    // the tile that the target falls into
    uint64_t run_mass = 0, all = 0;
    {
        uint64_t v = 0;
        for (int t = tid; t < a.tiles; t += TOKEN_THREADS) v += sums[t];
        block_scan<TOKEN_THREADS>(v, part, all);
    }
    const uint64_t want = mass_before(a.uniforms[r], all);
    if (tid == 0) sp.at = 0;
    for (int t0 = 0; t0 < a.tiles; t0 += TOKEN_THREADS) {
        uint64_t here;
        const uint64_t v = t0 + tid < a.tiles ? (uint64_t)sums[t0 + tid] : 0;
        const uint64_t end = block_scan<TOKEN_THREADS>(v, part, here) + run_mass;
        if (v && end - v <= want && end > want) {
            sp.at = t0 + tid;
            sp.passed = end - v;
        }
        run_mass += here;
    }
    __syncthreads();
    const int tile = sp.at;
    run_mass = sp.passed;
    __syncthreads();
    // each thread a run of the tile's tokens, from LDS (a run and a bit apart, so that the threads read different banks)
    constexpr int E = TILE / TOKEN_THREADS, RUN = E + 1;
    float* const logit = reinterpret_cast<float*>(list);
    {
        TileChunks<T, TOKEN_THREADS> c;
        c.load(row, tile, a.vocab);
        c.each(tile, [&](int i, float v) { logit[(i - tile * TILE) / E * RUN + (i - tile * TILE) % E] = v; });
    }
    __syncthreads();
    uint64_t mass[E], mine = 0, unused;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = tile * TILE + tid * E + e;
        const float v = logit[tid * RUN + e];
        const double w = x.weight(v);
        const bool in = i < a.vocab && (x.bin(v) < lo || order_of(order_key(v), i) >= least) && (w >= x.min_p || i == x.at);
        mine += mass[e] = in ? x.fixed(w) : 0;
    }
    uint64_t before = run_mass + block_scan<TOKEN_THREADS>(mine, part, unused) - mine;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (mass[e] && before <= want && before + mass[e] > want) a.out[r] = tile * TILE + tid * E + e;
        before += mass[e];
    }
}

}  // namespace kush

using namespace kush;

extern "C" int kush_block_table(const int32_t* req_to_token, int64_t map_row_stride, int64_t map_rows, int64_t map_cols,
                                const void* req, int32_t wide_req, const void* seq_lens, int32_t wide_lens,
                                int64_t n_reqs, int64_t pages, int32_t* table, int64_t table_row_stride, int32_t* lens_out,
                                int32_t* slots_out, void* stream) {
    if (n_reqs < 0 || n_reqs > 0x7fffffff || pages < 0 || pages > 65535ll * 256 || map_rows < 0 || map_cols < 0 ||
        table_row_stride < pages)
        return kush_fail(-2, "kush_block_table: bad n_reqs %lld / pages %lld / table_row_stride %lld", (long long)n_reqs,
                         (long long)pages, (long long)table_row_stride);
    if (n_reqs == 0) return 0;
    block_table_kernel<<<dim3((unsigned)n_reqs, (unsigned)std::max<int64_t>(1, (pages + 255) / 256)), dim3(256), 0,
                         (hipStream_t)stream>>>(req_to_token, map_row_stride, map_rows, map_cols, req, wide_req, seq_lens,
                                                wide_lens, pages, table, table_row_stride, lens_out, slots_out);
    return kush_check_launch("kush_block_table");
}

extern "C" int kush_step_maps(const int32_t* new_tokens, const int32_t* history, const int32_t* slots,
                              const int32_t* block_table, int64_t bt_row_stride, int64_t bt_cols, int64_t n_reqs,
                              int32_t window, int32_t sinks, int64_t jobs, int64_t pages, int64_t tails, int64_t tokens,
                              int32_t* q_start, int32_t* key_start, int32_t* seq_lens, int32_t* job_seq, int32_t* job_page,
                              int32_t* page_blk, int32_t* page_dst, int32_t* tail_blk, int32_t* tail_info,
                              int32_t* new_dst, int64_t* slot_map, void* stream) {
    if (n_reqs < 0 || n_reqs > 65536 || window < 0 || sinks < 0 || jobs < 0 || pages < 0 || tails < 0 || tokens < 0 ||
        jobs > 0x7fffffff || pages > 0x7fffffff || tails > 0x7fffffff || tokens > 0x7fffffff)
        return kush_fail(-2, "kush_step_maps: bad n_reqs %lld (at most 65536) / window %d / sinks %d / sizes %lld, %lld, %lld, %lld",
                         (long long)n_reqs, window, sinks, (long long)jobs, (long long)pages, (long long)tails,
                         (long long)tokens);
    if (n_reqs == 0) return 0;
    const MapArgs a{new_tokens, history, slots,    block_table, bt_row_stride, bt_cols,  (int)n_reqs, window,
                    sinks,      jobs,    pages,    tails,       tokens,        q_start,  key_start,   seq_lens,
                    job_seq,    job_page, page_blk, page_dst,   tail_blk,      tail_info, new_dst,    slot_map};
    const int64_t parts = std::min<int64_t>(64, std::max<int64_t>(1, (tokens + pages) / (n_reqs * 1024)));
    step_maps_kernel<<<dim3((unsigned)n_reqs, (unsigned)parts), dim3(256), 0, (hipStream_t)stream>>>(a);
    return kush_check_launch("kush_step_maps");
}

// Tiles of a row to a workgroup, for about three workgroups per CU, and 4 at most (64 rows of 152,000: 4 49.8 us, 7 60.9, 2
// 53.6, 1 67.5; 400 rows with top-p: 4 325 us, 20 413)
static int64_t tiles_each(int64_t rows, int64_t tiles) { return std::min<int64_t>({tiles, (rows * tiles + 767) / 768, 4}); }

constexpr int64_t SAMPLE_ROWS = 1024;            // rows of one launch; more go in turn, over the same scratch

// Scratch of a launch, by 16-byte aligned pieces
struct SampleScratch {
    int64_t parts, mass, sums, count, length, list, bytes;
    SampleScratch(int64_t rows, int64_t vocab) {
        const int64_t tiles = (vocab + TILE - 1) / TILE;
        int64_t at = 0;
        const auto piece = [&](int64_t n) {
            const int64_t p = at;
            at = (at + n + 15) & ~int64_t(15);
            return p;
        };
        parts = piece(rows * tiles * (int64_t)sizeof(SamplePart));
        mass = piece(rows * BINS * 8);
        sums = piece(rows * tiles * 8);
        count = piece(rows * BINS * 4);
        length = piece(rows * 4);
        list = piece(rows * LIST * 8);
        bytes = at;
    }
};

extern "C" int64_t kush_sample_scratch(int64_t rows, int64_t vocab) {
    if (rows < 0 || vocab < 1 || vocab > (1 << 24)) return 0;
    return SampleScratch(std::min(rows, SAMPLE_ROWS), vocab).bytes;
}

extern "C" int kush_sample(int dtype, const void* logits, int64_t row_stride, int64_t rows, int64_t vocab,
                           const float* uniforms, double temperature, const float* temperatures, int32_t top_k,
                           const int32_t* top_ks, double top_p, const float* top_ps, double min_p, const float* min_ps,
                           int64_t* out, void* scratch, int64_t scratch_bytes, void* stream) {
    if (rows < 0 || rows > 0x7fffffff || vocab < 1 || vocab > (1 << 24) || row_stride < 0)
        return kush_fail(-2, "kush_sample: bad rows %lld / vocab %lld (1 .. 2^24) / row_stride %lld", (long long)rows,
                         (long long)vocab, (long long)row_stride);
    if (dtype < 0 || dtype > 2) return kush_fail(-1, "kush_sample: unsupported dtype code %d (0 fp32, 1 fp16, 2 bf16)", dtype);
    if (rows == 0) return 0;
    const SampleScratch at(std::min(rows, SAMPLE_ROWS), vocab);
    if (scratch == nullptr || ((uintptr_t)scratch & 15) || scratch_bytes < at.bytes)
        return kush_fail(-2, "kush_sample: needs %lld bytes of 16-byte aligned scratch (kush_sample_scratch)", (long long)at.bytes);
    int log = 0;
    while ((1ll << log) < vocab) ++log;
    uint8_t* const base = (uint8_t*)scratch;
    SampleArgs a{logits,       row_stride, (int)vocab, std::min(50, 63 - log), (int)((vocab + TILE - 1) / TILE),
                 0,            uniforms,   temperature, top_p,                 min_p,
                 top_k,        temperatures, top_ps,   min_ps,                 top_ks,
                 out,          (SamplePart*)(base + at.parts),                 (uint64_t*)(base + at.mass),
                 (uint64_t*)(base + at.sums), (uint32_t*)(base + at.count),    (uint32_t*)(base + at.length),
                 (uint2*)(base + at.list),    std::max(1, log),                0};
    const bool cuts = top_ks || top_ps || top_k > 0 || top_p < 1.0;
    hipStream_t st = (hipStream_t)stream;
    const auto go = [&](auto in) {
        using T = decltype(in);
        for (; a.row0 < rows; a.row0 += SAMPLE_ROWS) {
            const int64_t n = std::min(SAMPLE_ROWS, rows - a.row0);
            if (vocab <= TILE) {
                sample_small<T><<<dim3((unsigned)n), dim3(TOKEN_THREADS), 0, st>>>(a);
                continue;
            }
            a.per = (int)tiles_each(n, a.tiles);
            const int pieces = (a.tiles + a.per - 1) / a.per;
            const dim3 grid((unsigned)pieces, (unsigned)n);
            sample_max<T><<<grid, dim3(PIECE_THREADS), 0, st>>>(a);
            if (cuts) sample_bins<T><<<grid, dim3(PIECE_THREADS), 0, st>>>(a);
            sample_pick<T><<<grid, dim3(PIECE_THREADS), 0, st>>>(a);
            sample_token<T><<<dim3((unsigned)n), dim3(TOKEN_THREADS), 0, st>>>(a, pieces);
        }
        return kush_check_launch("kush_sample");
    };
    return dtype == 0 ? go(float{}) : (dtype == 1 ? go(_Float16{}) : go(bf16_t{}));
}
