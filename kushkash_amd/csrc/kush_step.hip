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

// What one request adds to each array
struct MapCounts {
    int tokens, keys, pages, jobs, tails;
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
    return MapCounts{t, h - PAGE * gap + t, h / PAGE - gap, t > 0 ? (h + t - 1) / PAGE - h / PAGE + 1 : 0, h % PAGE != 0};
}

__device__ __forceinline__ int wave_sum(int x) {
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
    const int full = h / PAGE, gap = full - mine.pages, kept = h - PAGE * gap;
    const int first = a.sinks / PAGE + (a.sinks % PAGE != 0);
    const int32_t* const table = a.table + (int64_t)r * a.stride;
    const auto block = [&](int p) { return p < a.cols ? table[p] : 0; };
    if (tid == 0 && blockIdx.y == 0) {
        a.q_start[r] = before.tokens;
        a.key_start[r] = before.keys;
        a.seq_lens[r] = h + t;
        if (r == a.n - 1) {
            a.q_start[a.n] = before.tokens + mine.tokens;
            a.key_start[a.n] = before.keys + mine.keys;
        }
        if (mine.tails && before.tails < a.tails) {
            a.tail_blk[before.tails] = block(full);
            int32_t* const info = a.tail_info + 3 * (int64_t)before.tails;
            info[0] = before.keys + PAGE * mine.pages;
            info[1] = h % PAGE;
            info[2] = a.slots[r];
        }
    }
    const int i0 = (int)blockIdx.y * 256 + tid, step = (int)gridDim.y * 256;
    for (int i = i0; i < mine.jobs && before.jobs + i < a.jobs; i += step) {
        a.job_seq[before.jobs + i] = r;
        a.job_page[before.jobs + i] = full + i;
    }
    for (int i = i0; i < mine.pages && before.pages + i < a.pages; i += step) {
        a.page_blk[before.pages + i] = block(i < first ? i : i + gap);
        a.page_dst[before.pages + i] = before.keys + PAGE * i;
    }
    for (int i = i0; i < t && before.tokens + i < a.tokens; i += step) {
        const int at = h + i;
        a.new_dst[before.tokens + i] = before.keys + kept + i;
        a.slot_map[before.tokens + i] = (int64_t)block(at / PAGE) * PAGE + at % PAGE;
    }
}

// ------------------------------------------------------------------ sampling
struct SampleArgs {
    const void* logits;
    int64_t stride;
    int vocab, bits;                 // weights are held as multiples of 2^-bits
    const float* uniforms;
    double temperature, top_p, min_p;
    int top_k;
    const float *temperatures, *top_ps, *min_ps;
    const int32_t* top_ks;
    int64_t* out;
};

constexpr int SAMPLE_THREADS = 1024, SAMPLE_WAVES = SAMPLE_THREADS / WAVE;
constexpr int BINS = 2048;           // of a radix pass: 11, 11 and 10 bits of a logit's order

// logits in an order of their own: larger logit, larger key; -0 and 0 alike
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

// E elements of T from p, whatever its alignment
template <typename T, int E>
__device__ __forceinline__ void load_elems(const T* p, float (&x)[E]) {
    T v[E];
    __builtin_memcpy(v, p, sizeof(v));
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = to_f32(v[e]);
}

// What a row's tokens are kept by: those above key, and of those at key the first `ties` by index
struct Cut {
    uint32_t key;
    int ties;
};

template <typename T>
struct Sampler {
    static constexpr int E = 16 / sizeof(T), TILE = SAMPLE_THREADS * E;
    const T* row;
    int vocab, tid, lane, w;
    float most;
    double inv_t;
    int bits;

    // fn(index, value) of every logit, index ascending within a thread; a wave's lanes take adjacent runs of E
    template <typename Fn>
    __device__ __forceinline__ void each(Fn&& fn) const {
        for (int i0 = tid * E; i0 < vocab; i0 += TILE) {
            float x[E];
            if (i0 + E <= vocab) {
                load_elems<T, E>(row + i0, x);
#pragma unroll
                for (int e = 0; e < E; ++e) fn(i0 + e, x[e]);
            } else {
                for (int i = i0; i < vocab; ++i) fn(i, to_f32(row[i]));
            }
        }
    }
    // w in multiples of 2^-bits; at least 1 of them where w is above 0
    __device__ __forceinline__ uint64_t weight(float x, double& wd) const {
        wd = x == most ? 1.0 : exp(((double)x - (double)most) * inv_t);
        return wd > 0.0 ? max((uint64_t)1, (uint64_t)(wd * (double)(1ull << bits) + 0.5)) : 0;
    }
};

template <typename X>
__device__ __forceinline__ X block_sum(X x, X* part, int lane, int w) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) x += __shfl_xor(x, m, WAVE);
    __syncthreads();
    if (lane == 0) part[w] = x;
    __syncthreads();
    x = part[0];
    for (int i = 1; i < SAMPLE_WAVES; ++i) x += part[i];
    return x;
}

// grid rows, block 1024: one row. The weights are held as 64-bit multiples of 2^-bits (bits such that their sum over the
// vocabulary fits): sums are exact, so no order of atomics or lanes changes a token, and each weight is off by 2^-bits-1,
// far below what a 24-bit random number resolves.
template <typename T>
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_kernel(const SampleArgs a) {
    __shared__ uint64_t mass[BINS];
    __shared__ uint32_t count[BINS];
    __shared__ uint64_t part[SAMPLE_WAVES];
    __shared__ uint64_t found_mass;
    __shared__ int found_bin, found_count;
    Sampler<T> s;
    const int64_t r = blockIdx.x;
    s.row = reinterpret_cast<const T*>(a.logits) + r * a.stride;
    s.vocab = a.vocab;
    s.tid = threadIdx.x;
    s.lane = s.tid % WAVE;
    s.w = s.tid / WAVE;
    s.bits = a.bits;
    const double temp = a.temperatures ? (double)a.temperatures[r] : a.temperature;
    const double top_p = a.top_ps ? (double)a.top_ps[r] : a.top_p, min_p = a.min_ps ? (double)a.min_ps[r] : a.min_p;
    const int top_k = a.top_ks ? a.top_ks[r] : a.top_k;

    // the largest logit and its first index; NaN
    float mx = -__builtin_inff();
    int at = 0x7fffffff, bad = 0;
    s.each([&](int i, float x) {
        bad |= x != x;
        if (x > mx) {
            mx = x;
            at = i;
        }
    });
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        const float ox = __shfl_xor(mx, m, WAVE);
        const int oi = __shfl_xor(at, m, WAVE);
        bad |= __shfl_xor(bad, m, WAVE);
        if (ox > mx || (ox == mx && oi < at)) {
            mx = ox;
            at = oi;
        }
    }
    if (s.lane == 0) {
        mass[s.w] = ((uint64_t)order_key(mx) << 32) | (uint32_t)~at;
        count[s.w] = bad;
    }
    __syncthreads();
    uint64_t best = 0;
    for (int i = 0; i < SAMPLE_WAVES; ++i) {
        best = max(best, mass[i]);
        bad |= count[i];
    }
    at = (int)~(uint32_t)best;
    const uint32_t top_key = (uint32_t)(best >> 32);
    s.most = __uint_as_float(top_key ^ ((top_key >> 31) ? 0x80000000u : 0xFFFFFFFFu));
    __syncthreads();
    if (bad || s.most == -__builtin_inff()) {
        if (s.tid == 0) a.out[r] = -1;
        return;
    }
    if (!(temp > 0.0)) {
        if (s.tid == 0) a.out[r] = at;
        return;
    }
    s.inv_t = 1.0 / temp;

    // The cut after the first `want` tokens (by_mass: after the tokens with less than `limit` mass before them) of what
    // `cut` keeps: a radix search over the keys, 11 bits a pass. before: the mass above the bins searched.
    const auto narrow = [&](Cut cut, bool by_mass, int want, double limit, uint64_t& kept_mass) -> Cut {
        uint32_t prefix = 0;
        uint64_t above_mass = 0;
        int above = 0;
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), nb = pass == 2 ? 1024 : 2048;
            for (int i = s.tid; i < BINS; i += SAMPLE_THREADS) {
                mass[i] = 0;
                count[i] = 0;
            }
            __syncthreads();
            s.each([&](int, float x) {
                const uint32_t k = order_key(x);
                if (k < cut.key || (pass > 0 && (k >> (shift + (pass == 1 ? 11 : 10))) != prefix)) return;
                double wd;
                const uint32_t b = (k >> shift) & (nb - 1);
                atomicAdd(&count[b], 1u);
                atomicAdd((unsigned long long*)&mass[b], (unsigned long long)s.weight(x, wd));
            });
            __syncthreads();
            // the bins from the top: each thread's two, then a scan over the threads (2 bins each, the highest first)
            const int b1 = nb - 1 - 2 * s.tid, b0 = b1 - 1;
            const bool live = b0 >= 0;
            uint32_t c1 = live ? count[b1] : 0, c0 = live ? count[b0] : 0;
            uint64_t m1 = live ? mass[b1] : 0, m0 = live ? mass[b0] : 0;
            // tokens at cut.key count as far as the cut keeps them (all of one key: the last pass's bin)
            uint64_t cs = c1 + c0, ms = m1 + m0;
            for (int d = 1; d < WAVE; d <<= 1) {
                const uint64_t oc = __shfl_up(cs, d, WAVE), om = __shfl_up(ms, d, WAVE);
                if (s.lane >= d) {
                    cs += oc;
                    ms += om;
                }
            }
            __syncthreads();
            if (s.lane == WAVE - 1) part[s.w] = ms;
            __syncthreads();
            uint64_t base_m = 0;
            for (int i = 0; i < s.w; ++i) base_m += part[i];
            __syncthreads();
            if (s.lane == WAVE - 1) part[s.w] = cs;
            if (s.tid == 0) found_bin = -1;
            __syncthreads();
            uint64_t base_c = 0;
            for (int i = 0; i < s.w; ++i) base_c += part[i];
            // the first bin behind which the cut lies
            uint64_t cb = above + base_c + cs - c1 - c0, mb = above_mass + base_m + ms - m1 - m0;
            if (live) {
                for (int j = 0; j < 2; ++j) {
                    const uint32_t c = j == 0 ? c1 : c0;
                    const uint64_t m = j == 0 ? m1 : m0;
                    const bool here = by_mass ? (double)mb < limit && !((double)(mb + m) < limit) : cb < (uint64_t)want && cb + c >= (uint64_t)want;
                    if (here && c > 0) {
                        found_bin = j == 0 ? b1 : b0;
                        found_mass = mb;
                        found_count = (int)cb;
                    }
                    cb += c;
                    mb += m;
                }
            }
            __syncthreads();
            if (found_bin < 0) return cut;                               // everything is kept
            above = found_count;
            above_mass = found_mass;
            prefix = pass == 0 ? found_bin : ((prefix << (pass == 1 ? 11 : 10)) | found_bin);
            __syncthreads();
        }
        // all of one key: equal weights
        double wd;
        const uint32_t kb = prefix ^ ((prefix >> 31) ? 0x80000000u : 0xFFFFFFFFu);
        const uint64_t each = s.weight(__uint_as_float(kb), wd);
        int ties;
        if (by_mass) {
            const double left = (limit - (double)above_mass) / (double)max(each, (uint64_t)1);
            ties = (int)fmin(ceil(left), 2147483647.0);
        } else {
            ties = want - above;
        }
        if (prefix == cut.key) ties = min(ties, cut.ties);
        kept_mass = above_mass + each * (uint64_t)ties;
        return Cut{prefix, max(ties, 1)};
    };

    Cut cut{0, 0x7fffffff};
    if (top_k > 0 || top_p < 1.0) {
        uint64_t total = 0;
        s.each([&](int, float x) {
            double wd;
            total += s.weight(x, wd);
        });
        total = block_sum(total, part, s.lane, s.w);
        if (top_k > 0 && top_k < s.vocab) cut = narrow(cut, false, top_k, 0.0, total);
        if (top_p < 1.0) {
            uint64_t unused = 0;
            cut = narrow(cut, true, 0, fmax(top_p * (double)total, 0.5), unused);
        }
    }

    // The running sum in index order: tiles in turn, each wave's kept mass and ties of a tile, the tile that the target
    // falls into, the wave, the lane. Two rounds: the sum of all, then the search.
    const auto tile_mass = [&](int i0, int& tie_base, uint64_t (&wt)[Sampler<T>::E]) -> uint64_t {
        constexpr int E = Sampler<T>::E;
        uint64_t sum = 0;
        int ties = 0;
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = i0 + e < s.vocab ? to_f32(s.row[i0 + e]) : -__builtin_inff();
            ties += i0 + e < s.vocab && order_key(x[e]) == cut.key;
        }
        // ties before this lane's in the tile
        int scan = ties;
        for (int d = 1; d < WAVE; d <<= 1) {
            const int o = __shfl_up(scan, d, WAVE);
            if (s.lane >= d) scan += o;
        }
        __syncthreads();
        if (s.lane == WAVE - 1) count[s.w] = scan;
        __syncthreads();
        int base = tie_base, all = 0;
        for (int i = 0; i < SAMPLE_WAVES; ++i) {
            if (i < s.w) base += count[i];
            all += count[i];
        }
        base += scan - ties;
        tie_base += all;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            wt[e] = 0;
            if (i0 + e >= s.vocab) continue;
            const uint32_t k = order_key(x[e]);
            double wd;
            const uint64_t m = s.weight(x[e], wd);
            const bool kept = (k > cut.key || (k == cut.key && base++ < cut.ties)) && (wd >= min_p || i0 + e == at);
            wt[e] = kept ? m : 0;
            sum += wt[e];
        }
        return sum;
    };
    uint64_t mine = 0;
    int tie_base = 0;
    uint64_t wt[Sampler<T>::E];
    for (int t0 = 0; t0 < s.vocab; t0 += Sampler<T>::TILE) mine += tile_mass(t0 + s.tid * Sampler<T>::E, tie_base, wt);
    const uint64_t all = block_sum(mine, part, s.lane, s.w);
    const float u = a.uniforms[r];
    // the largest target is the last kept token's
    const double want = fmin((double)fmaxf(u, 0.0f) * (double)all, (double)(all - 1));
    uint64_t run = 0;
    tie_base = 0;
    if (s.tid == 0) found_bin = -1;
    __syncthreads();
    for (int t0 = 0; t0 < s.vocab; t0 += Sampler<T>::TILE) {
        const int i0 = t0 + s.tid * Sampler<T>::E;
        const uint64_t sum = tile_mass(i0, tie_base, wt);
        uint64_t scan = sum;
        for (int d = 1; d < WAVE; d <<= 1) {
            const uint64_t o = __shfl_up(scan, d, WAVE);
            if (s.lane >= d) scan += o;
        }
        if (s.lane == WAVE - 1) part[s.w] = scan;
        __syncthreads();
        uint64_t before = run, tile = 0;
        for (int i = 0; i < SAMPLE_WAVES; ++i) {
            if (i < s.w) before += part[i];
            tile += part[i];
        }
        before += scan - sum;
        if ((double)before <= want && (double)(before + sum) > want && sum > 0) {
            for (int e = 0; e < Sampler<T>::E; ++e) {
                before += wt[e];
                if ((double)before > want) {
                    found_bin = i0 + e;
                    break;
                }
            }
        }
        run += tile;
        __syncthreads();
        if (found_bin >= 0) break;
    }
    if (s.tid == 0) a.out[r] = found_bin >= 0 ? found_bin : at;
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

extern "C" int kush_sample(int dtype, const void* logits, int64_t row_stride, int64_t rows, int64_t vocab,
                           const float* uniforms, double temperature, const float* temperatures, int32_t top_k,
                           const int32_t* top_ks, double top_p, const float* top_ps, double min_p, const float* min_ps,
                           int64_t* out, void* stream) {
    if (rows < 0 || rows > 0x7fffffff || vocab < 1 || vocab > (1 << 24) || row_stride < 0)
        return kush_fail(-2, "kush_sample: bad rows %lld / vocab %lld (1 .. 2^24) / row_stride %lld", (long long)rows,
                         (long long)vocab, (long long)row_stride);
    if (dtype < 0 || dtype > 2) return kush_fail(-1, "kush_sample: unsupported dtype code %d (0 fp32, 1 fp16, 2 bf16)", dtype);
    if (rows == 0) return 0;
    int log = 0;
    while ((1ll << log) < vocab) ++log;
    const SampleArgs a{logits,      row_stride, (int)vocab,   61 - log, uniforms, temperature, top_p, min_p, top_k,
                       temperatures, top_ps,     min_ps,       top_ks,   out};
    const dim3 grid((unsigned)rows), block(SAMPLE_THREADS);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == 0)
        sample_kernel<float><<<grid, block, 0, st>>>(a);
    else if (dtype == 1)
        sample_kernel<_Float16><<<grid, block, 0, st>>>(a);
    else
        sample_kernel<bf16_t><<<grid, block, 0, st>>>(a);
    return kush_check_launch("kush_sample");
}
