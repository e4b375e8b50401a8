// Paged attention of a batch over one shared prefix and each sequence's own
// pages (sdl_prefix_attention).
//
// Row (b, j, h) with kv head g = h / ratio attends P prefix keys and own keys
// [0, starts[b] + j] in one softmax:
//   o = (sum_i 2^(s_i - m) v_i) / (sum_i 2^(s_i - m)),  s_i = q . k_i * scale * log2(e)
// Softmax sums over disjoint key sets merge exactly: a set leaves (m, l, O)
// with O = sum 2^(s - m) v and l = sum 2^(s - m), and the row is
//   sum_x 2^(m_x - M) O_x / sum_x 2^(m_x - M) l_x,  M = max_x m_x.
// So the prefix is read once for all sequences: the query rows of every
// sequence stand in one matrix per kv head, flat row f = (b * chunk + j) *
// ratio + h % ratio, and a work item is a tile of flat rows against a range of
// prefix keys, or the rows of one sequence against a range of its own keys.
// Items write fp32 partials [g][f][slot], prefix ranges first, then own
// ranges; prefix_merge_kernel joins them (fixed order: results do not depend
// on scheduling).
//
// Times below are of whole calls in a captured graph of 30, over three sets of
// inputs in turn; those of 50 us and more move by up to 5 % with the clock that
// the power limit leaves.  A call through Python takes 10 to 13 us at least.
#include "sdl_common.cuh"

#include <cuda.h>
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstring>
#include <type_traits>

namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct PfxParams {
    const void* q;
    int64_t q_sb, q_sj, q_sh;
    void* out;
    int64_t o_sb, o_sj, o_sh;
    int out_dtype, dtype;
    const char* k_pool;
    const char* v_pool;
    const int32_t* table;
    int width, capacity, layer, block_size, table_rows;
    const int32_t* rows;
    const int32_t* starts;
    const int32_t* valid_rows;
    int prefix_row, prefix_len;
    int max_limit;    // own keys at and past it are not attended
    int B, chunk, Hq, Hkv, ratio, hd;
    int F;            // flat rows of one kv head: B * chunk * ratio
    int row_tile;     // flat rows of one own item
    int ptile;        // flat rows of one prefix item
    int ptiles;       // row tiles of the prefix
    int nsp, ppk;     // prefix splits and keys of each
    int mtiles;       // row tiles of one sequence
    int nsm, mpk;     // own splits (grid bound) and keys of each
    int nslot;        // partial slots of one row: nsp + nsm
    int own_direct;   // > 0: the merge attends the own keys itself, at most a page of them
    int p_split;      // 16-bit weights as a hi + lo pair (fp32 output)
    int out_vec;      // out rows take 4-element stores
    float scale_log2;
    float* o_part;    // [Hkv][F][nslot][hd]
    float* ml_part;   // [Hkv][F][nslot][2]
    int32_t* err;
};

SDL_DEV int pfx_nvalid(const PfxParams& p, int b) {
    return p.valid_rows ? max(0, min(p.valid_rows[b], p.chunk)) : p.chunk;
}

// Own keys that row j of sequence b attends: starts[b] + j + 1, within [0,
// max_limit].  `over` where the bound cuts some off (the merge reports it).
SDL_DEV int pfx_limit(const PfxParams& p, int b, int j, bool& over) {
    const int start = p.starts[b];
    over = start > p.max_limit - 1 - j;  // so written, nothing overflows
    return over ? p.max_limit : max(0, start + j + 1);
}

// One item: flat rows [f0, f1) of kv head g against keys [k0, k1) of the
// block-table row `seq`, into partial slot `slot`.
struct Item {
    int g, f0, f1, k0, k1, seq, slot;
    bool own;  // own keys: row limits apply
};

// Items of the prefix: row tiles fastest (they share their keys in L2), then
// kv heads, then key ranges.  Own items: kv heads fastest (a token row holds
// all heads), then row tiles, sequences and key ranges.  False: nothing to do.
SDL_DEV bool pfx_item(const PfxParams& p, int64_t i, Item& it) {
    const int64_t npre = (int64_t)p.ptiles * p.Hkv * p.nsp;
    if (i < npre) {
        const int t = (int)(i % p.ptiles);
        it.g = (int)(i / p.ptiles % p.Hkv);
        it.slot = (int)(i / p.ptiles / p.Hkv);
        it.f0 = t * p.ptile;
        it.f1 = min(p.F, it.f0 + p.ptile);
        it.k0 = it.slot * p.ppk;
        it.k1 = min(p.prefix_len, it.k0 + p.ppk);
        it.seq = p.prefix_row;
        it.own = false;
        return it.k0 < it.k1;
    }
    i -= npre;
    it.g = (int)(i % p.Hkv);
    const int t = (int)(i / p.Hkv % p.mtiles);
    const int b = (int)(i / p.Hkv / p.mtiles % p.B);
    const int s = (int)(i / p.Hkv / p.mtiles / p.B);
    const int R = p.chunk * p.ratio;
    const int nvalid = pfx_nvalid(p, b);
    const int r0 = t * p.row_tile, r1 = min(R, min(r0 + p.row_tile, nvalid * p.ratio));
    if (r0 >= r1) return false;
    bool over;
    const int lmax = pfx_limit(p, b, (r1 - 1) / p.ratio, over);  // keys the tile's last row attends
    it.k0 = s * p.mpk;
    it.k1 = min(lmax, it.k0 + p.mpk);
    it.f0 = b * R + r0;
    it.f1 = b * R + r1;
    it.seq = p.rows[b];
    it.slot = p.nsp + s;
    it.own = true;
    return it.k0 < it.k1;
}

// First pool token row of logical page `pg` of block-table row `seq`
// (out-of-range entries are reported and read page 0).
SDL_DEV int64_t pfx_page_row(const PfxParams& p, int seq, int pg) {
    int phys = pg < p.width && seq >= 0 && seq < p.table_rows ? p.table[(int64_t)seq * p.width + pg] : -1;
    if (phys < 0 || phys >= p.capacity) {
        sdl_raise(p.err, SDL_DEVERR_BAD_INDEX);
        phys = 0;
    }
    return ((int64_t)p.layer * p.capacity + phys) * p.block_size;
}

// The row of flat index f: its sequence, chunk row, q head and own key limit.
struct FlatRow {
    int b, j, h, limit;
    bool valid, over;
};

SDL_DEV FlatRow pfx_prefix_row(const PfxParams& p, int f, int g) {  // limit not set
    FlatRow r;
    const int bj = f / p.ratio;
    r.h = g * p.ratio + (f - bj * p.ratio);
    r.b = bj / p.chunk;
    r.j = bj - r.b * p.chunk;
    r.limit = 0;
    r.over = false;
    r.valid = r.j < pfx_nvalid(p, r.b);
    return r;
}

SDL_DEV FlatRow pfx_row(const PfxParams& p, int f, int g) {
    FlatRow r = pfx_prefix_row(p, f, g);
    r.limit = pfx_limit(p, r.b, r.j, r.over);
    return r;
}

// Launch order.  The tcgen05 plan launches the prefix items first and the own
// items behind them: the own grid starts once every prefix CTA is resident and
// fills the SMs that the prefix leaves free or finishes with.  The prefix grid
// waits for what precedes it (griddepcontrol.wait) and only then lets its
// dependents start, so an own CTA that runs sees q, the pages and the
// workspace's last use complete without a wait of its own.  CTA 0 of the own
// grid stands in its wait before it exits instead, which keeps the merge behind
// both grids (the others leave at once: items without keys must not hold a slot
// until the prefix is done).
SDL_DEV void pfx_enter(int behind) {
    if (!behind) pdl_wait();
    pdl_launch_dependents();
}
SDL_DEV void pfx_leave(int behind) {
    if (behind && blockIdx.x == 0) pdl_wait();
}

// --------------------------------------------------------- CUDA-core kernel
// Any dtype, head_dim <= 256 and page size, in two forms.  The narrow one, for
// few rows: 128 threads take 32 flat rows against tiles of 32 keys held in
// shared memory as fp32: thread (rg, kg) owns rows 2 rg, 2 rg + 1, keys
// kg + 8 i of S and dims kg + 8 i of O (strided, so a quarter warp reads
// consecutive words).
constexpr int kGenRows = 32, kGenKeys = 32, kGenThreads = 128;

inline size_t gen_smem(int hd) {
    return sizeof(float) * ((size_t)kGenRows * (hd + 1) + (size_t)kGenKeys * (hd + 1) + (size_t)kGenKeys * hd +
                            kGenRows * (kGenKeys + 1));
}

template <typename T, int ND>
__global__ void __launch_bounds__(kGenThreads)
prefix_generic_kernel(const PfxParams p, const int64_t item0, const int behind) {
    extern __shared__ __align__(16) float sh[];
    const int hd = p.hd;
    float* sQ = sh;                              // [32][hd + 1]
    float* sK = sQ + kGenRows * (hd + 1);        // [32][hd + 1]
    float* sV = sK + kGenKeys * (hd + 1);        // [32][hd]
    float* sP = sV + kGenKeys * hd;              // [32][33]
    __shared__ int64_t s_tok[kGenKeys];
    __shared__ int s_lim[kGenRows];
    pfx_enter(behind);
    Item it;
    if (!pfx_item(p, item0 + blockIdx.x, it)) {
        pfx_leave(behind);
        return;
    }
    const int tid = threadIdx.x, rg = tid >> 3, kg = tid & 7;
    const int nrow = it.f1 - it.f0;
    if (tid < kGenRows) {
        int lim = 0;
        if (tid < nrow) {
            const FlatRow r = pfx_row(p, it.f0 + tid, it.g);
            lim = !r.valid ? 0 : it.own ? min(r.limit, it.k1) : it.k1;
        }
        s_lim[tid] = lim;
    }
    for (int i = tid; i < kGenRows * hd; i += kGenThreads) {
        const int r = i / hd, e = i - r * hd;
        float x = 0.f;
        if (r < nrow) {
            const FlatRow fr = pfx_row(p, it.f0 + r, it.g);
            if (fr.valid)
                x = to_f32<T>(reinterpret_cast<const T*>(p.q)[fr.b * p.q_sb + fr.j * p.q_sj + fr.h * p.q_sh + e]);
        }
        sQ[r * (hd + 1) + e] = x;
    }
    float o[2][ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) o[0][i] = o[1][i] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const int64_t row_elems = (int64_t)p.Hkv * hd;
    for (int k0 = it.k0; k0 < it.k1; k0 += kGenKeys) {
        __syncthreads();
        if (tid < kGenKeys) {
            const int key = k0 + tid;
            int64_t tok = -1;
            if (key < it.k1) tok = pfx_page_row(p, it.seq, key / p.block_size) + key % p.block_size;
            s_tok[tid] = tok;
        }
        __syncthreads();
        for (int i = tid; i < kGenKeys * hd; i += kGenThreads) {
            const int r = i / hd, e = i - r * hd;
            const int64_t tok = s_tok[r];
            float kx = 0.f, vx = 0.f;  // rows past the range stay zero, whatever the pool holds there
            if (tok >= 0) {
                const int64_t at = tok * row_elems + (int64_t)it.g * hd + e;
                kx = to_f32<T>(reinterpret_cast<const T*>(p.k_pool)[at]);
                vx = to_f32<T>(reinterpret_cast<const T*>(p.v_pool)[at]);
            }
            sK[r * (hd + 1) + e] = kx;
            sV[r * hd + e] = vx;
        }
        __syncthreads();
        float s[2][4] = {};
        for (int e = 0; e < hd; ++e) {
            const float q0 = sQ[(2 * rg) * (hd + 1) + e], q1 = sQ[(2 * rg + 1) * (hd + 1) + e];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float kx = sK[(kg + 8 * i) * (hd + 1) + e];
                s[0][i] = fmaf(q0, kx, s[0][i]);
                s[1][i] = fmaf(q1, kx, s[1][i]);
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int lim = s_lim[2 * rg + u];
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[u][i] = k0 + kg + 8 * i < lim ? s[u][i] * p.scale_log2 : -INFINITY;
                mx = fmaxf(mx, s[u][i]);
            }
#pragma unroll
            for (int w = 1; w < 8; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
            const float mn = fmaxf(m[u], mx);
            const float base = mn == -INFINITY ? 0.f : mn;
            const float alpha = exp2f(m[u] - base);
            m[u] = mn;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float pr = exp2f(s[u][i] - base);
                sP[(2 * rg + u) * (kGenKeys + 1) + kg + 8 * i] = pr;
                sum += pr;
            }
#pragma unroll
            for (int w = 1; w < 8; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
            l[u] = l[u] * alpha + sum;
#pragma unroll
            for (int i = 0; i < ND; ++i) o[u][i] *= alpha;
        }
        __syncwarp();  // a row's eight threads share a warp
        for (int r = 0; r < kGenKeys; ++r) {
            const float p0 = sP[(2 * rg) * (kGenKeys + 1) + r], p1 = sP[(2 * rg + 1) * (kGenKeys + 1) + r];
#pragma unroll
            for (int i = 0; i < ND; ++i) {
                const int e = kg + 8 * i;
                const float vx = e < hd ? sV[r * hd + e] : 0.f;
                o[0][i] = fmaf(p0, vx, o[0][i]);
                o[1][i] = fmaf(p1, vx, o[1][i]);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int r = 2 * rg + u;
        if (r >= nrow) continue;
        const int64_t idx = ((int64_t)it.g * p.F + it.f0 + r) * p.nslot + it.slot;
#pragma unroll
        for (int i = 0; i < ND; ++i)
            if (kg + 8 * i < hd) p.o_part[idx * hd + kg + 8 * i] = o[u][i];
        if (kg == 0) {
            p.ml_part[idx * 2] = m[u];
            p.ml_part[idx * 2 + 1] = l[u];
        }
    }
    pfx_leave(behind);
}

// Pairs of fp32 values as one 64-bit operand of the packed fp32 instructions.
SDL_DEV uint64_t pack_f32x2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
SDL_DEV void unpack_f32x2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
SDL_DEV uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
SDL_DEV uint64_t add_f32x2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// The wide form, for 64 rows against tiles of 64 keys, every operand of either
// product read from shared memory as 16-byte pieces along its summed axis:
// thread (rg, cg) owns rows rg + 16 u, keys cg + 8 i of S, and dims
// 32 i + 4 cg .. + 3 of O (i < NC = head_dim / 32, zero padded).  Rows are four
// words longer than the head, so eight lanes' pieces cover all banks.  Products
// are packed in pairs (fma.rn.f32x2; of dims in both products), fp32 tiles
// arrive by cp.async under the softmax and the other product.  Bound by the 12
// reads of 16 bytes for 128 products (shared memory 71 % busy, issue slots 47 %):
// 8192 rows x 2 heads behind 4096 + 1..300 keys, d 64, 621 us (29 TFLOP/s); 2304
// x 2 behind 2000 + 1..300, d 128, 340 us (15).  Plain loads cost 3 % and 15 %,
// products without pairs another 5 %.  Eight rows a thread read less and hide less (two blocks per SM):
// no gain.
constexpr int kWideRows = 64, kWideKeys = 64, kWidePitch = kWideKeys + 4;

inline size_t wide_smem(int nc) {
    const size_t hp = 32 * (size_t)nc;
    return sizeof(float) * ((kWideRows + kWideKeys) * (hp + 4) + kWideKeys * hp + kWideRows * kWidePitch);
}

// Four elements from `src`, the ones at and past `n` zero.
template <typename T>
SDL_DEV float4 load4(const T* src, int n, bool vec) {
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
    if (vec && n >= 4) {
        if constexpr (sizeof(T) == 4) {
            r = *reinterpret_cast<const float4*>(src);
        } else {
            const uint2 v = *reinterpret_cast<const uint2*>(src);
            const T* x = reinterpret_cast<const T*>(&v);
            r = make_float4(to_f32<T>(x[0]), to_f32<T>(x[1]), to_f32<T>(x[2]), to_f32<T>(x[3]));
        }
    } else {
        if (n > 0) r.x = to_f32<T>(src[0]);
        if (n > 1) r.y = to_f32<T>(src[1]);
        if (n > 2) r.z = to_f32<T>(src[2]);
        if (n > 3) r.w = to_f32<T>(src[3]);
    }
    return r;
}

// 16 bytes to shared memory, zeros where `on` is false.
SDL_DEV void cp_async16_zfill(void* dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16 : 0)
                 : "memory");
}
SDL_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> SDL_DEV void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T, int NC>
__global__ void __launch_bounds__(kGenThreads, NC <= 2 ? 3 : 1)
prefix_wide_kernel(const PfxParams p, const int64_t item0, const int behind) {
    extern __shared__ __align__(16) float sh[];
    constexpr int HP = 32 * NC, PITCH = HP + 4;   // padded head_dim, and a row of Q or K
    const int hd = p.hd;
    float* sQ = sh;                               // [64][PITCH]
    float* sK = sQ + kWideRows * PITCH;           // [64][PITCH]
    float* sV = sK + kWideKeys * PITCH;           // [64][HP]
    float* sP = sV + kWideKeys * HP;              // [64 rows][68]
    __shared__ int64_t s_tok[2][kWideKeys];  // a tile's tokens, by its parity
    __shared__ int s_lim[kWideRows];
    pfx_enter(behind);
    Item it;
    if (!pfx_item(p, item0 + blockIdx.x, it)) {
        pfx_leave(behind);
        return;
    }
    const int tid = threadIdx.x, rg = tid >> 3, cg = tid & 7;
    const int nrow = it.f1 - it.f0;
    const int64_t row_elems = (int64_t)p.Hkv * hd;
    const int align = 4 * (int)sizeof(T);
    const bool vec = hd % 4 == 0 && reinterpret_cast<uintptr_t>(p.k_pool) % align == 0 &&
                     reinterpret_cast<uintptr_t>(p.v_pool) % align == 0;
    for (int r = tid >> 3; r < kWideRows; r += kGenThreads / 8) {  // eight lanes load a row
        const FlatRow fr = pfx_row(p, min(it.f0 + r, p.F - 1), it.g);
        const bool on = r < nrow && fr.valid;
        if (cg == 0) s_lim[r] = !on ? 0 : it.own ? min(fr.limit, it.k1) : it.k1;
        const T* q = reinterpret_cast<const T*>(p.q) + fr.b * p.q_sb + fr.j * p.q_sj + fr.h * p.q_sh;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int e = 32 * i + 4 * cg;
            *reinterpret_cast<float4*>(sQ + r * PITCH + e) = load4<T>(q + e, on ? hd - e : 0, false);
        }
    }
    uint64_t o[4][NC][2];  // pairs of dims
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < NC; ++i) o[u][i][0] = o[u][i][1] = 0ull;
    float m[4], l[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        m[u] = -INFINITY;
        l[u] = 0.f;
    }
    // fp32 tiles arrive by cp.async, K of the next one under this one's softmax
    // and O, V under the next S; other types are converted on the way
    const bool async = sizeof(T) == 4 && vec;
    int phys = 0;  // threads of a key: its page of the next tile, read a tile ahead
    auto read_page = [&](int k0) {
        const int key = k0 + tid, pg = key / p.block_size;
        phys = key < it.k1 && pg < p.width && it.seq >= 0 && it.seq < p.table_rows
                   ? p.table[(int64_t)it.seq * p.width + pg]
                   : -1;
    };
    auto set_tok = [&](int k0, int at) {  // as pfx_page_row
        const int key = k0 + tid;
        int64_t tok = -1;
        if (key < it.k1) {
            if (phys < 0 || phys >= p.capacity) {
                sdl_raise(p.err, SDL_DEVERR_BAD_INDEX);
                phys = 0;
            }
            tok = ((int64_t)p.layer * p.capacity + phys) * p.block_size + key % p.block_size;
        }
        s_tok[at][tid] = tok;
    };
    auto copy_tile = [&](const char* pool, float* dst, int pitch, int at) {
#pragma unroll
        for (int j = 0; j < kWideKeys / (kGenThreads / 8); ++j) {
            const int r = (tid >> 3) + j * (kGenThreads / 8);
            const int64_t tok = s_tok[at][r];
            const T* src = reinterpret_cast<const T*>(pool) + max((int64_t)0, tok) * row_elems + (int64_t)it.g * hd;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                const int e = 32 * i + 4 * cg;
                const bool on = tok >= 0 && e < hd;  // zeros elsewhere, whatever the pool holds there
                cp_async16_zfill(dst + r * pitch + e, src + (on ? e : 0), on);
            }
        }
        cp_async_commit();
    };
    if (async) {
        if (tid < kWideKeys) {
            read_page(it.k0);
            set_tok(it.k0, 0);
            read_page(it.k0 + kWideKeys);
        }
        __syncthreads();
        copy_tile(p.k_pool, sK, PITCH, 0);
        copy_tile(p.v_pool, sV, HP, 0);
        cp_async_wait<1>();
        __syncthreads();
    }
    int next = 1;  // parity of the next tile
    for (int k0 = it.k0; k0 < it.k1; k0 += kWideKeys, next ^= 1) {
        const bool more = k0 + kWideKeys < it.k1;
        if (async) {
            if (tid < kWideKeys && more) {
                set_tok(k0 + kWideKeys, next);
                read_page(k0 + 2 * kWideKeys);
            }
        } else {
            __syncthreads();
            if (tid < kWideKeys) {
                read_page(k0);
                set_tok(k0, 0);
            }
            __syncthreads();
#pragma unroll 4
            for (int r = tid >> 3; r < kWideKeys; r += kGenThreads / 8) {
                const int64_t tok = s_tok[0][r];
                const int64_t at = max((int64_t)0, tok) * row_elems + (int64_t)it.g * hd;
#pragma unroll
                for (int i = 0; i < NC; ++i) {
                    const int e = 32 * i + 4 * cg, n = tok >= 0 ? hd - e : 0;
                    const float4 kx = load4<T>(reinterpret_cast<const T*>(p.k_pool) + at + e, n, vec);
                    const float4 vx = load4<T>(reinterpret_cast<const T*>(p.v_pool) + at + e, n, vec);
                    *reinterpret_cast<float4*>(sK + r * PITCH + e) = kx;
                    *reinterpret_cast<float4*>(sV + r * HP + e) = vx;
                }
            }
            __syncthreads();
        }
        float s[4][8];
        {
            uint64_t s2[4][8];  // even and odd dims
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) s2[u][i] = 0ull;
#pragma unroll 2
            for (int e = 0; e < hd; e += 4) {
                ulonglong2 q[4];
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    q[u] = *reinterpret_cast<const ulonglong2*>(sQ + (rg + 16 * u) * PITCH + e);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(sK + (cg + 8 * i) * PITCH + e);
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        s2[u][i] = fma_f32x2(q[u].x, k.x, s2[u][i]);
                        s2[u][i] = fma_f32x2(q[u].y, k.y, s2[u][i]);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float lo, hi;
                    unpack_f32x2(s2[u][i], lo, hi);
                    s[u][i] = lo + hi;
                }
        }
        if (async && more) {
            __syncthreads();  // every thread has read K, and the next tile's tokens stand
            copy_tile(p.k_pool, sK, PITCH, next);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int lim = s_lim[rg + 16 * u];
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s[u][i] = k0 + cg + 8 * i < lim ? s[u][i] * p.scale_log2 : -INFINITY;
                mx = fmaxf(mx, s[u][i]);
            }
#pragma unroll
            for (int w = 1; w < 8; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
            const float mn = fmaxf(m[u], mx);
            const float base = mn == -INFINITY ? 0.f : mn;
            const float alpha = ex2_approx(m[u] - base);
            m[u] = mn;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float pr = ex2_approx(s[u][i] - base);
                sP[(rg + 16 * u) * kWidePitch + cg + 8 * i] = pr;
                sum += pr;
            }
            l[u] = l[u] * alpha + sum;  // this thread's keys; the row's eight threads join at the end
            const uint64_t alpha2 = pack_f32x2(alpha, alpha);
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                o[u][i][0] = fma_f32x2(o[u][i][0], alpha2, 0ull);
                o[u][i][1] = fma_f32x2(o[u][i][1], alpha2, 0ull);
            }
        }
        __syncwarp();  // a row's eight threads share a warp
        if (async) {  // V of this tile
            if (more) cp_async_wait<1>();
            else cp_async_wait<0>();
            __syncthreads();
        }
#pragma unroll 2
        for (int r = 0; r < kWideKeys; r += 4) {
            float pr[4][4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float4 v = *reinterpret_cast<const float4*>(sP + (rg + 16 * u) * kWidePitch + r);
                pr[u][0] = v.x;
                pr[u][1] = v.y;
                pr[u][2] = v.z;
                pr[u][3] = v.w;
            }
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int i = 0; i < NC; ++i) {
                    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(sV + (r + x) * HP + 32 * i + 4 * cg);
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint64_t w = pack_f32x2(pr[u][x], pr[u][x]);
                        o[u][i][0] = fma_f32x2(w, v.x, o[u][i][0]);
                        o[u][i][1] = fma_f32x2(w, v.y, o[u][i][1]);
                    }
                }
        }
        if (async && more) {
            cp_async_wait<0>();  // the next K
            __syncthreads();     // ... of every thread, and every thread has read V
            copy_tile(p.v_pool, sV, HP, next);
        }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int w = 1; w < 8; w <<= 1) l[u] += __shfl_xor_sync(0xffffffffu, l[u], w);
        const int r = rg + 16 * u;
        if (r >= nrow) continue;
        const int64_t idx = ((int64_t)it.g * p.F + it.f0 + r) * p.nslot + it.slot;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float x[4];
            unpack_f32x2(o[u][i][0], x[0], x[1]);
            unpack_f32x2(o[u][i][1], x[2], x[3]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int e = 32 * i + 4 * cg + j;
                if (e < hd) p.o_part[idx * hd + e] = x[j];
            }
        }
        if (cg == 0) {
            p.ml_part[idx * 2] = m[u];
            p.ml_part[idx * 2 + 1] = l[u];
        }
    }
    pfx_leave(behind);
}

// ----------------------------------------------------------- mma.sync kernel
// bf16 / f16, head_dim 64 / 128, 16-token pages.  Four producer warps, one per
// page, stream stages of 64 keys (K and V in 2 KB 128-byte-swizzled boxes)
// through a TMA ring: a warp issues a box in 176 cycles whatever the number of
// issuing warps (11.6 bytes a cycle with one, 46 with four; measured from L2),
// so one producer alone would hold a 32 KB stage back by 2800 cycles.  Four
// consumer warps compute S = Q K^T and O += P V with
// mma.sync m16n8k16, query rows on M, the softmax in registers (row maxima by
// quad shuffles, rescaled only when a maximum grows by more than 2^8, so P
// stays below 2^8), S's accumulators repacked in place as P's operand.
// Two ways to share a stage:
//   rows  -- each warp owns 16 of the item's up to 64 rows and reads all four
//            pages (prefix tiles, verify and extension blocks);
//   keys  -- every warp takes the same 16 rows and one of the four pages
//            (items of at most 16 rows: decode), and the four partial
//            softmaxes merge through shared memory at the end.
// The keys form keeps all four warps busy on a decode row group (6 of 16 MMA
// rows filled, but the item is bound by its 32 KB stages, not by the MMAs).
constexpr int kPage = 16;
constexpr int kBox = kPage * 128;   // one [16 tokens][64 columns] 16-bit box
constexpr int kStagePages = 4;
constexpr int kStageKeys = kStagePages * kPage;
constexpr int kMmaWarps = 4;
constexpr int kMmaRows = 16 * kMmaWarps;
constexpr int kMmaThreads = (kMmaWarps + kStagePages) * 32;  // a producer warp per page of a stage
constexpr uint32_t kWaitLimit = 1u << 20;
constexpr float kLazyLog2 = 8.f;

template <int HD>
struct MmaCfg {
    static constexpr int DO = HD / 64;
    static constexpr int kPageBytes = 2 * DO * kBox;          // K halves, then V halves
    static constexpr int kStage = kStagePages * kPageBytes;   // 32 KB at d 128
    // d 128: two CTAs per SM, 96 KB rings; 256 threads launch with 128 registers
    // each, of which the consumer warpgroup takes 200 and the producers keep 56
    // (128 * 200 + 128 * 56 = 256 * 128).  d 64: three CTAs, 64 KB rings, 80
    // registers shared as 128 and 32 (256 decode rows behind 2051 keys: 23.9
    // us, 26.2 with two CTAs; 200 rows of 8 kv heads: 47.4 and 56.2).
    static constexpr int kCtas = HD == 128 ? 2 : 3;
    static constexpr int kStages = HD == 128 ? 3 : 4;
    static constexpr int kRegs = HD == 128 ? 200 : 128, kHelpRegs = HD == 128 ? 56 : 32;
    static constexpr int kSmem = kStages * kStage + 1024;
};

SDL_DEV uint32_t ld_u32(const void* x) { return *reinterpret_cast<const uint32_t*>(x); }

// One warp's running softmax over 16 rows: rows gq and gq + 8 of this thread.
template <int HD>
struct MmaState {
    float o[HD / 8][4];
    float m_a, m_b, l_a, l_b;
};

// One stage for one warp: NP pages from page `pg`, whose first key is `pos0`.
template <int HD, typename T, int NP>
SDL_DEV void mma_stage(const PfxParams& p, uint32_t sb, int pg, int pos0, int lim_a, int lim_b, int lim_min, int k1,
                       const uint32_t (&qa)[HD / 16][4], MmaState<HD>& st) {
    using C = MmaCfg<HD>;
    constexpr int KS = HD / 16, ON = HD / 8, SN = 2 * NP, DO = C::DO;
    const int lane = threadIdx.x & 31, t4 = lane & 3;
    const int sw = lane & 7, mq = lane >> 3;
    float s[SN][4];
#pragma unroll
    for (int nt = 0; nt < SN; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
    // ldmatrix offsets: 16-byte chunk c of token row r sits at chunk c ^ (r & 7)
    const uint32_t pbase = sb + pg * C::kPageBytes;
#pragma unroll
    for (int ks = 0; ks < KS; ks += 2) {
        const int c = 2 * ks + mq;
        const uint32_t co = (c >> 3) * kBox + (((c & 7) ^ sw) << 4);
#pragma unroll
        for (int nt = 0; nt < SN; ++nt) {
            uint32_t b0, b1, b2, b3;
            ldmatrix_x4(pbase + (nt >> 1) * C::kPageBytes + ((nt & 1) * 8 + sw) * 128 + co, b0, b1, b2, b3);
            mma_16816<T>(s[nt], qa[ks], b0, b1);
            mma_16816<T>(s[nt], qa[ks + 1], b2, b3);
        }
    }
    const bool whole = pos0 + NP * kPage <= lim_min;  // every row attends every key
    float mxa = -INFINITY, mxb = -INFINITY;
#pragma unroll
    for (int nt = 0; nt < SN; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (!whole) {
                const int key = pos0 + nt * 8 + 2 * t4 + e;
                if (key >= lim_a) s[nt][e] = -INFINITY;
                if (key >= lim_b) s[nt][2 + e] = -INFINITY;
            }
            mxa = fmaxf(mxa, s[nt][e]);
            mxb = fmaxf(mxb, s[nt][2 + e]);
        }
    mxa = fmaxf(mxa, __shfl_xor_sync(0xffffffffu, mxa, 1));
    mxa = fmaxf(mxa, __shfl_xor_sync(0xffffffffu, mxa, 2));
    mxb = fmaxf(mxb, __shfl_xor_sync(0xffffffffu, mxb, 1));
    mxb = fmaxf(mxb, __shfl_xor_sync(0xffffffffu, mxb, 2));
    mxa *= p.scale_log2;
    mxb *= p.scale_log2;
    const bool na = mxa > st.m_a + kLazyLog2, nb = mxb > st.m_b + kLazyLog2;
    if (__any_sync(0xffffffffu, na || nb)) {
        const float aa = na ? ex2_approx(st.m_a - mxa) : 1.f;  // 0 on the first keys
        const float ab = nb ? ex2_approx(st.m_b - mxb) : 1.f;
        if (na) st.m_a = mxa;
        if (nb) st.m_b = mxb;
        st.l_a *= aa;
        st.l_b *= ab;
#pragma unroll
        for (int dn = 0; dn < ON; ++dn) {
            st.o[dn][0] *= aa;
            st.o[dn][1] *= aa;
            st.o[dn][2] *= ab;
            st.o[dn][3] *= ab;
        }
    }
    const float ua = st.m_a == -INFINITY ? 0.f : st.m_a, ub = st.m_b == -INFINITY ? 0.f : st.m_b;
#pragma unroll
    for (int kk = 0; kk < NP; ++kk) {
        uint32_t pa[4], pl[4];
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            const float* sv = s[2 * kk + hf];
            const float p0 = ex2_approx(fmaf(sv[0], p.scale_log2, -ua));
            const float p1 = ex2_approx(fmaf(sv[1], p.scale_log2, -ua));
            const float p2 = ex2_approx(fmaf(sv[2], p.scale_log2, -ub));
            const float p3 = ex2_approx(fmaf(sv[3], p.scale_log2, -ub));
            st.l_a += p0 + p1;
            st.l_b += p2 + p3;
            // one rounding of the weights: it weighs an element as its own
            // output rounding does (fp32 outputs carry a second, low part)
            pa[2 * hf] = pack2<T>(p0, p1);
            pa[2 * hf + 1] = pack2<T>(p2, p3);
            if (p.p_split) {
                pl[2 * hf] = pack2<T>(p0 - round_trip<T>(p0), p1 - round_trip<T>(p1));
                pl[2 * hf + 1] = pack2<T>(p2 - round_trip<T>(p2), p3 - round_trip<T>(p3));
            }
        }
        // V rows past the item's last key are zeroed: 0 * stale NaN is NaN
        const int key = pos0 + kk * kPage + 2 * t4;
        const bool tail = pos0 + (kk + 1) * kPage > k1;
        const uint32_t z0 = (key < k1 ? 0xffffu : 0u) | (key + 1 < k1 ? 0xffff0000u : 0u);
        const uint32_t z1 = (key + 8 < k1 ? 0xffffu : 0u) | (key + 9 < k1 ? 0xffff0000u : 0u);
        const uint32_t vrow = pbase + kk * C::kPageBytes + ((mq & 1) * 8 + sw) * 128;
#pragma unroll
        for (int dn = 0; dn < ON; dn += 2) {
            const int c = dn + (mq >> 1);
            uint32_t v0, v1, v2, v3;
            ldmatrix_x4_trans(vrow + (DO + (c >> 3)) * kBox + (((c & 7) ^ sw) << 4), v0, v1, v2, v3);
            if (tail) {
                v0 &= z0;
                v1 &= z1;
                v2 &= z0;
                v3 &= z1;
            }
            mma_16816<T>(st.o[dn], pa, v0, v1);
            mma_16816<T>(st.o[dn + 1], pa, v2, v3);
            if (p.p_split) {
                mma_16816<T>(st.o[dn], pl, v0, v1);
                mma_16816<T>(st.o[dn + 1], pl, v2, v3);
            }
        }
    }
}

template <int HD, typename T>
__global__ void __launch_bounds__(kMmaThreads, MmaCfg<HD>::kCtas)
prefix_mma_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const PfxParams p,
                  const int64_t item0, const int behind) {
    using C = MmaCfg<HD>;
    constexpr int DO = C::DO, KS = HD / 16, ON = HD / 8, NS = C::kStages;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t full[NS], empty[NS];
    __shared__ float s_ml[kMmaWarps][16][2];
    __shared__ int s_abort_flag;
    volatile int* s_abort = &s_abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        *s_abort = 0;
        for (int i = 0; i < NS; ++i) {
            mbar_init(&full[i], kStagePages);
            mbar_init(&empty[i], kMmaWarps);
        }
        fence_mbar_init();
        prefetch_tmap(&tmk);
        prefetch_tmap(&tmv);
    }
    pfx_enter(behind);
    Item it;
    if (!pfx_item(p, item0 + blockIdx.x, it)) {
        pfx_leave(behind);
        return;
    }
    __syncthreads();
    const int npages = (it.k1 - it.k0 + kPage - 1) / kPage;
    const int nst = (npages + kStagePages - 1) / kStagePages;

    if (warp >= kMmaWarps) {
        // ------------------------------------------------------ producers
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kHelpRegs));
        const int u = warp - kMmaWarps;  // this warp's page of every stage
        int issued = 0;
        bool stop = false;
        for (int i0 = 0; i0 < nst && !stop; i0 += 32) {  // one page-table read for 32 stages
            // pages past the range repeat its last one: their keys are masked
            const int tok = (int)pfx_page_row(p, it.seq,
                                              it.k0 / kPage + min((i0 + lane) * kStagePages + u, npages - 1));
            for (int i = i0; i < min(nst, i0 + 32); ++i) {
                const int st = i % NS;
                const int tu = __shfl_sync(0xffffffffu, tok, i - i0);
                int ok = 1;
                if (lane == 0) {
                    if (i >= NS) ok = mbar_wait_bounded(&empty[st], ((i / NS) - 1) & 1, kWaitLimit) ? 1 : 0;
                    if (!ok) sdl_raise(p.err, SDL_DEVERR_TIMEOUT);
                    if (!ok || *s_abort) {
                        ok = 0;
                        *s_abort = 1;
                    } else {
                        mbar_arrive_expect_tx(&full[st], C::kPageBytes);
                        uint8_t* dst = smem + st * C::kStage + u * C::kPageBytes;
#pragma unroll
                        for (int dd = 0; dd < DO; ++dd) tma_load_4d(dst + dd * kBox, &tmk, &full[st], 0, dd, it.g, tu);
#pragma unroll
                        for (int dd = 0; dd < DO; ++dd)
                            tma_load_4d(dst + (DO + dd) * kBox, &tmv, &full[st], 0, dd, it.g, tu);
                    }
                }
                if (!__shfl_sync(0xffffffffu, ok, 0)) {
                    stop = true;
                    break;
                }
                issued = i + 1;
            }
        }
        // never leave the CTA with bulk copies still landing in shared memory
        for (int i = max(0, issued - NS); i < issued; ++i)
            (void)mbar_wait_bounded(&full[i % NS], (i / NS) & 1, kWaitLimit);
        pfx_leave(behind);
        return;
    }

    // ----------------------------------------------------------- consumers
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegs));
    const int nrow = it.f1 - it.f0;
    const bool by_keys = nrow <= 16;
    const int t4 = lane & 3, gq = lane >> 2;
    const int ra = (by_keys ? 0 : warp * 16) + gq, rb = ra + 8;
    const FlatRow fa = pfx_row(p, min(it.f0 + ra, p.F - 1), it.g), fb = pfx_row(p, min(it.f0 + rb, p.F - 1), it.g);
    const bool va = ra < nrow && fa.valid, vb = rb < nrow && fb.valid;
    const bool active = by_keys || warp * 16 < nrow;
    // rows that are not attended keep the tile's limit (finite values, never stored)
    const int lim_a = va && it.own ? min(fa.limit, it.k1) : it.k1;
    const int lim_b = vb && it.own ? min(fb.limit, it.k1) : it.k1;
    const int lim_min = __reduce_min_sync(0xffffffffu, min(lim_a, lim_b));
    uint32_t qa[KS][4];
    {
        const T* q0 = reinterpret_cast<const T*>(p.q);
        const T* qpa = q0 + fa.b * p.q_sb + fa.j * p.q_sj + fa.h * p.q_sh + 2 * t4;
        const T* qpb = q0 + fb.b * p.q_sb + fb.j * p.q_sj + fb.h * p.q_sh + 2 * t4;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            qa[ks][0] = va ? ld_u32(qpa + ks * 16) : 0u;
            qa[ks][1] = vb ? ld_u32(qpb + ks * 16) : 0u;
            qa[ks][2] = va ? ld_u32(qpa + ks * 16 + 8) : 0u;
            qa[ks][3] = vb ? ld_u32(qpb + ks * 16 + 8) : 0u;
        }
    }
    MmaState<HD> st;
#pragma unroll
    for (int dn = 0; dn < ON; ++dn)
#pragma unroll
        for (int e = 0; e < 4; ++e) st.o[dn][e] = 0.f;
    st.m_a = st.m_b = -INFINITY;
    st.l_a = st.l_b = 0.f;
    bool aborted = false;
    for (int i = 0; i < nst; ++i) {
        const int sg = i % NS;
        const bool ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full[sg], (i / NS) & 1, kWaitLimit));
        if (!ok) {
            if (lane == 0) {
                sdl_raise(p.err, SDL_DEVERR_TIMEOUT);
                *s_abort = 1;
            }
            aborted = true;
            break;
        }
        const uint32_t sb = smem_u32(smem) + sg * C::kStage;
        const int pos0 = it.k0 + i * kStageKeys;
        if (by_keys) {
            if (pos0 + warp * kPage < it.k1)
                mma_stage<HD, T, 1>(p, sb, warp, pos0 + warp * kPage, lim_a, lim_b, lim_min, it.k1, qa, st);
        } else if (active) {
            mma_stage<HD, T, kStagePages>(p, sb, 0, pos0, lim_a, lim_b, lim_min, it.k1, qa, st);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[sg]);
    }
    st.l_a += __shfl_xor_sync(0xffffffffu, st.l_a, 1);
    st.l_a += __shfl_xor_sync(0xffffffffu, st.l_a, 2);
    st.l_b += __shfl_xor_sync(0xffffffffu, st.l_b, 1);
    st.l_b += __shfl_xor_sync(0xffffffffu, st.l_b, 2);
    const int64_t part0 = ((int64_t)it.g * p.F + it.f0) * p.nslot + it.slot;  // row r: + r * nslot
    if (!by_keys) {
        if (aborted || !active) return;
#pragma unroll
        for (int hr = 0; hr < 2; ++hr) {
            if (!(hr ? vb : va)) continue;
            const int64_t idx = part0 + (int64_t)(hr ? rb : ra) * p.nslot;
            float* op = p.o_part + idx * HD + 2 * t4;
#pragma unroll
            for (int dn = 0; dn < ON; ++dn)
                *reinterpret_cast<float2*>(op + dn * 8) = make_float2(st.o[dn][2 * hr], st.o[dn][2 * hr + 1]);
            if (t4 == 0)
                *reinterpret_cast<float2*>(p.ml_part + idx * 2) =
                    hr ? make_float2(st.m_b, st.l_b) : make_float2(st.m_a, st.l_a);
        }
        return;
    }
    // The four warps' softmaxes over the same rows merge in the ring's memory
    // (every copy has landed: each consumer waited for each stage).
    named_bar_sync(1, kMmaWarps * 32);
    float* so = reinterpret_cast<float*>(smem);  // [warp][16][HD]
#pragma unroll
    for (int hr = 0; hr < 2; ++hr) {
        const int r = gq + 8 * hr;
#pragma unroll
        for (int dn = 0; dn < ON; ++dn)
            *reinterpret_cast<float2*>(so + (warp * 16 + r) * HD + dn * 8 + 2 * t4) =
                make_float2(st.o[dn][2 * hr], st.o[dn][2 * hr + 1]);
        if (t4 == 0) {
            s_ml[warp][r][0] = hr ? st.m_b : st.m_a;
            s_ml[warp][r][1] = hr ? st.l_b : st.l_a;
        }
    }
    named_bar_sync(1, kMmaWarps * 32);
    if (aborted || *s_abort) return;
    constexpr int kQuads = HD / 4;  // threads per row
    for (int i = threadIdx.x; i < nrow * kQuads; i += kMmaWarps * 32) {
        const int r = i / kQuads, d0 = i % kQuads * 4;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kMmaWarps; ++w) M = fmaxf(M, s_ml[w][r][0]);
        const float base = M == -INFINITY ? 0.f : M;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < kMmaWarps; ++w) {
            const float wt = ex2_approx(s_ml[w][r][0] - base);
            const float4 o = *reinterpret_cast<const float4*>(so + (w * 16 + r) * HD + d0);
            acc.x = fmaf(wt, o.x, acc.x);
            acc.y = fmaf(wt, o.y, acc.y);
            acc.z = fmaf(wt, o.z, acc.z);
            acc.w = fmaf(wt, o.w, acc.w);
            l = fmaf(wt, s_ml[w][r][1], l);
        }
        const int64_t idx = part0 + (int64_t)r * p.nslot;
        *reinterpret_cast<float4*>(p.o_part + idx * HD + d0) = acc;
        if (d0 == 0) *reinterpret_cast<float2*>(p.ml_part + idx * 2) = make_float2(M, l);
    }
}

// ------------------------------------------------------------ tcgen05 kernel
// The 5th-generation tensor cores, in two forms of one kernel:
//   TILES = 2, the prefix of large batches (d 128): one CTA per SM takes 256
//        flat rows of a kv head (two row tiles of 128) against a key range;
//   TILES = 1: two CTAs per SM, each up to 128 flat rows against a key range of
//        the prefix, or (kOwn) up to 128 rows of one sequence against a range
//        of its own keys, with every row's causal limit (verify and extension
//        blocks).
// A step is 64 keys.  Warps:
//   4 per row tile  softmax: a thread owns one row, reads its 64 scores from
//        TMEM, and writes the 16-bit weights back over the first 32 of the
//        score columns (two keys per 32-bit column);
//   4 (2)   TMA producers, each its pages of every tile (a warp issues a 2 KB
//        box in 100 to 180 cycles, however many warps issue): K and V tiles of
//        four pages alternate in one ring;
//   1 per row tile  issues S_t(i) = Q_t K_i^T (both operands in shared memory,
//        128-byte swizzle) for row tile t and step i;
//   1 per row tile  issues O_t += P_t V_i (P from TMEM, V MN-major in shared
//        memory).
// Each tile has two score buffers, so S_t(i + 1) runs under the softmax of
// step i and a softmax warp always finds its next scores; S_t(i + 2) waits for
// PV_t(i), whose P lies in its columns.  A row whose maximum grew by more than
// 2^8 (rare after the first steps) waits for PV_t(i - 1) and rescales O_t in
// place.  Each product of each tile has a warp of its own because a thread that
// has issued MMAs sees its next barrier only once the pipe has taken them.
// Measured for 4608 rows x 2 kv heads behind 8192 keys, cycles per 128 keys of
// a CTA (of which 128-key MMAs would need 2048): one issuing warp and one
// 128-key score buffer 5400, a warp per product 4440, two 64-key buffers and
// four producers 4200, elected issue and part of the exponentials on the FMA
// pipe 3200.  64-key S products read 6 KB of operands per 32 cycles of MMA, 48
// at the shared memory's 128 bytes a cycle (2560 a step): the overlap pays it.
// 256 x 6 rows of 12 heads behind 16384 keys alone take 150 us with the merge:
// 1.03 PFLOP/s (a large matrix product: 1.70 in a burst, 1.42 sustained).
// TMEM: score buffers (tile t, i & 1) of 64 columns, then O_t, 128 apart.
constexpr int kURows = 128;                 // rows of one tile (MMA M)
constexpr int kUKeys = 64;                  // keys per step
constexpr int kUPages = kUKeys / kPage;
// Registers: a thread launches with 128; a softmax thread holds a row of
// scores, so those warpgroups take 168 and the equally many warpgroups of the
// other warps keep 88.
constexpr int kUSoftRegs = 168, kUHelpRegs = 88;

template <int HD, int TILES>
struct UCfg {
    static constexpr int kThreads = 256 * TILES;
    static constexpr int kProducer = 4 * TILES;           // first producer warp
    static constexpr int kProducers = 2 * TILES;
    static constexpr int kMine = kUPages / kProducers;    // a producer's pages of a tile
    static constexpr int kMmaS = kProducer + kProducers, kMmaPV = kMmaS + TILES;  // + row tile
    static constexpr uint32_t kTmemCols = 256 * TILES;
    static constexpr int kOCol = 2 * TILES * kUKeys;      // first O column
    static constexpr int DO = HD / 64;
    static constexpr int kQHalf = kURows * 128;           // 64 columns of a Q tile: 16 KB
    static constexpr int kQ = TILES * DO * kQHalf;
    static constexpr int kHalf = kUKeys * 128;            // 64 columns of a K or V tile: 8 KB
    static constexpr int kSlot = DO * kHalf;              // one K or V tile
    static constexpr int kSlots = TILES == 2 ? 10 : HD == 128 ? 4 : 8;
    static constexpr int kSmem = kQ + kSlots * kSlot + 1024;
    static constexpr int kPitch = HD * 4 + 16;            // an O row in shared memory (over Q and the ring)
    static_assert(TILES * kURows * kPitch <= kQ + kSlots * kSlot, "O rows fit where Q and the ring were");
};

// D[tmem] = A[tmem] * B + (accumulate ? D : 0); issued by one thread.
SDL_DEV void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        :: "r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}

// True in one thread of a converged warp.  Warp-uniform loops around an elected
// issue let the compiler keep descriptors in uniform registers: eight MMAs
// issue in 115-180 cycles, against 480 from a thread that runs alone.
SDL_DEV bool elect_one() {
    uint32_t on;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
    return on != 0;
}

// Maximum of three, a NaN among them included (fmaxf would drop it).
SDL_DEV float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 2^x of a pair on the FMA pipe, for 16-bit weights: x = n + f with n the
// nearest integer (adding 1.5 * 2^23 + 127 leaves n + 127 in the low mantissa
// bits) and |f| <= 1/2, 2^f by the degree-4 minimax polynomial of that interval
// (relative error 2^-18.4 in fp32, fitted with the Remez exchange), times 2^n,
// whose exponent field is n + 127.  x is clamped at -127, where that field, and
// the weight, is zero: a masked key weighs nothing, whatever its value is.  So
// does a NaN (the caller's running maximum carries those).
SDL_DEV void ex2_poly2(float& a, float& b) {
    constexpr float kMagic = 12582912.f + 127.f;
    const uint64_t magic = pack_f32x2(kMagic, kMagic), minus = pack_f32x2(-kMagic, -kMagic);
    const uint64_t neg = pack_f32x2(-1.f, -1.f);
    const uint64_t x = pack_f32x2(fmaxf(a, -127.f), fmaxf(b, -127.f));
    const uint64_t t = add_f32x2(x, magic);
    const uint64_t f = fma_f32x2(add_f32x2(t, minus), neg, x);
    uint64_t r = pack_f32x2(0.009570102f, 0.009570102f);
    r = fma_f32x2(r, f, pack_f32x2(0.05591786f, 0.05591786f));
    r = fma_f32x2(r, f, pack_f32x2(0.24024744f, 0.24024744f));
    r = fma_f32x2(r, f, pack_f32x2(0.6931218f, 0.6931218f));
    r = fma_f32x2(r, f, pack_f32x2(0.9999993f, 0.9999993f));
    float t0, t1;
    unpack_f32x2(t, t0, t1);
    r = fma_f32x2(r, pack_f32x2(__int_as_float(__float_as_int(t0) << 23), __int_as_float(__float_as_int(t1) << 23)), 0ull);
    unpack_f32x2(r, a, b);
}

template <int HD, typename T, int TILES, bool kOwn>
__global__ void __launch_bounds__(256 * TILES, 3 - TILES)
prefix_umma_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const PfxParams p,
                   const int behind) {
    using C = UCfg<HD, TILES>;
    constexpr int DO = C::DO, NSL = C::kSlots, kMine = C::kMine;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    constexpr uint32_t kIdescS = umma_idesc_f16(kURows, kUKeys, kBf16, false);
    constexpr uint32_t kIdescO = umma_idesc_f16(kURows, HD, kBf16, true);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sKV = smem + C::kQ;
    __shared__ uint64_t kv_full[NSL], kv_empty[NSL], q_full[TILES], s_full[TILES][2], p_full[TILES][2],
        pv_done[TILES][2], s_end[TILES], pv_end, v_zeroed;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort_flag;
    volatile int* s_abort = &s_abort_flag;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    Item it;
    pfx_enter(behind);
    if (kOwn) {
        if (!pfx_item(p, (int64_t)p.ptiles * p.Hkv * p.nsp + blockIdx.x, it)) {
            pfx_leave(behind);
            return;
        }
    } else {
        // row tiles fastest (they share their keys in L2), kv heads, key ranges
        it.g = blockIdx.x / p.ptiles % p.Hkv;
        it.slot = blockIdx.x / p.ptiles / p.Hkv;
        it.f0 = blockIdx.x % p.ptiles * (TILES * kURows);
        it.f1 = min(p.F, it.f0 + TILES * kURows);
        it.k0 = it.slot * p.ppk;
        it.k1 = min(p.prefix_len, it.k0 + p.ppk);
        it.seq = p.prefix_row;
    }
    const int g = it.g, f0 = it.f0, k0 = it.k0, k1 = it.k1;
    const int nt = (it.f1 - f0 + kURows - 1) / kURows;  // row tiles of this item
    const int nk = (k1 - k0 + kUKeys - 1) / kUKeys;     // key steps (>= 1)

    if (threadIdx.x == 0) {
        *s_abort = 0;
        for (int i = 0; i < NSL; ++i) {
            mbar_init(&kv_full[i], C::kProducers);
            mbar_init(&kv_empty[i], nt);
        }
        for (int t = 0; t < TILES; ++t) {
            mbar_init(&s_end[t], 1);
            mbar_init(&q_full[t], 4);
            for (int x = 0; x < 2; ++x) {
                mbar_init(&s_full[t][x], 1);
                mbar_init(&p_full[t][x], 4);
                mbar_init(&pv_done[t][x], 1);
            }
        }
        mbar_init(&pv_end, nt);
        mbar_init(&v_zeroed, 4);
        fence_mbar_init();
        prefetch_tmap(&tmk);
        prefetch_tmap(&tmv);
    }
    if (warp == C::kMmaS) {
        tmem_alloc(&s_tmem, C::kTmemCols);
        tmem_relinquish();
    }
    // Before the barrier that publishes TMEM: the producers' first page-table
    // read, and the copies of Q.
    const int u0 = (warp - C::kProducer) * kMine;
    const int npages = (k1 - k0 + kPage - 1) / kPage;
    auto read_pages = [&](int i0) {  // 32 pages from step i0; past the range its last one (masked keys)
        const int pg = (i0 + lane / kMine) * kUPages + u0 + lane % kMine;
        return (int)pfx_page_row(p, it.seq, k0 / kPage + min(pg, npages - 1));
    };
    int tok = 0;
    if (warp >= C::kProducer && warp < C::kMmaS) tok = read_pages(0);
    const int m = 32 * (warp & 3) + lane;  // softmax warps: the thread's row within tile warp / 4
    FlatRow fr = {};
    bool live = false;
    if (warp < 4 * nt) {
        const int t = warp >> 2, f = f0 + t * kURows + m;
        fr = kOwn ? pfx_row(p, min(f, p.F - 1), g) : pfx_prefix_row(p, min(f, p.F - 1), g);
        live = f < it.f1 && fr.valid;
        // Q rows into the swizzled K-major layout: HD / 8 lanes copy one row
        const T* qrow = reinterpret_cast<const T*>(p.q) + fr.b * p.q_sb + fr.j * p.q_sj + fr.h * p.q_sh;
        constexpr int kLanes = HD / 8;  // 16-byte chunks of a row
        const int c = lane % kLanes;
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += 32 / kLanes) {
            const int r = r0 + lane / kLanes;
            const T* src =
                reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(qrow), r));
            const bool on = __shfl_sync(0xffffffffu, live ? 1 : 0, r);
            const int row = 32 * (warp & 3) + r;
            uint8_t* dst = smem + (t * DO + (c >> 3)) * C::kQHalf + row * 128 + (((c & 7) ^ (row & 7)) << 4);
            if (on) cp_async16(dst, src + 8 * c);
            else *reinterpret_cast<uint4*>(dst) = make_uint4(0u, 0u, 0u, 0u);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    if (warp >= 4 * TILES) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kUHelpRegs));
        // bounded wait of a whole warp
        auto wait = [&](uint64_t* bar, int phase) {
            if (__all_sync(0xffffffffu, mbar_wait_bounded(bar, phase & 1, kWaitLimit))) return true;
            if (lane == 0) {
                sdl_raise(p.err, SDL_DEVERR_TIMEOUT);
                *s_abort = 1;
            }
            return false;
        };
        if (warp < C::kMmaS) {
            // -------------------------------------------------- producers
            int issued = 0;
            bool ok = true;
            for (int i0 = 0; i0 < nk && ok; i0 += 32 / kMine) {  // one page-table read for 32 pages
                if (i0 > 0) tok = read_pages(i0);
                for (int n = 2 * i0; n < min(2 * nk, 2 * (i0 + 32 / kMine)); ++n) {  // K tiles (even), V tiles (odd)
                    const int st = n % NSL;
                    int tu[kMine];
#pragma unroll
                    for (int u = 0; u < kMine; ++u) tu[u] = __shfl_sync(0xffffffffu, tok, ((n >> 1) - i0) * kMine + u);
                    if (n >= NSL && !(ok = wait(&kv_empty[st], (n / NSL) - 1))) break;
                    if (elect_one()) {
                        mbar_arrive_expect_tx(&kv_full[st], kMine * DO * kBox);
                        const CUtensorMap* tm = (n & 1) ? &tmv : &tmk;
#pragma unroll
                        for (int u = 0; u < kMine; ++u)
#pragma unroll
                            for (int dd = 0; dd < DO; ++dd)
                                tma_load_4d(sKV + st * C::kSlot + dd * C::kHalf + (u0 + u) * kBox, tm, &kv_full[st], 0,
                                            dd, g, tu[u]);
                    }
                    __syncwarp();
                    issued = n + 1;
                }
            }
            // never leave the CTA with bulk copies still landing in shared memory
            for (int n = max(0, issued - NSL); n < issued; ++n)
                (void)mbar_wait_bounded(&kv_full[n % NSL], (n / NSL) & 1, kWaitLimit);
        } else if (warp < C::kMmaPV && warp - C::kMmaS < nt) {
            // ------------------------------------------------ S_t = Q_t K^T
            const int t = warp - C::kMmaS;
            const uint64_t dQ = umma_desc_sw128(smem_u32(smem) + t * DO * C::kQHalf, 16, 1024);
            const uint64_t dK = umma_desc_sw128(smem_u32(sKV), 16, 1024);
            bool ok = wait(&q_full[t], 0);
            for (int i = 0; i < nk && ok; ++i) {
                const int n = 2 * i, st = n % NSL;
                ok = wait(&kv_full[st], n / NSL) && (i < 2 || wait(&pv_done[t][i & 1], (i >> 1) - 1));
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        const uint32_t qo = (k >> 2) * C::kQHalf + (k & 3) * 32;
                        const uint32_t ko = st * C::kSlot + (k >> 2) * C::kHalf + (k & 3) * 32;
                        umma_f16(tmem + (2 * t + (i & 1)) * kUKeys, dQ + (qo >> 4), dK + (ko >> 4), kIdescS,
                                 k > 0 ? 1u : 0u);
                    }
                    umma_commit(&s_full[t][i & 1]);
                    umma_commit(&kv_empty[st]);
                    if (i == nk - 1) umma_commit(&s_end[t]);
                }
                __syncwarp();
            }
            // every issued MMA completes before TMEM is released
            if (!ok && elect_one()) umma_commit(&s_end[t]);
            __syncwarp();
            (void)mbar_wait_bounded(&s_end[t], 0, kWaitLimit);
        } else if (warp >= C::kMmaPV && warp - C::kMmaPV < nt) {
            // ------------------------------------------------- O_t += P_t V
            const int t = warp - C::kMmaPV;
            const uint64_t dV = umma_desc_sw128(smem_u32(sKV), C::kHalf, 1024);
            bool ok = true;
            for (int i = 0; i < nk && ok; ++i) {
                const int n = 2 * i + 1, st = n % NSL;
                ok = wait(&kv_full[st], n / NSL) && wait(&p_full[t][i & 1], i >> 1);
                if (ok && (i + 1) * kUKeys > k1 - k0) ok = wait(&v_zeroed, 0);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < kUKeys / 16; ++k) {
                        const uint32_t vo = st * C::kSlot + k * 2048;
                        umma_f16_ts(tmem + C::kOCol + t * 128, tmem + (2 * t + (i & 1)) * kUKeys + 8 * k, dV + (vo >> 4),
                                    kIdescO, (i > 0 || k > 0) ? 1u : 0u);
                    }
                    umma_commit(&pv_done[t][i & 1]);
                    umma_commit(&kv_empty[st]);
                    if (i == nk - 1) umma_commit(&pv_end);
                }
                __syncwarp();
            }
            if (!ok && elect_one()) umma_commit(&pv_end);
            __syncwarp();
            (void)mbar_wait_bounded(&pv_end, 0, kWaitLimit);
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kUSoftRegs));
        const int t = warp >> 2;
        if (t < nt) {
            // ---------------------------------------------------- softmax
            const int f = f0 + t * kURows + m;
            const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
            const uint32_t tS = tmem + lanes + 2 * t * kUKeys, tO = tmem + lanes + C::kOCol + t * 128;
            cp_async_wait_all();
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[t]);
            // rows that are not attended keep the tile's limit (finite values, never stored)
            const int lim = kOwn && live ? min(fr.limit, k1) : k1;
            bool ok = true;
            float m_run = -INFINITY, l_run = 0.f;
            for (int i = 0; i < nk; ++i) {
                ok = __all_sync(0xffffffffu, mbar_wait_bounded(&s_full[t][i & 1], (i >> 1) & 1, kWaitLimit));
                if (!ok) break;
                tc_fence_after();
                float s[kUKeys];
#pragma unroll
                for (int c = 0; c < kUKeys; c += 32)
                    tmem_ld32(tS + (i & 1) * kUKeys + c, reinterpret_cast<uint32_t*>(s + c));
                tmem_wait_ld();
                const int left = k1 - k0 - i * kUKeys;         // keys of this step (any row)
                const int mine = kOwn ? lim - k0 - i * kUKeys : left;  // those this row attends
                if (kOwn ? __any_sync(0xffffffffu, mine < kUKeys) : mine < kUKeys) {
#pragma unroll
                    for (int c = 0; c < kUKeys; ++c) s[c] = c < mine ? s[c] : -INFINITY;
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < kUKeys; c += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = max3_nan(mx[e], s[c + e], s[c + e + 4]);
                float tmax = max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]) * p.scale_log2;
                // a NaN or infinite score makes the maximum, and with it the row, NaN
                const bool need = !(tmax <= m_run + kLazyLog2);
                if (__any_sync(0xffffffffu, need)) {
                    tmax += need ? tmax - tmax : 0.f;
                    const float alpha = need ? ex2_approx(m_run - tmax) : 1.f;  // 0 on the first keys
                    if (need) m_run = tmax;
                    l_run *= alpha;
                    if (i > 0) {  // rescale O_t once PV_t(i - 1) has landed
                        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&pv_done[t][(i - 1) & 1], ((i - 1) >> 1) & 1,
                                                                       kWaitLimit));
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (int c = 0; c < HD; c += 32) {
                            uint32_t o[32];
                            tmem_ld32(tO + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                            tmem_st32(tO + c, o);
                        }
                    }
                }
                if (t == 0 && left < kUKeys) {
                    // V rows past the range are zeroed (0 * stale NaN is NaN)
                    // before any PV of this last step
                    const int st = (2 * i + 1) % NSL;
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(&kv_full[st], ((2 * i + 1) / NSL) & 1, kWaitLimit));
                    if (!ok) break;
                    for (int x = threadIdx.x; x < (kUKeys - left) * DO * 8; x += 128) {
                        const int row = left + x / (DO * 8), c = x % (DO * 8);
                        *reinterpret_cast<uint4*>(sKV + st * C::kSlot + (c >> 3) * C::kHalf + row * 128 +
                                                  ((c & 7) << 4)) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&v_zeroed);
                }
                const float base = m_run == -INFINITY ? 0.f : m_run;
                const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2), base2 = pack_f32x2(-base, -base);
                uint64_t sum2[2] = {0ull, 0ull};
                uint32_t w[kUKeys / 2];
#pragma unroll
                for (int e = 0; e < kUKeys / 2; ++e) {
                    float p0, p1;
                    unpack_f32x2(fma_f32x2(pack_f32x2(s[2 * e], s[2 * e + 1]), scale2, base2), p0, p1);
                    // one pair of four on the FMA pipe, as the special function
                    // unit needs 8 cycles for a warp's value (16 x 96 rows
                    // behind 6000 keys: none 92 us, 1/8 93, 1/4 90, 3/8 92,
                    // 1/2 95; 256 x 6 behind 16384: 188, 187, 188, 193, 195)
                    if ((e & 3) == 1) {
                        ex2_poly2(p0, p1);
                    } else {
                        p0 = ex2_approx(p0);
                        p1 = ex2_approx(p1);
                    }
                    sum2[e & 1] = add_f32x2(sum2[e & 1], pack_f32x2(p0, p1));
                    w[e] = pack2<T>(p0, p1);  // rounded once: as the output's own rounding
                }
                tmem_st32(tS + (i & 1) * kUKeys, w);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t][i & 1]);
                float a0, a1, b0, b1;
                unpack_f32x2(sum2[0], a0, a1);
                unpack_f32x2(sum2[1], b0, b1);
                l_run += (a0 + a1) + (b0 + b1);
            }
            // Every PV (and so every S) of the item: Q and the ring are free.
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait_bounded(&pv_end, 0, kWaitLimit) && !*s_abort);
            if (ok) {
                tc_fence_after();
                // O rows leave through shared memory: a thread holds a row, a
                // warp's store writes whole rows (nslot rows apart)
                const int64_t idx = ((int64_t)g * p.F + f) * p.nslot + it.slot;
                constexpr int kPitch = C::kPitch;
                uint8_t* so = smem + (t * kURows + 32 * (warp & 3)) * kPitch;
#pragma unroll
                for (int c = 0; c < HD; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(tO + c, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        *reinterpret_cast<uint4*>(so + lane * kPitch + c * 4 + e * 16) =
                            make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                }
                if (live) *reinterpret_cast<float2*>(p.ml_part + idx * 2) = make_float2(m_run, l_run);
                __syncwarp();
                constexpr int kLanes = HD / 4;  // 16-byte pieces of a row
                const uint32_t on = __ballot_sync(0xffffffffu, live);
                const int r0 = lane / kLanes, pc = lane % kLanes;
                // flat rows lie nslot partial rows apart
                const int64_t first = __shfl_sync(0xffffffffu, idx, 0);
                float* dst = p.o_part + (first + (int64_t)r0 * p.nslot) * HD + pc * 4;
                const uint8_t* src = so + r0 * kPitch + pc * 16;
                const int64_t step = (int64_t)(32 / kLanes) * p.nslot * HD;
#pragma unroll 8
                for (int r = r0; r < 32; r += 32 / kLanes) {
                    const uint4 v = *reinterpret_cast<const uint4*>(src);
                    if (on >> r & 1) *reinterpret_cast<uint4*>(dst) = v;
                    dst += step;
                    src += 32 / kLanes * kPitch;
                }
            } else if (lane == 0) {
                sdl_raise(p.err, SDL_DEVERR_TIMEOUT);
                *s_abort = 1;
            }
        }
    }
    pfx_leave(behind);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == C::kMmaS) tmem_dealloc(tmem, C::kTmemCols);
}

// -------------------------------------------------------------------- merge
// A row reads its prefix slots and the own slots that start below its limit;
// they lie side by side.  A slot whose keys it does not attend holds m = -inf
// and weighs 0.  HD / 4 lanes take a row (16 bytes of every slot each), four
// slots at a time with all loads in flight before the first use, in a running
// softmax.  Where no sequence has more than a page of own keys (own_direct), it
// attends them here, four keys at a time, in place of a launch whose items
// would last longer than their keys (105 decode rows of 32 / 8 heads with 2 to 4
// own keys behind 2707: 21.6 us, 25.8 with 840 own items).  WARPS = 1: a warp
// takes whole rows; WARPS = 4 (many slots, few rows): a block's warps share a
// row's slots and join in shared memory.
constexpr int kMergeWarps = 4;
constexpr int kMergeMany = 12;  // slots from which a row takes four warps

SDL_DEV void store4(const PfxParams& p, int64_t at, float4 a, float inv) {
    a = make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv);
    if (!p.out_vec) {
        store_from_f32(p.out, at, p.out_dtype, a.x);
        store_from_f32(p.out, at + 1, p.out_dtype, a.y);
        store_from_f32(p.out, at + 2, p.out_dtype, a.z);
        store_from_f32(p.out, at + 3, p.out_dtype, a.w);
    } else if (p.out_dtype == SDL_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = a;
    } else {
        const uint2 v = p.out_dtype == SDL_BF16
                            ? make_uint2(pack2<__nv_bfloat16>(a.x, a.y), pack2<__nv_bfloat16>(a.z, a.w))
                            : make_uint2(pack2<__half>(a.x, a.y), pack2<__half>(a.z, a.w));
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = v;
    }
}

template <typename T> SDL_DEV float half_of(uint32_t v, int i) { return to_f32<T>(reinterpret_cast<const T*>(&v)[i]); }

struct MergeState {
    float m, l;
    float4 o;
};

SDL_DEV void merge_in(MergeState& s, float m, float l, float4 o) {
    const float mn = fmaxf(s.m, m);
    const float base = mn == -INFINITY ? 0.f : mn;
    const float a = ex2_approx(s.m - base), b = ex2_approx(m - base);
    s.m = mn;
    s.l = s.l * a + l * b;
    s.o.x = s.o.x * a + o.x * b;
    s.o.y = s.o.y * a + o.y * b;
    s.o.z = s.o.z * a + o.z * b;
    s.o.w = s.o.w * a + o.w * b;
}

// Four 16-bit elements.
SDL_DEV float4 half4(uint2 v, int dtype) {
    if (dtype == SDL_BF16)
        return make_float4(half_of<__nv_bfloat16>(v.x, 0), half_of<__nv_bfloat16>(v.x, 1), half_of<__nv_bfloat16>(v.y, 0),
                           half_of<__nv_bfloat16>(v.y, 1));
    return make_float4(half_of<__half>(v.x, 0), half_of<__half>(v.x, 1), half_of<__half>(v.y, 0), half_of<__half>(v.y, 1));
}

// The own keys of one row, `first` and every `step` groups of four from there:
// LANES lanes hold the row's dims, four each.
template <int LANES>
SDL_DEV void merge_own(const PfxParams& p, const FlatRow& r, int g, int d0, int first, int step, MergeState& s) {
    constexpr int U = 4;
    const uint32_t group = LANES == 32 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16);  // the row's lanes
    const int n = r.limit;
    if (first >= n) return;
    const int64_t at = (pfx_page_row(p, p.rows[r.b], 0) * p.Hkv + g) * p.hd + d0;
    const uint16_t* k = reinterpret_cast<const uint16_t*>(p.k_pool) + at;
    const uint16_t* v = reinterpret_cast<const uint16_t*>(p.v_pool) + at;
    const float4 q = half4(*reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p.q) + r.b * p.q_sb +
                                                           r.j * p.q_sj + r.h * p.q_sh + d0), p.dtype);
    for (int k0 = first; k0 < n; k0 += U * step) {
        uint2 kx[U], vx[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (k0 + u < n) {
                kx[u] = *reinterpret_cast<const uint2*>(k + (int64_t)(k0 + u) * p.Hkv * p.hd);
                vx[u] = *reinterpret_cast<const uint2*>(v + (int64_t)(k0 + u) * p.Hkv * p.hd);
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k0 + u >= n) break;
            const float4 kf = half4(kx[u], p.dtype);
            float dot = q.x * kf.x + q.y * kf.y + q.z * kf.z + q.w * kf.w;
#pragma unroll
            for (int w = LANES / 2; w > 0; w >>= 1) dot += __shfl_xor_sync(group, dot, w);
            merge_in(s, dot * p.scale_log2, 1.f, half4(vx[u], p.dtype));
        }
    }
}

// The slots of row w from `first`, `per` side by side, every `step`, once more,
// its own ranges key by key.  An item multiplies every V row of its keys by every
// query row's weights, and the weight 0 of a key behind a row's limit times an
// infinity or a NaN is not 0: a row whose values came out so while its sum did
// not is joined again without the keys that it does not attend.  `lanes` lanes
// hold the row, dims d0 + i * dstep each.
template <int ND>
SDL_DEV void merge_again(const PfxParams& p, const FlatRow& r, int g, int64_t w, int ns, int first, int per, int step,
                         int d0, int dstep, int lanes, uint32_t group, float& m, float& l, float (&o)[ND]) {
    float q[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) {
        const int d = d0 + i * dstep;
        q[i] = d < p.hd ? load_as_f32(p.q, r.b * p.q_sb + r.j * p.q_sj + r.h * p.q_sh + d, p.dtype) : 0.f;
        o[i] = 0.f;
    }
    m = -INFINITY;
    l = 0.f;
    auto join = [&](float mx, float mul, const float* x) {
        const float mn = fmaxf(m, mx);
        const float base = mn == -INFINITY ? 0.f : mn;
        const float a = ex2_approx(m - base), b = ex2_approx(mx - base);
        m = mn;
        l = l * a + mul * b;
#pragma unroll
        for (int i = 0; i < ND; ++i) o[i] = o[i] * a + x[i] * b;
    };
    float x[ND];
#pragma unroll 1
    for (int s0 = first; s0 < ns; s0 += step)
#pragma unroll 1
        for (int s = s0; s < min(ns, s0 + per); ++s) {
            if (s < p.nsp) {
                const int64_t at = w * p.nslot + s;
#pragma unroll
                for (int i = 0; i < ND; ++i) {
                    const int d = d0 + i * dstep;
                    x[i] = d < p.hd ? p.o_part[at * p.hd + d] : 0.f;
                }
                join(p.ml_part[at * 2], p.ml_part[at * 2 + 1], x);
                continue;
            }
            const int k0 = (s - p.nsp) * p.mpk, k1 = min(r.limit, k0 + p.mpk);
#pragma unroll 1
            for (int key = k0; key < k1; ++key) {
                const int64_t tok = pfx_page_row(p, p.rows[r.b], key / p.block_size) + key % p.block_size;
                const int64_t at = (tok * p.Hkv + g) * p.hd;
                float dot = 0.f;
#pragma unroll
                for (int i = 0; i < ND; ++i) {
                    const int d = d0 + i * dstep;
                    x[i] = d < p.hd ? load_as_f32(p.v_pool, at + d, p.dtype) : 0.f;
                    if (d < p.hd) dot = fmaf(q[i], load_as_f32(p.k_pool, at + d, p.dtype), dot);
                }
                for (int x2 = lanes / 2; x2 > 0; x2 >>= 1) dot += __shfl_xor_sync(group, dot, x2);
                join(dot * p.scale_log2, 1.f, x);
            }
        }
}

// 1 / l; no keys give zeros, a NaN stays one.
SDL_DEV float merge_inv(float l) { return l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l); }

template <int LANES, int WARPS>
__global__ void __launch_bounds__(kMergeWarps * 32) prefix_merge_kernel(const __grid_constant__ PfxParams p) {
    constexpr int HD = 4 * LANES, U = 4;
    __shared__ float s_part[WARPS > 1 ? kMergeWarps : 1][WARPS > 1 ? HD + 2 : 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int kRows = WARPS > 1 ? 1 : 32 / LANES;  // rows of a warp
    const int64_t w = WARPS > 1 ? (int64_t)blockIdx.x
                                : ((int64_t)blockIdx.x * kMergeWarps + warp) * kRows + lane / LANES;
    const bool in = w < (int64_t)p.F * p.Hkv;
    const int g = in ? (int)(w / p.F) : 0, f = in ? (int)(w - (int64_t)g * p.F) : 0;
    if (p.nsp + p.nsm == 0) pdl_wait();  // no items: the call's first kernel
    const FlatRow r = pfx_row(p, f, g);
    const int ns = in && r.valid ? p.nsp + min(p.nsm, (r.limit + p.mpk - 1) / p.mpk) : 0;  // nsm 0 with own_direct
    if (in && r.valid && r.over && lane % LANES == 0) sdl_raise(p.err, SDL_DEVERR_BAD_INDEX);
    // the row's metadata was read under the items' tail: whatever wrote it was
    // complete before they ran; the partials only now
    pdl_wait();
    pdl_launch_dependents();
    if (WARPS == 1 && !(in && r.valid)) return;
    const int d0 = (lane % LANES) * 4;
    const float* op = p.o_part + w * p.nslot * HD + d0;
    const float2* mlp = reinterpret_cast<const float2*>(p.ml_part) + w * p.nslot;
    // a row of half a warp leaves the other half idle where four warps share it
    const bool mine = WARPS == 1 || lane < LANES;
    MergeState s = {-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
    if (mine) {
        for (int s0 = WARPS > 1 ? warp * U : 0; s0 < ns; s0 += U * WARPS) {
            float2 ml[U];
            float4 o[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                ml[u] = make_float2(-INFINITY, 0.f);
                o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (s0 + u < ns) {
                    ml[u] = mlp[s0 + u];
                    o[u] = *reinterpret_cast<const float4*>(op + (int64_t)(s0 + u) * HD);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) merge_in(s, ml[u].x, ml[u].y, o[u]);
        }
        const float any = s.o.x + s.o.y + s.o.z + s.o.w;
        const uint32_t group = LANES == 32 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16);  // the row's lanes
        if (ns > p.nsp && s.l == s.l && __any_sync(group, !(any - any == 0.f))) {
            float o[4];
            merge_again<4>(p, r, g, w, ns, WARPS > 1 ? warp * U : 0, U, U * WARPS, d0, 1, LANES, group, s.m, s.l, o);
            s.o = make_float4(o[0], o[1], o[2], o[3]);
        }
        if (p.own_direct && r.valid) merge_own<LANES>(p, r, g, d0, WARPS > 1 ? warp * U : 0, WARPS, s);
    }
    const int64_t ob = r.b * p.o_sb + r.j * p.o_sj + r.h * p.o_sh + d0;
    if (WARPS == 1) {
        store4(p, ob, s.o, merge_inv(s.l));
        return;
    }
    if (mine) {
        *reinterpret_cast<float2*>(&s_part[warp][d0]) = make_float2(s.o.x, s.o.y);
        *reinterpret_cast<float2*>(&s_part[warp][d0 + 2]) = make_float2(s.o.z, s.o.w);
        if (lane == 0) *reinterpret_cast<float2*>(&s_part[warp][HD]) = make_float2(s.m, s.l);
    }
    __syncthreads();
    if (warp > 0 || !mine || !r.valid) return;
#pragma unroll
    for (int x = 1; x < kMergeWarps; ++x)
        merge_in(s, s_part[x][HD], s_part[x][HD + 1],
                 make_float4(s_part[x][d0], s_part[x][d0 + 1], s_part[x][d0 + 2], s_part[x][d0 + 3]));
    store4(p, ob, s.o, merge_inv(s.l));
}

// Any head_dim: one warp per row, a lane per dim.
__global__ void __launch_bounds__(kMergeWarps * 32) prefix_merge_any_kernel(const __grid_constant__ PfxParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * kMergeWarps + (threadIdx.x >> 5);
    if (w >= (int64_t)p.F * p.Hkv) return;
    const int g = (int)(w / p.F), f = (int)(w - (int64_t)g * p.F);
    const FlatRow r = pfx_row(p, f, g);
    if (!r.valid) return;
    if (r.over && lane == 0) sdl_raise(p.err, SDL_DEVERR_BAD_INDEX);
    const int ns = p.nsp + min(p.nsm, (r.limit + p.mpk - 1) / p.mpk);
    const int64_t idx0 = w * p.nslot;
    float M = -INFINITY;
    for (int s = lane; s < ns; s += 32) M = fmaxf(M, p.ml_part[(idx0 + s) * 2]);
    M = warp_max(M);
    const float base = M == -INFINITY ? 0.f : M;
    float den = 0.f;
    for (int s = lane; s < ns; s += 32) den += ex2_approx(p.ml_part[(idx0 + s) * 2] - base) * p.ml_part[(idx0 + s) * 2 + 1];
    den = warp_sum(den);
    constexpr int ND = 8;  // head_dim <= 256
    float o[ND];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < ND; ++i) {
        const int d = lane + 32 * i;
        if (d >= p.hd) break;
        float acc = 0.f;
#pragma unroll 4
        for (int s = 0; s < ns; ++s)
            acc = fmaf(ex2_approx(p.ml_part[(idx0 + s) * 2] - base), p.o_part[(idx0 + s) * p.hd + d], acc);
        o[i] = acc;
        bad = bad || !(acc - acc == 0.f);
    }
    if (ns > p.nsp && den == den && __any_sync(0xffffffffu, bad))
        merge_again<ND>(p, r, g, w, ns, 0, ns, ns, lane, 32, 32, 0xffffffffu, M, den, o);
    const float inv = merge_inv(den);
    const int64_t ob = r.b * p.o_sb + r.j * p.o_sj + r.h * p.o_sh;
#pragma unroll
    for (int i = 0; i < ND; ++i)
        if (lane + 32 * i < p.hd) store_from_f32(p.out, ob + lane + 32 * i, p.out_dtype, o[i] * inv);
}

// --------------------------------------------------------------------- host
struct Plan {
    int kernel = 1;
    int ptile = 0;          // plan 3: rows of a prefix item
    bool own_umma = false;  // plan 3: own items on the tcgen05 kernel too
    bool wide_pre = false, wide_own = false;  // plan 1: the wide form for prefix / own items
    PfxParams p = {};
    int64_t items = 0;
    size_t ws_bytes = 0;
};

int invalid(const char* msg) { return sdl::fail(SDL_ERR_INVALID, (std::string("sdl_prefix_attention: ") + msg).c_str()); }
int unsupported(const char* msg) {
    return sdl::fail(SDL_ERR_UNSUPPORTED, (std::string("sdl_prefix_attention: ") + msg).c_str());
}

int validate(const sdl_prefix_args* x) {
    if (!x) return invalid("args is NULL");
    const sdl_attn_args* a = &x->attn;
    if (a->B < 0 || a->chunk < 1 || a->Hq < 1 || a->Hkv < 1 || a->Hq % a->Hkv || a->head_dim < 1 || a->head_dim > 256)
        return invalid("bad shape arguments");
    if (a->dtype != SDL_F32 && a->dtype != SDL_BF16 && a->dtype != SDL_F16) return unsupported("unsupported dtype");
    if (a->out_dtype != SDL_F32 && a->out_dtype != SDL_BF16 && a->out_dtype != SDL_F16)
        return unsupported("unsupported out dtype");
    if (!a->k_pool || !a->v_pool || !a->block_table || a->width < 1 || a->capacity < 1 || a->block_size < 1 ||
        a->layer < 0 || a->layer >= a->num_layers)
        return invalid("a paged pool with its block table is needed");
    if (a->k_new || a->v_new || a->rope_cos || a->rope_sin || a->k_dense || a->v_dense)
        return unsupported("k_new, RoPE and dense K/V are not taken (append first)");
    if (a->B > 0 && (!a->q || !a->out || !a->rows || !a->starts)) return invalid("q, out, rows or starts is NULL");
    if (x->table_rows < 1 || (x->prefix_len > 0 && x->prefix_row >= x->table_rows))
        return invalid("the prefix is not a row of the block table");
    if (x->prefix_row < 0 || x->prefix_len < 0 || x->kernel < 0 || x->kernel > 3 || x->prefix_split < 0 ||
        x->own_split < 0)
        return invalid("bad prefix or plan arguments");
    if ((int64_t)x->prefix_len > (int64_t)a->width * a->block_size) return invalid("the prefix exceeds the block table");
    if ((int64_t)a->max_limit > (int64_t)a->width * a->block_size) return invalid("max_limit exceeds the block table");
    if ((int64_t)a->num_layers * a->capacity * a->block_size >= (int64_t(1) << 31))
        return unsupported("pool exceeds 2^31 token rows");
    if ((int64_t)std::max(1, a->B) * a->chunk * (a->Hq / a->Hkv) >= (int64_t(1) << 30))
        return unsupported("too many query rows");
    if (x->prefix_len >= 1 << 30 || a->max_limit >= 1 << 30) return unsupported("more than 2^30 keys");
    // the running maxima are taken of the unscaled scores
    if (!(a->scale > 0.f) || !std::isfinite(a->scale * kLog2e)) return invalid("scale must be positive and finite");
    return SDL_OK;
}

int cdiv(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }
int round_up(int64_t a, int64_t b) { return (int)((a + b - 1) / b * b); }

bool aligned(const void* x, size_t n) { return reinterpret_cast<uintptr_t>(x) % n == 0; }

// Whether the tensor-core kernels take these arguments: 16-bit pools of
// 16-token pages and q rows on 16-byte boundaries (TMA and 16-byte loads).
bool tensor_cores_apply(const sdl_attn_args* a) {
    if ((a->dtype != SDL_BF16 && a->dtype != SDL_F16) || (a->head_dim != 64 && a->head_dim != 128) ||
        a->block_size != kPage || !aligned(a->k_pool, 16) || !aligned(a->v_pool, 16) || !aligned(a->q, 16))
        return false;
    return (a->q_sb | a->q_sj | a->q_sh) % 8 == 0;
}

constexpr int kSms = 148;
constexpr int64_t kOwnPartials = int64_t(1) << 30;  // bytes of partials from which own ranges are not cut further
constexpr int kMaxSmem = 225 * 1024;  // dynamic shared memory of a block beside 2 KB of static

// Keys per prefix range of the tcgen05 kernel: the number of ranges with the
// least cost, in ns.  `slots` CTAs are resident (two per SM, or one of the
// 256-row form, beside which an own item counts half); a prefix item costs 6500
// + 12.5 per key, an own item 4000 + 12 per key.  Prefix items run in waves;
// own items fill what they leave, and begin late where the slots do not hold
// all.  Every range writes, and the merge reads, a partial of `elems` fp32
// values in all, at about 6 bytes per ps and 50 ns of latency.  (Fitted to sweeps; 64
// decode rows behind 8192 keys with up to 1024 own: 512 keys 20.9 us, 384 24.8,
// 1024 24.1; 16 x 96 rows behind 6000: 2048 91 us, 1024 113, 6000 100.)
int umma_prefix_split(int prefix, int64_t tiles, bool big, int64_t elems, int64_t own_items, int64_t own_keys) {
    const int64_t slots = big ? kSms : 2 * kSms;
    const int64_t own = big ? (own_items + 1) / 2 : own_items, t_own = own_items ? 4000 + 12 * own_keys : 0;
    int best = kUKeys;
    int64_t least = INT64_MAX;
    for (int n = 1; n <= 64; ++n) {
        const int keys = round_up(cdiv(prefix, n), kUKeys);
        const int64_t ranges = cdiv(prefix, keys), items = tiles * ranges;
        const int64_t t_item = 6500 + 25 * (int64_t)keys / 2;
        const int64_t waves = (items + slots - 1) / slots * t_item;
        const int64_t all = items + own <= slots
                                ? std::max(t_item, t_own)
                                : std::max(waves, (items * t_item + own * t_own) / slots + std::min(t_item, t_own));
        const int64_t cost = all + ranges * (elems * 8 / 6000 + 50);
        if (cost < least) {
            least = cost;
            best = keys;
        }
    }
    return best;
}

// Whether the prefix goes to the tcgen05 kernel, a launch more than mma.sync
// alone: wherever the rows are more than one mma.sync operand holds (24 rows x
// 2 kv heads, d 128, behind 256 keys: 10.2 us with mma.sync, 8.8 with tcgen05;
// 28 x 2, d 64: 7.5 and 6.7), and fewer rows only over a long prefix in many
// heads (4 x 8, d 128, behind 4096 keys: 8.7 and 10.0; behind 16384: 22.6 and
// 19.0; at d 64, 15.1 and 15.6).
bool tcgen05_pays(const sdl_prefix_args* x) {
    const sdl_attn_args* a = &x->attn;
    const int64_t rows = (int64_t)a->B * a->chunk * (a->Hq / a->Hkv), keys = (int64_t)x->prefix_len * a->Hkv;
    if (keys == 0 || a->out_dtype == SDL_F32) return false;
    return rows > 16 || (a->head_dim == 128 && keys >= 100000);
}

int make_plan(const sdl_prefix_args* x, Plan& pl) {
    const sdl_attn_args* a = &x->attn;
    const bool tc = tensor_cores_apply(a);
    if (x->kernel >= 2 && !tc) return unsupported("this kernel does not take these arguments");
    if (x->kernel == 3 && (x->prefix_len == 0 || a->out_dtype == SDL_F32))
        return unsupported("the tcgen05 kernel needs a prefix and 16-bit output");
    pl.kernel = x->kernel ? x->kernel : !tc ? 1 : tcgen05_pays(x) ? 3 : 2;
    PfxParams& p = pl.p;
    p.q = a->q; p.q_sb = a->q_sb; p.q_sj = a->q_sj; p.q_sh = a->q_sh;
    p.out = a->out; p.o_sb = a->o_sb; p.o_sj = a->o_sj; p.o_sh = a->o_sh;
    p.out_dtype = a->out_dtype; p.dtype = a->dtype;
    p.k_pool = static_cast<const char*>(a->k_pool); p.v_pool = static_cast<const char*>(a->v_pool);
    p.table = a->block_table; p.width = a->width; p.capacity = a->capacity; p.layer = a->layer;
    p.block_size = a->block_size; p.table_rows = x->table_rows;
    p.rows = a->rows; p.starts = a->starts; p.valid_rows = a->valid_rows;
    p.prefix_row = x->prefix_row; p.prefix_len = x->prefix_len;
    p.max_limit = std::max(0, a->max_limit);
    p.B = a->B; p.chunk = a->chunk; p.Hq = a->Hq; p.Hkv = a->Hkv; p.ratio = a->Hq / a->Hkv; p.hd = a->head_dim;
    p.scale_log2 = a->scale * kLog2e;
    p.err = a->err;
    p.p_split = a->out_dtype == SDL_F32;
    p.out_vec = ((a->o_sb | a->o_sj | a->o_sh) % 4 == 0) && aligned(a->out, 4 * sdl::dtype_bytes(a->out_dtype));
    p.F = a->B * a->chunk * p.ratio;
    // own items of more rows than one mma.sync operand holds take the tcgen05
    // kernel: mma.sync runs them at an eighth of its rate
    pl.own_umma = pl.kernel == 3 && a->chunk * p.ratio > 16;
    pl.wide_own = pl.kernel == 1 && a->chunk * p.ratio >= 48;
    pl.wide_pre = pl.kernel == 1 && p.F >= 48;
    p.row_tile = pl.kernel == 1 ? (pl.wide_own ? kWideRows : kGenRows) : pl.own_umma ? kURows : kMmaRows;
    // Prefix items of 256 rows share their K and V, which pays where they fill
    // the SMs at head_dim 128; otherwise items of 128 rows at two CTAs per SM mix
    // with the own items on every SM (us with 128 / 256 rows: 32 x 6 verify
    // rows, 10 items of 256, 19.2 / 21.8; 160 x 6, 46 items, 49.7 / 49.6; 256 x 6
    // behind 16384 keys, 72 items, 194 / 188; at d 64, 300 x 6, 100 items, 71.3 /
    // 74.7).
    if (pl.kernel == 3) {
        pl.ptile = p.hd == 128 && (int64_t)cdiv(p.F, 2 * kURows) * p.Hkv >= 64 ? 2 * kURows : kURows;
    } else {
        pl.ptile = pl.wide_pre ? kWideRows : p.row_tile;
    }
    p.ptile = pl.ptile;
    p.ptiles = cdiv(p.F, pl.ptile);
    p.mtiles = cdiv(a->chunk * p.ratio, p.row_tile);
    const int64_t ptiles = (int64_t)p.ptiles * p.Hkv;
    const int64_t mtiles = (int64_t)p.mtiles * p.Hkv * std::max(1, a->B);
    const int span = p.max_limit;
    // mean own keys of a sequence (the bound where the host gives no count)
    const int64_t mean = a->key_count > 0 && a->B > 0 ? std::min<int64_t>(span, a->key_count / a->B + 1) : span;
    const int page = pl.kernel == 1 ? 1 : kPage;
    // At most a page of own keys each: in the merge, where own items would fill
    // more than a wave and the rows are not many (us in the merge / as items, behind
    // 2000 keys: 500 decode rows x 12 heads 24.8 / 33.5; 32 x 8 rows x 12 heads,
    // 64 items, 20.3 / 17.4; 60 x 8 x 32, 480 items, 46.7 / 43.3.  The row limit
    // is too low for decode: 1600 rows x 8 heads, d 64, 30.9 / 81.5).
    const bool own_direct = pl.kernel >= 2 && span > 0 && span <= kPage && !x->own_split && mtiles > 2 * kSms &&
                            (int64_t)p.F * p.Hkv <= 8192;
    if (pl.kernel == 1) {
        // CUDA cores: about eight blocks per SM, ranges of at least 64 keys
        const int64_t keys = (ptiles * x->prefix_len + mtiles * mean) / (kSms * 8);
        p.ppk = p.mpk = round_up(std::max<int64_t>(64, std::min<int64_t>(std::max(x->prefix_len, span), keys)), kWideKeys);
    } else {
        // own keys: one item per SM where sequences are few, in bounded ranges.
        // mma.sync (64 decode rows of 1..1024 own keys behind 8192: 512 20.6 us,
        // 256 23.9, 1024 25.6); tcgen05 (32 x 6 rows of 1..512 behind 4001: 256
        // 19.2 us, 128 24.1, 512 20.9; 256 x 6 of 64..1024 behind 16384: 1024 190,
        // 512 193, 256 207)
        const int64_t least = pl.own_umma ? 256 : 128, most = pl.own_umma ? 1024 : 512;
        p.mpk = round_up(std::max(least, std::min(most, mtiles * mean / kSms)), kStageKeys);
        const int64_t keys = ptiles * x->prefix_len + mtiles * mean;
        if (pl.kernel == 3) {
            // own items with keys: ragged lengths fill half a range more than their mean
            const int64_t own = span == 0 || own_direct ? 0 : span <= p.mpk ? mtiles : mtiles * (2 * mean + p.mpk) / (2 * p.mpk);
            p.ppk = umma_prefix_split(x->prefix_len, ptiles, pl.ptile == 2 * kURows, (int64_t)p.F * p.Hkv * a->head_dim,
                                      own, std::min<int64_t>(mean, p.mpk));
        } else {
            // two waves of two CTAs per SM, at least three or four stages (2
            // rows x 2 heads behind 2000 keys: 192 6.6 us, 256 7.2, 512 10.4;
            // behind 8000: 256 8.4, 192 7.7, 128 7.5)
            p.ppk = round_up(std::max<int64_t>((x->prefix_len <= 4096 ? 3 : 4) * kStageKeys, std::min<int64_t>(x->prefix_len, keys / (kSms * 4))),
                             kStageKeys);
        }
    }
    // Own ranges are bounded above, however many rows there are; where their
    // partials would pass 1 GiB the rows alone fill the SMs many times over, and
    // the ranges grow instead (256 x 128 rows of 32 heads with up to 32768 own
    // keys: 0.5 GiB in one range, 17 in ranges of 1024).
    const int64_t range = (int64_t)p.F * p.Hkv * (p.hd + 2) * (int64_t)sizeof(float);
    if (cdiv(span, p.mpk) * range > kOwnPartials)
        p.mpk = round_up(cdiv(span, std::max<int64_t>(1, kOwnPartials / range)), kStageKeys);
    if (x->prefix_split) p.ppk = round_up(std::min(x->prefix_split, 1 << 29), page);
    if (x->own_split) p.mpk = round_up(std::min(x->own_split, 1 << 29), page);
    p.nsp = cdiv(x->prefix_len, p.ppk);
    p.nsm = cdiv(span, p.mpk);
    if (own_direct) {
        p.own_direct = span;
        p.nsm = 0;
    }
    p.nslot = std::max(1, p.nsp + p.nsm);
    pl.items = ptiles * p.nsp + mtiles * p.nsm;
    if (pl.items > INT_MAX || (int64_t)p.F * p.Hkv > INT_MAX - 8) return unsupported("grid too large");
    const size_t rows = (size_t)p.F * p.Hkv * p.nslot;
    pl.ws_bytes = rows * (size_t)(p.hd + 2) * sizeof(float);
    return SDL_OK;
}

// Raises a kernel's dynamic shared memory limit once per device (`ready`: one
// bit per device; devices past 63 pay the call every time).
template <typename K>
bool smem_opt_in(K* kern, int smem, std::atomic<uint64_t>& ready) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (ready.load(std::memory_order_relaxed) & bit) return true;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return false;
    ready.fetch_or(bit, std::memory_order_relaxed);
    return true;
}

template <typename K>
int launch_cores(K* kern, size_t smem, std::atomic<uint64_t>& ready, const Plan& pl, int64_t item0, int64_t items,
                 bool behind, cudaStream_t st) {
    if (smem > 48 * 1024 && !smem_opt_in(kern, kMaxSmem, ready))
        return sdl::fail(SDL_ERR_CUDA, "sdl_prefix_attention: shared memory opt-in failed");
    const cudaError_t e = sdl::launch_pdl(kern, dim3((unsigned)items), dim3(kGenThreads), smem, st, pl.p, item0,
                                          behind ? 1 : 0);
    return e == cudaSuccess ? (int)SDL_OK : sdl::fail(SDL_ERR_CUDA, cudaGetErrorString(e));
}

template <typename T, int ND>
int launch_generic(const Plan& pl, int64_t item0, int64_t items, bool behind, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    return launch_cores(prefix_generic_kernel<T, ND>, gen_smem(pl.p.hd), ready, pl, item0, items, behind, st);
}

template <typename T, int NC>
int launch_wide(const Plan& pl, int64_t item0, int64_t items, bool behind, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    return launch_cores(prefix_wide_kernel<T, NC>, wide_smem(NC), ready, pl, item0, items, behind, st);
}

template <typename T>
int launch_items(const Plan& pl, bool wide, int64_t item0, int64_t items, bool behind, cudaStream_t st) {
    const int hd = pl.p.hd;
    if (items == 0) return SDL_OK;
    if (wide) {
        if (hd <= 32) return launch_wide<T, 1>(pl, item0, items, behind, st);
        if (hd <= 64) return launch_wide<T, 2>(pl, item0, items, behind, st);
        if (hd <= 128) return launch_wide<T, 4>(pl, item0, items, behind, st);
        return launch_wide<T, 8>(pl, item0, items, behind, st);
    }
    if (hd <= 64) return launch_generic<T, 8>(pl, item0, items, behind, st);
    if (hd <= 128) return launch_generic<T, 16>(pl, item0, items, behind, st);
    return launch_generic<T, 32>(pl, item0, items, behind, st);
}

template <typename T>
int launch_generic_dtype(const Plan& pl, cudaStream_t st) {
    const int64_t pre = (int64_t)pl.p.ptiles * pl.p.Hkv * pl.p.nsp;
    if (pl.wide_pre == pl.wide_own) return launch_items<T>(pl, pl.wide_own, 0, pl.items, false, st);
    const int rc = launch_items<T>(pl, pl.wide_pre, 0, pre, false, st);
    return rc != SDL_OK ? rc : launch_items<T>(pl, pl.wide_own, pre, pl.items - pre, pre > 0, st);
}

// Tensor maps of the pools: the caller's, or encoded here.
int pool_maps(const sdl_attn_args* a, CUtensorMap& mk, CUtensorMap& mv) {
    const int64_t ntok = (int64_t)a->num_layers * a->capacity * a->block_size;
    if (a->tmap_k && a->tmap_v) {
        memcpy(&mk, a->tmap_k, sizeof(mk));
        memcpy(&mv, a->tmap_v, sizeof(mv));
        return SDL_OK;
    }
    int rc = sdl_make_kv_tensor_map(&mk, a->k_pool, a->dtype, ntok, a->Hkv, a->head_dim);
    if (rc == SDL_OK) rc = sdl_make_kv_tensor_map(&mv, a->v_pool, a->dtype, ntok, a->Hkv, a->head_dim);
    return rc;
}

template <int HD, typename T>
int launch_mma(const Plan& pl, const CUtensorMap& mk, const CUtensorMap& mv, int64_t item0, bool behind,
               cudaStream_t st) {
    constexpr int smem = MmaCfg<HD>::kSmem;
    static std::atomic<uint64_t> ready{0};
    if (!smem_opt_in(prefix_mma_kernel<HD, T>, smem, ready))
        return sdl::fail(SDL_ERR_CUDA, "sdl_prefix_attention: shared memory opt-in failed");
    const cudaError_t e = sdl::launch_pdl(prefix_mma_kernel<HD, T>, dim3((unsigned)(pl.items - item0)),
                                          dim3(kMmaThreads), smem, st, mk, mv, pl.p, item0, behind ? 1 : 0);
    return e == cudaSuccess ? (int)SDL_OK : sdl::fail(SDL_ERR_CUDA, cudaGetErrorString(e));
}

// The tcgen05 kernel over the prefix (TILES = 2) or the own items (1).
template <int HD, typename T, int TILES, bool kOwn>
int launch_umma(const Plan& pl, const CUtensorMap& mk, const CUtensorMap& mv, int64_t grid, bool behind,
                cudaStream_t st) {
    using C = UCfg<HD, TILES>;
    static std::atomic<uint64_t> ready{0};
    if (!smem_opt_in(prefix_umma_kernel<HD, T, TILES, kOwn>, C::kSmem, ready))
        return sdl::fail(SDL_ERR_CUDA, "sdl_prefix_attention: shared memory opt-in failed");
    const cudaError_t e = sdl::launch_pdl(prefix_umma_kernel<HD, T, TILES, kOwn>, dim3((unsigned)grid), dim3(C::kThreads),
                                          C::kSmem, st, mk, mv, pl.p, behind ? 1 : 0);
    return e == cudaSuccess ? (int)SDL_OK : sdl::fail(SDL_ERR_CUDA, cudaGetErrorString(e));
}

template <typename T>
int launch_tensor(const Plan& pl, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
    // the tcgen05 kernel takes the prefix items of plan 3, and its own items where a sequence has enough rows
    const int64_t pre = pl.kernel == 3 ? (int64_t)pl.p.ptiles * pl.p.Hkv * pl.p.nsp : 0;
    const int64_t own = pl.items - pre;
    const bool d128 = pl.p.hd == 128;
    int rc = SDL_OK;
    if (pre > 0 && pl.ptile == kURows)
        rc = d128 ? launch_umma<128, T, 1, false>(pl, mk, mv, pre, false, st)
                  : launch_umma<64, T, 1, false>(pl, mk, mv, pre, false, st);
    else if (pre > 0)
        rc = launch_umma<128, T, 2, false>(pl, mk, mv, pre, false, st);
    if (rc != SDL_OK || own == 0) return rc;
    if (pl.own_umma)
        return d128 ? launch_umma<128, T, 1, true>(pl, mk, mv, own, pre > 0, st)
                    : launch_umma<64, T, 1, true>(pl, mk, mv, own, pre > 0, st);
    return d128 ? launch_mma<128, T>(pl, mk, mv, pre, pre > 0, st) : launch_mma<64, T>(pl, mk, mv, pre, pre > 0, st);
}

int launch_merge(const Plan& pl, cudaStream_t st) {
    const PfxParams& p = pl.p;
    const int64_t rows = (int64_t)p.F * p.Hkv;
    // few rows spread over more warps earlier (32 x 6 verify rows stand on the
    // border: 19.0 us in all, 18.4 with one warp a row)
    const bool many = p.nslot >= kMergeMany || (p.nslot >= 5 && p.hd == 128 && rows <= 4096);
    const int per = kMergeWarps * (p.hd == 64 ? 2 : 1);  // rows of a block
    const dim3 grid((unsigned)((p.hd == 64 || p.hd == 128) && many ? rows : (rows + per - 1) / per));
    const dim3 block(kMergeWarps * 32);
    cudaError_t e;
    if (p.hd == 128) {
        e = many ? sdl::launch_pdl(prefix_merge_kernel<32, kMergeWarps>, grid, block, 0, st, p)
                 : sdl::launch_pdl(prefix_merge_kernel<32, 1>, grid, block, 0, st, p);
    } else if (p.hd == 64) {
        e = many ? sdl::launch_pdl(prefix_merge_kernel<16, kMergeWarps>, grid, block, 0, st, p)
                 : sdl::launch_pdl(prefix_merge_kernel<16, 1>, grid, block, 0, st, p);
    } else {
        e = sdl::launch_pdl(prefix_merge_any_kernel, grid, block, 0, st, p);
    }
    return e == cudaSuccess ? (int)SDL_OK : sdl::fail(SDL_ERR_CUDA, cudaGetErrorString(e));
}

}  // namespace

extern "C" size_t sdl_prefix_attention_workspace_bytes(const sdl_prefix_args* args) {
    Plan pl;
    if (validate(args) != SDL_OK || make_plan(args, pl) != SDL_OK) return 0;
    return pl.ws_bytes;
}

extern "C" int sdl_prefix_attention_kernel(const sdl_prefix_args* args) {
    Plan pl;
    if (validate(args) != SDL_OK || make_plan(args, pl) != SDL_OK) return -1;
    return pl.kernel;
}

extern "C" int sdl_prefix_attention(const sdl_prefix_args* args, void* stream) {
    Plan pl;
    int rc = validate(args);
    if (rc != SDL_OK || (rc = make_plan(args, pl)) != SDL_OK) return rc;
    if (args->attn.B == 0) return SDL_OK;
    if (pl.ws_bytes > args->attn.workspace_bytes || !args->attn.workspace ||
        reinterpret_cast<uintptr_t>(args->attn.workspace) % 16)
        return sdl::fail(SDL_ERR_WORKSPACE, "sdl_prefix_attention: workspace too small or not 16-byte aligned");
    PfxParams& p = pl.p;
    // O first (16-byte rows where head_dim allows), then the (m, l) pairs
    p.o_part = args->attn.workspace;
    p.ml_part = p.o_part + (size_t)p.F * p.Hkv * p.nslot * p.hd;
    cudaStream_t st = sdl::as_stream(stream);
    if (pl.items > 0 && pl.kernel >= 2) {
        CUtensorMap mk, mv;
        if ((rc = pool_maps(&args->attn, mk, mv)) != SDL_OK) return rc;
        rc = p.dtype == SDL_BF16 ? launch_tensor<__nv_bfloat16>(pl, mk, mv, st) : launch_tensor<__half>(pl, mk, mv, st);
        if (rc != SDL_OK) return rc;
    } else if (pl.items > 0) {
        if (p.dtype == SDL_BF16) rc = launch_generic_dtype<__nv_bfloat16>(pl, st);
        else if (p.dtype == SDL_F16) rc = launch_generic_dtype<__half>(pl, st);
        else rc = launch_generic_dtype<float>(pl, st);
        if (rc != SDL_OK) return rc;
    }
    return launch_merge(pl, st);
}
