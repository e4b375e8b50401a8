// Rotate-half RoPE of q and k rows straight from a position table, with one
// position per axis, and the same fused with the append to the paged pool.
//
// For a row at positions p_0 .. p_{A-1} and pair i (0 <= i < R/2, R = the
// rotary dims, dims i and i + R/2), with a(i) the axis whose section holds i
// and (c, s) = table[p_a(i)][0/1][i]:
//   y_i        = x_i c - x_{i+R/2} s
//   y_{i+R/2}  = x_{i+R/2} c + x_i s
// in fp32, rounded once; dims past R are copied.  (sdl_rope instead takes
// gathered 16-bit cos / sin rows and keeps the framework chain's roundings.)
//
// Bound by memory: each q / k / v element is read once and written once (a
// 16-byte piece in flight for 4 heads x 2 halves a thread), and a row's R/2 cos
// and sin values once per thread, from L1 or L2.  A thread owns one 16-byte
// piece of the first rotary half and its partner piece R/2 dims on, so the
// pairs meet in its registers, and applies its 8 (4 in fp32) angles to
// kHeadsPerThread heads, whose loads are all in flight before the first use.
// v's heads and the dims past R ride along as plain 16-byte copies.
#include "sdl_common.cuh"

#include <algorithm>
#include <climits>

namespace {

constexpr int kMaxAxes = 4;
constexpr int kHeadsPerThread = 4;

struct RopeParams {
    const char* q;   // [T][Hq][d], row strides below in bytes; NULL = none
    const char* k;   // [T][Hkv][d]; NULL = none
    const char* v;   // [T][Hkv][d]; NULL = none (rotation only)
    char* q_out;
    char* k_out;     // row outputs of the rotation-only form
    int64_t q_rs, k_rs, v_rs, qo_rs, ko_rs;
    char* k_pool;    // append form: rows of Hkv*d at `slot`; NULL = rotation only
    char* v_pool;
    const int32_t* slots;
    int64_t num_slots;     // capacity * block_size of one layer (the pools point at it)
    const float* table;    // [table_rows][2][R]
    int64_t table_rows;
    const void* positions; // [A][T]
    int64_t pos_stride;    // elements between axes
    int pos64;             // positions are int64 (else int32)
    int axes;
    int sec_end[kMaxAxes]; // exclusive end of each axis' section, in pairs
    int T, hq, hkv, d, R;
    int32_t* err;
};

SDL_DEV int64_t rope_position(const RopeParams& p, int axis, int t) {
    const int64_t at = (int64_t)axis * p.pos_stride + t;
    return p.pos64 ? static_cast<const int64_t*>(p.positions)[at]
                   : (int64_t) static_cast<const int32_t*>(p.positions)[at];
}

SDL_DEV int axis_of_pair(const RopeParams& p, int pair) {
    int a = 0;
#pragma unroll
    for (int i = 0; i < kMaxAxes - 1; ++i)
        if (i < p.axes - 1 && pair >= p.sec_end[i]) a = i + 1;
    return a;
}

// cos / sin of `n` consecutive pairs from `pair`; false when a position lies
// outside the table (the angles of its pairs are then NaN).
template <int n>
SDL_DEV bool load_angles(const RopeParams& p, int t, int pair, float (&c)[n], float (&s)[n]) {
    const int a0 = axis_of_pair(p, pair);
    const float nan = __int_as_float(0x7fc00000);
    bool ok = true;
    if (a0 == axis_of_pair(p, pair + n - 1)) {
        const int64_t pos = rope_position(p, a0, t);
        ok = pos >= 0 && pos < p.table_rows;
        if (!ok) {
#pragma unroll
            for (int e = 0; e < n; ++e) c[e] = s[e] = nan;
        } else {
            const float* row = p.table + pos * 2 * p.R + pair;
#pragma unroll
            for (int e = 0; e < n; e += 4) {
                const float4 cv = __ldg(reinterpret_cast<const float4*>(row + e));
                const float4 sv = __ldg(reinterpret_cast<const float4*>(row + p.R + e));
                c[e] = cv.x; c[e + 1] = cv.y; c[e + 2] = cv.z; c[e + 3] = cv.w;
                s[e] = sv.x; s[e + 1] = sv.y; s[e + 2] = sv.z; s[e + 3] = sv.w;
            }
        }
    } else {  // a section ends inside the piece
#pragma unroll
        for (int e = 0; e < n; ++e) {
            const int64_t pos = rope_position(p, axis_of_pair(p, pair + e), t);
            const bool in = pos >= 0 && pos < p.table_rows;
            ok = ok && in;
            c[e] = in ? __ldg(p.table + pos * 2 * p.R + pair + e) : nan;
            s[e] = in ? __ldg(p.table + (pos * 2 + 1) * p.R + pair + e) : nan;
        }
    }
    return ok;
}

// Rotates one pair: returns (x c - y s, y c + x s).
SDL_DEV float2 turn(float x, float y, float c, float s) {
    return make_float2(fmaf(x, c, -(y * s)), fmaf(y, c, x * s));
}

template <typename T>
SDL_DEV void turn_piece(uint4& lo, uint4& hi, const float (&c)[16 / sizeof(T)], const float (&s)[16 / sizeof(T)]) {
    if constexpr (sizeof(T) == 4) {
        float* a = reinterpret_cast<float*>(&lo);
        float* b = reinterpret_cast<float*>(&hi);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 r = turn(a[e], b[e], c[e], s[e]);
            a[e] = r.x;
            b[e] = r.y;
        }
    } else {
        uint32_t* a = reinterpret_cast<uint32_t*>(&lo);
        uint32_t* b = reinterpret_cast<uint32_t*>(&hi);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const T* at = reinterpret_cast<const T*>(&a[w]);
            const T* bt = reinterpret_cast<const T*>(&b[w]);
            const float2 r0 = turn(to_f32<T>(at[0]), to_f32<T>(bt[0]), c[2 * w], s[2 * w]);
            const float2 r1 = turn(to_f32<T>(at[1]), to_f32<T>(bt[1]), c[2 * w + 1], s[2 * w + 1]);
            a[w] = pack2<T>(r0.x, r1.x);
            b[w] = pack2<T>(r0.y, r1.y);
        }
    }
}

// Where row t of head h (q heads, then k heads, then v heads) is read.
SDL_DEV const char* head_src(const RopeParams& p, int t, int h, int64_t hb) {
    if (h < p.hq) return p.q + t * p.q_rs + h * hb;
    h -= p.hq;
    return h < p.hkv ? p.k + t * p.k_rs + h * hb : p.v + t * p.v_rs + (h - p.hkv) * hb;
}

// ... and written; NULL = not written (`slot` negative).
SDL_DEV char* head_dst(const RopeParams& p, int t, int h, int64_t hb, int64_t slot) {
    if (h < p.hq) return p.q_out + t * p.qo_rs + h * hb;
    h -= p.hq;
    if (!p.k_pool) return p.k_out + t * p.ko_rs + h * hb;
    if (slot < 0) return nullptr;
    return h < p.hkv ? p.k_pool + (slot * p.hkv + h) * hb : p.v_pool + (slot * p.hkv + h - p.hkv) * hb;
}

SDL_DEV bool head_turns(const RopeParams& p, int h) { return h < p.hq + p.hkv; }

// The row's slot: -1 = padding (nothing stored, q comes out zero), -2 = the
// slot lies outside the pool (reported, nothing stored).
SDL_DEV int64_t row_slot(const RopeParams& p, int t, bool report) {
    if (!p.k_pool) return 0;
    const int64_t slot = p.slots[t];
    if (slot < 0) return -1;
    if (slot >= p.num_slots) {
        if (report) sdl_raise(p.err, SDL_DEVERR_BAD_SLOT);
        return -2;
    }
    return slot;
}

// Block (pieces, head groups, tokens): see the file comment.  Pieces past the
// rotary half copy two 16-byte pieces of the dims past R.  A row's data is in
// flight before its positions and table rows are read.  Three blocks per SM (80
// registers) and streaming loads and stores, as a call touches each byte once
// (20250 rows of 32 + 8 heads, d 128: 68.5 us, 0.95 of a copy's rate; 81.5 with
// two blocks.  Append of 17946 rows of 12 + 2 + 2 heads, a sixth of them
// padding: 24.8 us; 27.6 without the streaming hints, 28.9 loading the padding
// rows too).
template <typename T>
__global__ void __launch_bounds__(256, 3) rope_vec_kernel(const RopeParams p) {
    constexpr int VE = 16 / (int)sizeof(T);
    pdl_wait();
    pdl_launch_dependents();
    const int t = blockIdx.x * blockDim.z + threadIdx.z;
    if (t >= p.T) return;
    const int x = threadIdx.x;
    const int half_pieces = p.R / 2 / VE;
    const int nheads = p.hq + (p.v ? 2 : 1) * p.hkv;
    const int64_t hb = (int64_t)p.d * (int)sizeof(T);
    const bool first = x == 0 && threadIdx.y == 0;
    const bool turning = x < half_pieces;
    // byte offsets of this thread's two pieces within a head
    const int off0 = (turning ? x : p.R / VE + 2 * (x - half_pieces)) * 16;
    const int off1 = turning ? off0 + half_pieces * 16 : off0 + 16;
    const bool two = turning || off1 < p.d * (int)sizeof(T);

    const int64_t slot = row_slot(p, t, first);
    uint4 a[kHeadsPerThread], b[kHeadsPerThread];
#pragma unroll
    for (int u = 0; u < kHeadsPerThread; ++u) {
        const int h = threadIdx.y + u * blockDim.y;
        if (h < nheads && slot != -1) {
            const char* src = head_src(p, t, h, hb);
            a[u] = __ldcs(reinterpret_cast<const uint4*>(src + off0));
            if (two) b[u] = __ldcs(reinterpret_cast<const uint4*>(src + off1));
        }
    }
    const bool pad = slot == -1;
    float c[VE], s[VE];
    bool ok = true;
    if (!pad) {
        if (turning) ok = load_angles<VE>(p, t, x * VE, c, s);
        if (p.k_pool)  // a row any of whose positions is bad stores nothing
            for (int ax = 0; ax < p.axes; ++ax) {
                const int64_t pos = rope_position(p, ax, t);
                ok = ok && pos >= 0 && pos < p.table_rows;
            }
        if (!ok && threadIdx.y == 0) sdl_raise(p.err, SDL_DEVERR_BAD_INDEX);
    }
#pragma unroll
    for (int u = 0; u < kHeadsPerThread; ++u) {
        const int h = threadIdx.y + u * blockDim.y;
        if (h >= nheads) continue;
        char* dst = head_dst(p, t, h, hb, slot);
        if (dst == nullptr || (p.k_pool && !ok && h >= p.hq)) continue;
        if (pad) a[u] = b[u] = make_uint4(0u, 0u, 0u, 0u);  // q rows only: the others have no dst
        else if (turning && head_turns(p, h)) turn_piece<T>(a[u], b[u], c, s);
        __stcs(reinterpret_cast<uint4*>(dst + off0), a[u]);
        if (two) __stcs(reinterpret_cast<uint4*>(dst + off1), b[u]);
    }
}

// Any alignment, head_dim and rotary width: one thread per pair or copied dim
// of one head of one row.
template <typename T>
__global__ void __launch_bounds__(256) rope_scalar_kernel(const RopeParams p) {
    pdl_wait();
    pdl_launch_dependents();
    const int nheads = p.hq + (p.v ? 2 : 1) * p.hkv;
    const int half = p.R / 2;
    const int per = half + (p.d - p.R);  // pairs, then copied dims
    const int64_t total = (int64_t)p.T * nheads * per;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int e = (int)(i % per);
        const int h = (int)(i / per % nheads);
        const int t = (int)(i / per / nheads);
        const bool first = e == 0 && h == 0;
        const int64_t slot = row_slot(p, t, first);
        const int64_t hb = (int64_t)p.d * (int)sizeof(T);
        const bool pad = slot == -1;
        bool ok = true;
        if (!pad && p.k_pool)
            for (int ax = 0; ax < p.axes; ++ax) {
                const int64_t pos = rope_position(p, ax, t);
                ok = ok && pos >= 0 && pos < p.table_rows;
            }
        if (!ok && first) sdl_raise(p.err, SDL_DEVERR_BAD_INDEX);
        const T* src = reinterpret_cast<const T*>(head_src(p, t, h, hb));
        T* dst = reinterpret_cast<T*>(head_dst(p, t, h, hb, slot));
        if (dst == nullptr || (p.k_pool && !ok && h >= p.hq)) continue;
        const int e0 = e < half ? e : e + half;
        if (pad) {
            dst[e0] = from_f32<T>(0.f);
            if (e < half) dst[e0 + half] = from_f32<T>(0.f);
        } else if (e < half && head_turns(p, h)) {
            const int64_t pos = rope_position(p, axis_of_pair(p, e), t);
            const bool in = pos >= 0 && pos < p.table_rows;
            if (!in && h == 0) sdl_raise(p.err, SDL_DEVERR_BAD_INDEX);
            const float c = in ? __ldg(p.table + pos * 2 * p.R + e) : __int_as_float(0x7fc00000);
            const float s = in ? __ldg(p.table + (pos * 2 + 1) * p.R + e) : __int_as_float(0x7fc00000);
            const float2 r = turn(to_f32<T>(src[e]), to_f32<T>(src[e + half]), c, s);
            dst[e] = from_f32<T>(r.x);
            dst[e + half] = from_f32<T>(r.y);
        } else {
            dst[e0] = src[e0];
            if (e < half) dst[e0 + half] = src[e0 + half];
        }
    }
}

bool al16(const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 == 0; }

// Whether every row, head and piece the call touches is 16-byte aligned.
bool vectorizable(const RopeParams& p, int es) {
    const int ve = 16 / es;
    if (p.R / 2 % ve || p.d % ve || !al16(p.table)) return false;
    if (p.q && (!al16(p.q) || !al16(p.q_out) || p.q_rs % 16 || p.qo_rs % 16)) return false;
    if (p.k && (!al16(p.k) || p.k_rs % 16)) return false;
    if (p.v && (!al16(p.v) || p.v_rs % 16)) return false;
    if (p.k_pool) {
        if (!al16(p.k_pool) || !al16(p.v_pool)) return false;
    } else if (p.k && (!al16(p.k_out) || p.ko_rs % 16)) {
        return false;
    }
    const int pieces = p.R / 2 / ve + ((p.d - p.R) / ve + 1) / 2;
    const int nheads = p.hq + (p.v ? 2 : 1) * p.hkv;
    const int groups = (nheads + kHeadsPerThread - 1) / kHeadsPerThread;
    return pieces * groups <= 256;
}

template <typename T>
int launch_rope(const RopeParams& p, cudaStream_t st, const char* what) {
    cudaError_t e;
    if (vectorizable(p, (int)sizeof(T))) {
        constexpr int VE = 16 / (int)sizeof(T);
        const int pieces = p.R / 2 / VE + ((p.d - p.R) / VE + 1) / 2;
        const int nheads = p.hq + (p.v ? 2 : 1) * p.hkv;
        const int groups = (nheads + kHeadsPerThread - 1) / kHeadsPerThread;
        const int tokens = std::max(1, std::min(64, 256 / (pieces * groups)));
        const dim3 block(pieces, groups, std::min(tokens, p.T));
        e = sdl::launch_pdl(rope_vec_kernel<T>, dim3((p.T + block.z - 1) / block.z), block, 0, st, p);
    } else {
        const int64_t per = p.R / 2 + (p.d - p.R);
        const int64_t total = (int64_t)p.T * (p.hq + (p.v ? 2 : 1) * p.hkv) * per;
        const int64_t blocks = std::min<int64_t>((total + 255) / 256, 148 * 32);
        e = sdl::launch_pdl(rope_scalar_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, st, p);
    }
    if (e != cudaSuccess) {
        sdl::set_last_error(std::string(what) + ": " + cudaGetErrorString(e));
        return (int)SDL_ERR_CUDA;
    }
    return (int)SDL_OK;
}

int run_rope(const sdl_rope_args* a, bool append, void* stream, const char* what) {
    auto bad = [&](sdl_status code, const char* msg) {
        sdl::set_last_error(std::string(what) + ": " + msg);
        return (int)code;
    };
    if (!a) return bad(SDL_ERR_INVALID, "args is NULL");
    if (a->dtype != SDL_F32 && a->dtype != SDL_BF16 && a->dtype != SDL_F16)
        return bad(SDL_ERR_UNSUPPORTED, "unsupported dtype");
    if (a->num_tokens < 0 || a->Hq < 0 || a->Hkv < 0 || a->head_dim < 1 || a->head_dim > 1024)
        return bad(SDL_ERR_INVALID, "bad shape arguments");
    if (a->num_tokens > INT_MAX - 64) return bad(SDL_ERR_UNSUPPORTED, "too many rows");  // of blocks of up to 64
    if (a->num_tokens == 0) return SDL_OK;
    if (!a->table || a->table_rows < 1 || a->rotary < 2 || a->rotary % 2 || a->rotary > a->head_dim)
        return bad(SDL_ERR_INVALID, "table needs rows of cos and sin over an even rotary width of at most head_dim");
    if (!a->positions || a->axes < 1 || a->axes > kMaxAxes)
        return bad(SDL_ERR_INVALID, "positions of one to four axes are needed");
    if ((a->Hq > 0) != (a->q != nullptr) || (a->q && !a->q_out)) return bad(SDL_ERR_INVALID, "q, q_out and Hq disagree");
    if (append ? (!a->k || !a->v || !a->k_pool || !a->v_pool || !a->slots || a->Hkv < 1 || a->num_layers < 1 ||
                  a->layer < 0 || a->layer >= a->num_layers || a->capacity < 1 || a->block_size < 1)
               : ((a->Hkv > 0) != (a->k != nullptr) || (a->k && !a->k_out) || (!a->k && !a->q)))
        return bad(SDL_ERR_INVALID, append ? "bad k, v, pool or slot arguments" : "k, k_out and Hkv disagree");
    const int es = sdl::dtype_bytes(a->dtype);
    RopeParams p = {};
    p.q = static_cast<const char*>(a->q);
    p.k = static_cast<const char*>(a->k);
    p.q_out = static_cast<char*>(a->q_out);
    p.q_rs = a->q_row_stride * es;
    p.qo_rs = a->q_out_row_stride * es;
    p.k_rs = a->k_row_stride * es;
    if (append) {
        const int64_t layer_bytes = (int64_t)a->layer * a->capacity * a->block_size * a->Hkv * a->head_dim * es;
        p.v = static_cast<const char*>(a->v);
        p.v_rs = a->v_row_stride * es;
        p.k_pool = static_cast<char*>(a->k_pool) + layer_bytes;
        p.v_pool = static_cast<char*>(a->v_pool) + layer_bytes;
        p.slots = a->slots;
        p.num_slots = (int64_t)a->capacity * a->block_size;
    } else {
        p.k_out = static_cast<char*>(a->k_out);
        p.ko_rs = a->k_out_row_stride * es;
    }
    p.table = a->table;
    p.table_rows = a->table_rows;
    p.positions = a->positions;
    p.pos_stride = a->pos_stride;
    p.pos64 = a->pos64;
    p.axes = a->axes;
    int end = 0;
    for (int i = 0; i < a->axes; ++i) {
        if (a->sections[i] < 0) return bad(SDL_ERR_INVALID, "a section is negative");
        end += a->sections[i];
        p.sec_end[i] = end;
    }
    if (end != a->rotary / 2) return bad(SDL_ERR_INVALID, "the sections must sum to half the rotary width");
    p.T = a->num_tokens;
    p.hq = a->Hq;
    p.hkv = a->Hkv;
    p.d = a->head_dim;
    p.R = a->rotary;
    p.err = a->err;
    cudaStream_t st = sdl::as_stream(stream);
    if (a->dtype == SDL_BF16) return launch_rope<__nv_bfloat16>(p, st, what);
    if (a->dtype == SDL_F16) return launch_rope<__half>(p, st, what);
    return launch_rope<float>(p, st, what);
}

}  // namespace

extern "C" int sdl_rope_axes(const sdl_rope_args* args, void* stream) {
    return run_rope(args, false, stream, "sdl_rope_axes");
}

extern "C" int sdl_kv_append_rotary(const sdl_rope_args* args, void* stream) {
    return run_rope(args, true, stream, "sdl_kv_append_rotary");
}
