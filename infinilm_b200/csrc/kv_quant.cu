// Writing the 8-bit key/value cache and reading it back.
//
// il_rope_store_quant: rotary encoding of q and k (pairs (i, i + rot/2), cos and sin times `mscale`), then k and v as codes into the page of the token's
// slot. The angle pos * inv_freq[i] is made and reduced in 64 bits (exact product, so a far position turns as it should), sine and
// cosine in 32; k is rounded once, from 32 bits to its code. qkv rows: [nh heads of q | nkv of k | nkv of v]; q goes to `q_out`, which
// may be the same place.
// il_kv_unpack: pages of requests as pages of bfloat16 or float32 values in the layout of the plain cache, [page][K, V][kv head][16][head_dim].
// Both are bound by memory: what they read and write is named at each kernel.
// Positions, entries, tables and lengths may come from the kernel in front (no caller vouches that they do not), so they are not declared __restrict__: such loads may be moved above the wait.
#include <algorithm>

#include "kv_quant.cuh"

// Angle of one pair: cos and sin, times mscale. The product is exact in 64 bits (24 bits by 31), the reduction by whole turns leaves an error near 1e-16 times the turns.
__device__ __forceinline__ void kvq_angle(int pos, float freq, float mscale, float* c, float* s) {
    const double a = (double)pos * (double)freq;
    const double turns = rint(a * 0.15915494309189535);        // 1 / (2 pi)
    const float r = (float)fma(turns, -2.4492935982947064e-16, fma(turns, -6.283185307179586, a));
    float sn, cs;
    sincosf(r, &sn, &cs);
    *c = cs * mscale, *s = sn * mscale;
}
// The products are rounded one by one, so that the code does not depend on how the compiler joins them.
__device__ __forceinline__ float kvq_lo(float x1, float x2, float c, float s) { return __fsub_rn(__fmul_rn(x1, c), __fmul_rn(x2, s)); }
__device__ __forceinline__ float kvq_hi(float x1, float x2, float c, float s) { return __fadd_rn(__fmul_rn(x2, c), __fmul_rn(x1, s)); }

template <typename TA> struct KvqEight { uint4 w[sizeof(TA) / 2]; };           // eight elements: one 16-byte load, or two
template <typename TA>
__device__ __forceinline__ KvqEight<TA> kvq_load8(const TA* p) {
    KvqEight<TA> v;
#pragma unroll
    for (int i = 0; i < (int)sizeof(TA) / 2; ++i) v.w[i] = reinterpret_cast<const uint4*>(p)[i];
    return v;
}
template <typename TA>
__device__ __forceinline__ void kvq_store8(TA* p, const float (&x)[8]) {
    KvqEight<TA> v;
    TA* e = reinterpret_cast<TA*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = il_from_f<TA>(x[i]);
#pragma unroll
    for (int i = 0; i < (int)sizeof(TA) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = v.w[i];
}
template <int KIND>
__device__ __forceinline__ uint2 kvq_codes8(const float (&x)[8], float f) {
    return make_uint2(kvq_codes4<KIND>(x[0] * f, x[1] * f, x[2] * f, x[3] * f), kvq_codes4<KIND>(x[4] * f, x[5] * f, x[6] * f, x[7] * f));
}

// Where the rotated pairs come in whole runs of eight: a lane takes 16 columns of a head, eight and the eight they turn with (or 16 neighbours of v and of what is
// not turned), PER lanes (a power of two) a head, which agree on the head's exponent by shuffles, 32 / PER heads of one token a warp at a time. A lane's columns are the same in every
// head, so its eight angles are made once; the lanes of a warp that need the same ones make them together. One pass, each element read once and written once; bound by
// memory, so what matters is loads under way: the next round's while one is worked on, no barrier, registers for four blocks an SM (more rounds ahead with fewer blocks: 65 to 78 us for
// what takes 61). `wpt`: warps a token, many where the tokens are few. 9,420 tokens, 32 heads on 8 of
// 128, bfloat16, us: 230 with a column a lane at a time, 103 with a block a token and its angles in shared memory, 43 so, 40 with two columns rotated an instruction.
constexpr int KVS_AHEAD = 1, KVS_WARPS = 148 * 16;
template <typename TA, int KIND, int PER>
__global__ void __launch_bounds__(256, 4) rope_store_quant_kernel(const TA* qkv, long long row_stride, TA* q_out, long long q_stride, const int* tok_pos,
                                                               const int* tok_entry, const int* block_table, int bt_stride,
                                                               unsigned char* cache, int T, int nh, int nkv, int hd, int rot, const float* __restrict__ inv_freq, float mscale,
                                                               int wpt) {
    constexpr int HEADS = 32 / PER, OWN = 8 / HEADS > 0 ? 8 / HEADS : 1;      // heads of a round, angles that a lane makes
    il_pdl_begin();
    const int lane = threadIdx.x & 31, j = lane % PER, g = lane / PER;
    const int gw = blockIdx.x * 8 + (threadIdx.x >> 5), t = gw / wpt, part = gw - t * wpt;
    if (t >= T) return;
    const int half = rot >> 1, pairs = rot >> 4, lanes = hd >> 4, rows = cache ? nh + 2 * nkv : nh, pos = tok_pos[t];
    const TA* row0 = qkv + t * row_stride;
    TA* to0 = q_out + t * q_stride;
    unsigned char* page = nullptr;                // kv head 0's record; null: not stored
    if (cache) {
        const int id = block_table[(size_t)tok_entry[t] * bt_stride + pos / KVQ_PAGE];
        if (id >= 0) page = cache + (size_t)id * nkv * kvq_record(hd);            // the host reserves every page a step touches; never write elsewhere
    }
    const int key = pos % KVQ_PAGE;
    KvqEight<TA> va[KVS_AHEAD], vb[KVS_AHEAD];
    const auto place = [&](int r, int& a, int& b) {           // columns a .. a + 7 and b .. b + 7
        const bool turns = r < nh + nkv && j < pairs;
        a = turns ? j * 8 : j * 16, b = turns ? a + half : a + 8;
        return turns;
    };
    const auto load = [&](int first) {
#pragma unroll
        for (int u = 0; u < KVS_AHEAD; ++u) {
            const int r = first + u * wpt * HEADS + g;
            int a, b;
            place(r, a, b);
            if (r < rows && j < lanes) va[u] = kvq_load8(row0 + (size_t)r * hd + a), vb[u] = kvq_load8(row0 + (size_t)r * hd + b);
        }
    };
    load(part * HEADS);                           // on their way while the angles are made
    il_f2 c[4], s[4];
    if (rot) {
        float co[OWN], so[OWN];
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
            const int at = j * 8 + (g * OWN + i) % 8;
            co[i] = so[i] = 0.f;
            if (j < pairs) kvq_angle(pos, inv_freq[at], mscale, &co[i], &so[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const int a = i / OWN * PER + j, b = (i + 1) / OWN * PER + j;
            c[i / 2] = il_f2_make(__shfl_sync(0xffffffffu, co[i % OWN], a), __shfl_sync(0xffffffffu, co[(i + 1) % OWN], b));
            s[i / 2] = il_f2_make(__shfl_sync(0xffffffffu, so[i % OWN], a), __shfl_sync(0xffffffffu, so[(i + 1) % OWN], b));
        }
    }
    for (int first = part * HEADS; first < rows; first += KVS_AHEAD * wpt * HEADS) {
        KvqEight<TA> wa[KVS_AHEAD], wb[KVS_AHEAD];
#pragma unroll
        for (int u = 0; u < KVS_AHEAD; ++u) wa[u] = va[u], wb[u] = vb[u];
        load(first + KVS_AHEAD * wpt * HEADS);
#pragma unroll
        for (int u = 0; u < KVS_AHEAD; ++u) {
            const int r0 = first + u * wpt * HEADS, r = r0 + g;
            if (r0 >= rows) break;
            const bool mine = r < rows && j < lanes;
            int a, b;
            const bool turns = place(r, a, b);
            float x[8], y[8];
            const TA *pa = reinterpret_cast<const TA*>(&wa[u]), *pb = reinterpret_cast<const TA*>(&wb[u]);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = il_to_f(pa[i]), y[i] = il_to_f(pb[i]);
            if (turns) {                          // (kvq_lo and kvq_hi, two at a time)
                const il_f2 minus = il_f2_dup(-1.f);
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const il_f2 x1 = il_f2_make(x[i], x[i + 1]), x2 = il_f2_make(y[i], y[i + 1]);
                    il_f2_get(il_f2_fma(il_f2_mul(x2, s[i / 2]), minus, il_f2_mul(x1, c[i / 2])), x[i], x[i + 1]);
                    il_f2_get(il_f2_add(il_f2_mul(x2, c[i / 2]), il_f2_mul(x1, s[i / 2])), y[i], y[i + 1]);
                }
            }
            if (mine && r < nh) {
                TA* to = to0 + (size_t)r * hd;
                kvq_store8(to + a, x), kvq_store8(to + b, y);
            }
            if (r0 + HEADS <= nh || !page) continue;          // (the warp's heads are all queries)
            uint32_t most = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) most = max(most, max(__float_as_uint(x[i]) & 0x7fffffffu, __float_as_uint(y[i]) & 0x7fffffffu));
            if (!mine) most = 0u;
#pragma unroll
            for (int o = 1; o < PER; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            if (!mine || r < nh) continue;
            const int v = r >= nh + nkv, head = r - nh - v * nkv, e = kvq_exponent<KIND>(most), turn = kvq_turn(hd, v, key), l0 = key * lanes;
            unsigned char *rec = page + (size_t)head * kvq_record(hd), *plane = rec + v * KVQ_PAGE * hd;
            const float f = kvq_inverse(e);
            uint2 ca = make_uint2(0u, 0u), cb = ca;
            if (e != KVQ_NAN) ca = kvq_codes8<KIND>(x, f), cb = kvq_codes8<KIND>(y, f);
            if (!turns) {                         // 16 neighbours: one piece
                *reinterpret_cast<uint4*>(plane + (((l0 + a / 16) ^ turn) << 4)) = make_uint4(ca.x, ca.y, cb.x, cb.y);
            } else {
                *reinterpret_cast<uint2*>(plane + (((l0 + a / 16) ^ turn) << 4) + (a & 8)) = ca;
                *reinterpret_cast<uint2*>(plane + (((l0 + b / 16) ^ turn) << 4) + (b & 8)) = cb;
            }
            if (j == 0) rec[2 * KVQ_PAGE * hd + v * KVQ_PAGE + key] = (unsigned char)e;
        }
    }
}

// A warp a row (a head of q, k or v of one token), a lane the columns lane, lane + 32, ...: any even rot, any alignment.
template <typename TA, int KIND>
__global__ void __launch_bounds__(256) rope_store_quant_any_kernel(const TA* qkv, long long row_stride, TA* q_out, long long q_stride, const int* tok_pos,
                                                                   const int* tok_entry, const int* block_table, int bt_stride,
                                                                   unsigned char* cache, int T, int nh, int nkv, int hd, int rot, const float* __restrict__ inv_freq, float mscale) {
    il_pdl_begin();
    const int rows = cache ? nh + 2 * nkv : nh, lane = threadIdx.x & 31, half = rot >> 1;
    const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= (long long)T * rows) return;
    const int t = (int)(item / rows), r = (int)(item - (long long)t * rows), pos = tok_pos[t];
    const TA* row = qkv + t * row_stride + (size_t)r * hd;
    float x[8];                                   // head_dim <= 256
    uint32_t most = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        x[i] = 0.f;
        if (d < hd) {
            x[i] = il_to_f(row[d]);
            if (r < nh + nkv && d < rot) {
                float c, s;
                kvq_angle(pos, inv_freq[d < half ? d : d - half], mscale, &c, &s);
                x[i] = d < half ? kvq_lo(x[i], il_to_f(row[d + half]), c, s) : kvq_hi(il_to_f(row[d - half]), x[i], c, s);
            }
            most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
        }
    }
    if (r < nh) {
        __syncwarp();                             // (q_out may be the row itself: every lane has read)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < hd) q_out[t * q_stride + (size_t)r * hd + lane + 32 * i] = il_from_f<TA>(x[i]);
        return;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    const int page = block_table[(size_t)tok_entry[t] * bt_stride + pos / KVQ_PAGE], key = pos % KVQ_PAGE;
    if (page < 0) return;                         // the host reserves every page a step touches; never write elsewhere
    const int v = r >= nh + nkv, head = r - nh - v * nkv, b = kvq_exponent<KIND>(most);
    unsigned char* rec = cache + ((size_t)page * nkv + head) * kvq_record(hd);
    const float f = kvq_inverse(b);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        if (d < hd)
            rec[v * KVQ_PAGE * hd + (((key * (hd / 16) + d / 16) ^ kvq_turn(hd, v, key)) << 4) + d % 16] =
                b == KVQ_NAN ? 0 : (unsigned char)kvq_codes4<KIND>(x[i] * f, 0.f, 0.f, 0.f);
    }
    if (lane == 0) rec[2 * KVQ_PAGE * hd + v * KVQ_PAGE + key] = (unsigned char)b;
}

// Arguments come as one struct (addresses and strides first, then numbers of 32 bits): a call from Python with twenty arguments costs 3 us, one with a packed struct less than one.
struct KvqStoreArgs {
    const void* qkv;
    long long row_stride;
    void* q_out;
    long long q_stride;
    const int *tok_pos, *tok_entry, *block_table;
    void* cache;
    const float* inv_freq;
    cudaStream_t stream;
    int act_kind, bt_stride, kind, T, nh, nkv, hd, rot;
    float mscale;
};
static_assert(sizeof(KvqStoreArgs) == 120, "what ops.py packs, padding included");
IL_EXPORT int il_rope_store_quant(const KvqStoreArgs* args) {
    const auto [qkv, row_stride, q_out, q_stride, tok_pos, tok_entry, block_table, cache, inv_freq, stream, act_kind, bt_stride, kind, T, nh, nkv, hd, rot, mscale] = *args;
    if (T <= 0) return IL_OK;
    if (hd > 256) return IL_UNSUPPORTED;
    if (nh <= 0 || nkv <= 0 || hd <= 0 || hd % 16 || rot < 0 || rot > hd || (rot & 1) || (rot && !inv_freq)) return IL_BAD_ARG;
    if (row_stride < (long long)(nh + 2 * nkv) * hd || q_stride < (long long)nh * hd || ((uintptr_t)cache & 15)) return IL_BAD_ARG;
    if ((kind != KVQ_E4M3 && kind != KVQ_INT8) || (act_kind != IL_F32 && act_kind != IL_BF16)) return IL_BAD_ARG;
    const int sz = act_kind == IL_F32 ? 4 : 2;
    if (rot % 16 == 0 && !(((uintptr_t)qkv | (uintptr_t)q_out) & 15) && (row_stride * sz) % 16 == 0 && (q_stride * sz) % 16 == 0) {
        const int per = hd <= 16 ? 1 : hd <= 32 ? 2 : hd <= 64 ? 4 : hd <= 128 ? 8 : 16, rows = cache ? nh + 2 * nkv : nh;
        // a warp a round of heads where the tokens are few, as few warps a token as fill the device twice where they are many
        const int rounds = (rows * per + 31) / 32, wpt = (long long)T * rounds <= KVS_WARPS ? rounds : (int)std::min<long long>(std::max<long long>(KVS_WARPS / T, 1), rounds);
        const long long warps = (long long)T * wpt;
        if (warps > 0x7fffffffLL * 8 - 8) return IL_UNSUPPORTED;
#define KVS_GO(TA, KIND, PER)                                                                                                                                   \
    IL_LAUNCH((rope_store_quant_kernel<TA, KIND, PER>), (unsigned)((warps + 7) / 8), 256, 0, stream, (const TA*)qkv, row_stride, (TA*)q_out, q_stride, tok_pos, \
              tok_entry, block_table, bt_stride, (unsigned char*)cache, T, nh, nkv, hd, rot, inv_freq, mscale, wpt)
#define KVS_PER(TA, KIND)                                \
    do {                                                 \
        if (per == 1) KVS_GO(TA, KIND, 1);               \
        else if (per == 2) KVS_GO(TA, KIND, 2);          \
        else if (per == 4) KVS_GO(TA, KIND, 4);          \
        else if (per == 8) KVS_GO(TA, KIND, 8);          \
        else KVS_GO(TA, KIND, 16);                       \
    } while (0)
        if (act_kind == IL_F32) {
            if (kind == KVQ_E4M3) KVS_PER(float, KVQ_E4M3);
            else KVS_PER(float, KVQ_INT8);
        } else {
            if (kind == KVQ_E4M3) KVS_PER(__nv_bfloat16, KVQ_E4M3);
            else KVS_PER(__nv_bfloat16, KVQ_INT8);
        }
#undef KVS_PER
#undef KVS_GO
        IL_LAUNCH_CHECK();
        return IL_OK;
    }
    const long long items = (long long)T * (cache ? nh + 2 * nkv : nh), blocks = (items + 7) / 8;
    if (blocks > 0x7fffffffLL) return IL_UNSUPPORTED;
#define KVS_GO(TA, KIND)                                                                                                                                     \
    IL_LAUNCH((rope_store_quant_any_kernel<TA, KIND>), (unsigned)blocks, 256, 0, stream, (const TA*)qkv, row_stride, (TA*)q_out, q_stride, tok_pos, tok_entry, \
              block_table, bt_stride, (unsigned char*)cache, T, nh, nkv, hd, rot, inv_freq, mscale)
    if (act_kind == IL_F32) {
        if (kind == KVQ_E4M3) KVS_GO(float, KVQ_E4M3);
        else KVS_GO(float, KVQ_INT8);
    } else {
        if (kind == KVQ_E4M3) KVS_GO(__nv_bfloat16, KVQ_E4M3);
        else KVS_GO(__nv_bfloat16, KVQ_INT8);
    }
#undef KVS_GO
    IL_LAUNCH_CHECK();
    return IL_OK;
}

// The pages of a request that its portion sees: the first of them, and how many.
__device__ __forceinline__ int kvu_seen(const int* entry_kvlen, const int* entry_qstart, int window, int e, int width, int* first) {
    const int kvlen = entry_kvlen[e];
    *first = entry_qstart ? il_mask_lo(max(kvlen - (entry_qstart[e + 1] - entry_qstart[e]), 0), window) / KVQ_PAGE : 0;
    return max(min((kvlen + KVQ_PAGE - 1) / KVQ_PAGE, width) - *first, 0);
}

// A block a page of a request. room > 0: the pages that are seen lie one behind the other, request after request, up to `room` of them, and `table` says where (0 for the others: in bounds
// for who looks all the same; pages for which no room is left set *status); else page p of the i-th request lies at i * width + p. Pages in front of the one that holds the lowest position
// the request's portion sees (its first new token's, by the mask) and behind the last are left as they are, slots behind the request's end become zeros. A thread makes 16 bytes of output at a
// time, KVU_AHEAD of them at once: bound by memory, what matters is loads under way and few instructions between them. HD 0: any head size. 16 requests of up to 8,192 tokens, 8 kv heads of
// 128, e4m3 to bfloat16, us: 79.9 with places worked out for each piece, 71.0 so (6.0 TB/s); two pieces at a time 77, eight 69.9 (but more for few tokens), sixteen 81.
// Dealt out (below) they take 76; but 64 requests of 300 tokens with tables of 2,048 pages 26 for 187, one of 32,000 among them 58 for 216: a block that finds nothing costs a nanosecond,
// so tables of up to KVU_EACH pages together have a block a page.
constexpr int KVU_AHEAD = 4, KVU_EACH = 8192, KVU_BLOCKS = 148 * 16;
__device__ __forceinline__ void kvq_put4(float* o, float a, float b, float c, float d) { o[0] = a, o[1] = b, o[2] = c, o[3] = d; }
__device__ __forceinline__ void kvq_put4(__nv_bfloat16* o, float a, float b, float c, float d) {
    *reinterpret_cast<__nv_bfloat162*>(o) = __floats2bfloat162_rn(a, b), *reinterpret_cast<__nv_bfloat162*>(o + 2) = __floats2bfloat162_rn(c, d);
}
// One page: its records to the rows of `out`.
template <typename TO, int KIND, int HD>
__device__ __forceinline__ void kvu_page(const unsigned char* recs, TO* out, int n_keys, int nkv, int hd_arg, int told_by_key) {
    const int hd = HD ? HD : hd_arg;
    constexpr int VEC = 16 / sizeof(TO);
    const int rec_bytes = kvq_record(hd);
    const int per = hd / VEC, plane = KVQ_PAGE * per;         // pieces of a row and of a head
    // A thread has the same piece of one head after another: what it needs of the key and the column is made once. Small heads are several at a time.
    const bool several = 256 % plane == 0;
    const int step = several ? 256 / plane : 1, v0 = several ? threadIdx.x / plane : 0;
    for (int u = several ? threadIdx.x % plane : threadIdx.x; u < plane; u += 256) {
        const int key = u / per, d = (u - key * per) * VEC;
        const bool there = key < n_keys;
        const int at_k = (((key * (hd / 16) + d / 16) ^ kvq_turn(hd, false, key)) << 4) + d % 16;
        const int at_v = (((key * (hd / 16) + d / 16) ^ kvq_turn(hd, true, key)) << 4) + d % 16 + KVQ_PAGE * hd;
        for (int vh0 = v0; vh0 < 2 * nkv; vh0 += step * KVU_AHEAD) {
            uint2 code[KVU_AHEAD];
            int ke[KVU_AHEAD], ve[KVU_AHEAD];
#pragma unroll
            for (int k = 0; k < KVU_AHEAD; ++k) {
                const int vh = vh0 + k * step;
                const bool v = vh >= nkv;
                if (vh < 2 * nkv && there) {
                    const unsigned char* rec = recs + (size_t)(v ? vh - nkv : vh) * rec_bytes;
                    const unsigned char* at = rec + (v ? at_v : at_k);
                    if (VEC == 8) code[k] = *reinterpret_cast<const uint2*>(at);
                    else code[k].x = *reinterpret_cast<const uint32_t*>(at);
                    ke[k] = rec[2 * KVQ_PAGE * hd + key], ve[k] = rec[2 * KVQ_PAGE * hd + KVQ_PAGE + key];
                }
            }
#pragma unroll
            for (int k = 0; k < KVU_AHEAD; ++k) {
                const int vh = vh0 + k * step;
                if (vh >= 2 * nkv) break;
                const bool v = vh >= nkv;
                uint4 w = make_uint4(0u, 0u, 0u, 0u);
                if (there) {
                    // for the attention a row of V that is NaN is told by its key (a masked key then leaves no trace: its score is replaced, its value is zero)
                    const bool told = told_by_key && ve[k] == KVQ_NAN;
                    const float f = kvq_power(told ? KVQ_NAN : v ? ve[k] : ke[k]);
                    const uint32_t c[2] = {code[k].x, code[k].y};
                    TO* o = reinterpret_cast<TO*>(&w);
#pragma unroll
                    for (int x = 0; x < VEC / 4; ++x) {
                        const uint32_t raw = kvq_raw<KIND>(c[x]), h0 = kvq_low<KIND>(raw), h1 = kvq_high<KIND>(raw);
                        const float2 lo2 = __half22float2(*reinterpret_cast<const __half2*>(&h0)), hi2 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
                        kvq_put4(o + 4 * x, lo2.x * f, lo2.y * f, hi2.x * f, hi2.y * f);
                    }
                    if (told && v) w = make_uint4(0u, 0u, 0u, 0u);
                }
                *reinterpret_cast<uint4*>(out + ((size_t)vh * KVQ_PAGE + key) * hd + d) = w;
            }
        }
    }
}

template <typename TO, int KIND, int HD>
__global__ void __launch_bounds__(256, 4) kv_unpack_kernel(const unsigned char* cache, const int* block_table, int bt_stride, const int* entry_kvlen,
                                                        const int* entry_qstart, int window, int first_entry, int nkv, int hd_arg, TO* pages, int* table, int told_by_key, int room, int* status) {
    il_pdl_begin();
    const int hd = HD ? HD : hd_arg;
    const int i = blockIdx.y, e = first_entry + i, p = blockIdx.x;
    int first;
    const int n_seen = kvu_seen(entry_kvlen, entry_qstart, window, e, gridDim.x, &first), kvlen = entry_kvlen[e];
    const bool seen = p >= first && p - first < n_seen;
    size_t to = (size_t)i * gridDim.x + p;
    if (room > 0 && seen) {                       // behind the pages of the requests in front
        __shared__ int sums[8];
        int sum = 0, f;
        for (int k = threadIdx.x; k < i; k += 256) sum += kvu_seen(entry_kvlen, entry_qstart, window, first_entry + k, gridDim.x, &f);
        sum = __reduce_add_sync(0xffffffffu, sum);
        if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = sum;
        __syncthreads();
        sum = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += sums[k];
        to = (size_t)sum + (p - first);
    }
    const bool fits = room <= 0 || to < (size_t)room;
    if (threadIdx.x == 0) {
        if (table) table[(size_t)e * gridDim.x + p] = room > 0 && !(seen && fits) ? 0 : (int)to;
        if (seen && !fits) atomicExch(status, 92);
    }
    if (!seen || !fits) return;
    const int page = block_table[(size_t)e * bt_stride + p], rec_bytes = kvq_record(hd), n_keys = page < 0 ? 0 : min(KVQ_PAGE, kvlen - p * KVQ_PAGE);
    kvu_page<TO, KIND, HD>(cache + (size_t)max(page, 0) * nkv * rec_bytes, pages + to * 2 * nkv * KVQ_PAGE * hd, n_keys, nkv, hd, told_by_key);
}

// The same where tables are so wide, for so many requests, that most blocks of a page each might find nothing: the pages that are seen dealt out to KVU_BLOCKS blocks.
template <typename TO, int KIND, int HD>
__global__ void __launch_bounds__(256, 4) kv_unpack_dealt_kernel(const unsigned char* cache, const int* block_table, int bt_stride, const int* entry_kvlen,
                                                        const int* entry_qstart, int window, int first_entry, int n, int width, int nkv, int hd_arg, TO* pages, int* table, int told_by_key, int room,
                                                        int* status) {
    il_pdl_begin();
    const int hd = HD ? HD : hd_arg;
    const int lane = threadIdx.x & 31, rec_bytes = kvq_record(hd);
    // how many pages are seen, and the request that this block's first one belongs to, with how many lie in front of that request's (every warp for itself, a lane a request)
    int first, all = 0, n0 = 0;
    for (int i0 = 0; i0 < n; i0 += 32) {
        const int seen = i0 + lane < n ? kvu_seen(entry_kvlen, entry_qstart, window, first_entry + i0 + lane, width, &first) : 0;
        if (i0 == 0) n0 = seen;
        all += __reduce_add_sync(0xffffffffu, seen);
    }
    const int share = (int)(((unsigned)all + gridDim.x - 1) / gridDim.x);
    const long long from = (long long)blockIdx.x * share;
    if (from < all) {
        int i = 0, before = 0;
        for (int i0 = 0; i0 < n; i0 += 32) {
            const int seen = i0 == 0 ? n0 : i0 + lane < n ? kvu_seen(entry_kvlen, entry_qstart, window, first_entry + i0 + lane, width, &first) : 0;
            int sum = seen;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += x;
            }
            const unsigned past = __ballot_sync(0xffffffffu, before + sum > (int)from);
            if (past) {
                const int l = __ffs(past) - 1;
                i = i0 + l, before += __shfl_sync(0xffffffffu, sum - seen, l);
                break;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        int n_seen = kvu_seen(entry_kvlen, entry_qstart, window, first_entry + i, width, &first), kvlen = entry_kvlen[first_entry + i];
        for (int at = (int)from; at < min(from + share, (long long)all); ++at) {
            while (at >= before + n_seen) {
                before += n_seen, ++i;
                n_seen = kvu_seen(entry_kvlen, entry_qstart, window, first_entry + i, width, &first), kvlen = entry_kvlen[first_entry + i];
            }
            if (room > 0 && at >= room) {
                if (threadIdx.x == 0) atomicExch(status, 92);
                break;
            }
            const int p = first + at - before, page = block_table[(size_t)(first_entry + i) * bt_stride + p], n_keys = page < 0 ? 0 : min(KVQ_PAGE, kvlen - p * KVQ_PAGE);
            const size_t to = room > 0 ? at : (size_t)i * width + p;
            kvu_page<TO, KIND, HD>(cache + (size_t)max(page, 0) * nkv * rec_bytes, pages + to * 2 * nkv * KVQ_PAGE * hd, n_keys, nkv, hd, told_by_key);
        }
    }
    if (table)
        for (int i = blockIdx.x; i < n; i += gridDim.x) {
            int before = 0;
            for (int k = lane; k < i; k += 32) before += kvu_seen(entry_kvlen, entry_qstart, window, first_entry + k, width, &first);
            before = __reduce_add_sync(0xffffffffu, before);
            const int n_seen = kvu_seen(entry_kvlen, entry_qstart, window, first_entry + i, width, &first), n_fit = min(n_seen, max(room - before, 0));
            for (int p = threadIdx.x; p < width; p += 256)
                table[(size_t)(first_entry + i) * width + p] = room <= 0 ? i * width + p : p >= first && p - first < n_fit ? before + p - first : 0;
        }
}

struct KvqUnpackArgs {
    const void* cache;
    const int *block_table, *entry_kvlen, *entry_qstart;
    void* pages;
    int* table;
    cudaStream_t stream;
    int* status;
    int kind, bt_stride, window, first_entry, n_entries, width, nkv, hd, out_kind, told_by_key, room;
};
static_assert(sizeof(KvqUnpackArgs) == 112, "what ops.py packs, padding included");
IL_EXPORT int il_kv_unpack(const KvqUnpackArgs* args) {
    const auto [cache, block_table, entry_kvlen, entry_qstart, pages, table, stream, status, kind, bt_stride, window, first_entry, n_entries, width, nkv, hd, out_kind, told_by_key,
                room] = *args;
    const int n = n_entries - first_entry;
    if (n <= 0 || width <= 0) return IL_OK;
    if (hd > 256 || n > 65535) return IL_UNSUPPORTED;
    if (nkv <= 0 || hd <= 0 || hd % 16 || width > bt_stride || first_entry < 0 || (((uintptr_t)cache | (uintptr_t)pages) & 15)) return IL_BAD_ARG;
    if ((long long)n * width > 0x7fffffffLL) return IL_UNSUPPORTED;
    if (room < 0 || (room > 0 && (!table || !status))) return IL_BAD_ARG;
    if ((kind != KVQ_E4M3 && kind != KVQ_INT8) || (out_kind != IL_F32 && out_kind != IL_BF16)) return IL_BAD_ARG;
    const bool each = (long long)n * width <= KVU_EACH;
#define KVU_OF(TO, KIND, HD)                                                                                                                                     \
    do {                                                                                                                                                         \
        if (each)                                                                                                                                                \
            IL_LAUNCH((kv_unpack_kernel<TO, KIND, HD>), dim3(width, n), 256, 0, stream, (const unsigned char*)cache, block_table, bt_stride, entry_kvlen,        \
                      entry_qstart, window, first_entry, nkv, hd, (TO*)pages, table, told_by_key, room, status);                                                 \
        else                                                                                                                                                     \
            IL_LAUNCH((kv_unpack_dealt_kernel<TO, KIND, HD>), dim3(KVU_BLOCKS), 256, 0, stream, (const unsigned char*)cache, block_table, bt_stride, entry_kvlen, \
                      entry_qstart, window, first_entry, n, width, nkv, hd, (TO*)pages, table, told_by_key, room, status);                                       \
    } while (0)
#define KVU_GO(TO, KIND)                                 \
    do {                                                 \
        if (hd == 64) KVU_OF(TO, KIND, 64);              \
        else if (hd == 128) KVU_OF(TO, KIND, 128);       \
        else KVU_OF(TO, KIND, 0);                        \
    } while (0)
    if (out_kind == IL_F32) {
        if (kind == KVQ_E4M3) KVU_GO(float, KVQ_E4M3);
        else KVU_GO(float, KVQ_INT8);
    } else {
        if (kind == KVQ_E4M3) KVU_GO(__nv_bfloat16, KVQ_E4M3);
        else KVU_GO(__nv_bfloat16, KVQ_INT8);
    }
#undef KVU_OF
#undef KVU_GO
    IL_LAUNCH_CHECK();
    return IL_OK;
}
