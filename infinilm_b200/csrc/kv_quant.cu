// Writing the 8-bit key/value cache and reading it back.
//
// il_rope_store_quant: rotary encoding of q and k (pairs (i, i + rot/2), cos and sin times `mscale`), then k and v as codes into the page of the token's
// slot. The angle pos * inv_freq[i] is made and reduced in 64 bits (exact product, so a far position turns as it should), sine and
// cosine in 32; k is rounded once, from 32 bits to its code. qkv rows: [nh heads of q | nkv of k | nkv of v]; q goes to `q_out`, which
// may be the same place.
// il_kv_unpack: pages of requests as pages of bfloat16 or float32 values in the layout of the plain cache, [page][K, V][kv head][16][head_dim].
// Both are bound by memory: what they read and write is named at each kernel.
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

// A warp a row (a head of q, k or v of one token), a lane the columns lane, lane + 32, ...: any even rot, any alignment.
template <typename TA, int KIND>
__global__ void __launch_bounds__(256) rope_store_quant_any_kernel(const TA* qkv, long long row_stride, TA* q_out, long long q_stride, const int* __restrict__ tok_pos,
                                                                   const int* __restrict__ tok_entry, const int* __restrict__ block_table, int bt_stride,
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

IL_EXPORT int il_rope_store_quant(const void* qkv, int act_kind, long long row_stride, void* q_out, long long q_stride, const int* tok_pos, const int* tok_entry,
                                  const int* block_table, int bt_stride, void* cache, int kind, int T, int nh, int nkv, int hd, int rot,
                                  const float* inv_freq, float mscale, cudaStream_t stream) {
    if (T <= 0) return IL_OK;
    if (hd > 256) return IL_UNSUPPORTED;
    if (nh <= 0 || nkv <= 0 || hd <= 0 || hd % 16 || rot < 0 || rot > hd || (rot & 1) || (rot && !inv_freq)) return IL_BAD_ARG;
    if (row_stride < (long long)(nh + 2 * nkv) * hd || q_stride < (long long)nh * hd || ((uintptr_t)cache & 15)) return IL_BAD_ARG;
    if ((kind != KVQ_E4M3 && kind != KVQ_INT8) || (act_kind != IL_F32 && act_kind != IL_BF16)) return IL_BAD_ARG;
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

// A block a page of a request. first: the page of the lowest position that the request's portion sees (its first new token's, by the mask); pages in
// front of it and behind the last are left as they are, slots behind the request's end become zeros. A thread makes 16 bytes of output at a time.
template <typename TO, int KIND>
__global__ void __launch_bounds__(256) kv_unpack_kernel(const unsigned char* cache, const int* __restrict__ block_table, int bt_stride, const int* __restrict__ entry_kvlen,
                                                        const int* __restrict__ entry_qstart, int window, int first_entry, int nkv, int hd, TO* pages, int* table, int poison) {
    il_pdl_begin();
    constexpr int VEC = 16 / sizeof(TO);
    const int i = blockIdx.y, e = first_entry + i, p = blockIdx.x;
    const size_t to = (size_t)i * gridDim.x + p;
    if (table && threadIdx.x == 0) table[(size_t)e * gridDim.x + p] = (int)to;
    const int kvlen = entry_kvlen[e];
    const int lo = entry_qstart ? il_mask_lo(max(kvlen - (entry_qstart[e + 1] - entry_qstart[e]), 0), window) : 0;
    if (p < lo / KVQ_PAGE || p * KVQ_PAGE >= kvlen) return;
    const int page = block_table[(size_t)e * bt_stride + p], rec_bytes = kvq_record(hd), n_keys = page < 0 ? 0 : min(KVQ_PAGE, kvlen - p * KVQ_PAGE);
    const unsigned char* recs = cache + (size_t)max(page, 0) * nkv * rec_bytes;
    TO* out = pages + to * 2 * nkv * KVQ_PAGE * hd;
    const int per = hd / VEC, total = 2 * nkv * KVQ_PAGE * per;
    for (int u = threadIdx.x; u < total; u += 256) {
        const int row = u / per, d = (u - row * per) * VEC, key = row % KVQ_PAGE, vh = row / KVQ_PAGE, v = vh >= nkv, head = vh - v * nkv;
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (key < n_keys) {
            const unsigned char* rec = recs + (size_t)head * rec_bytes;
            const unsigned char* at = rec + v * KVQ_PAGE * hd + (((key * (hd / 16) + d / 16) ^ kvq_turn(hd, v, key)) << 4) + d % 16;
            const unsigned char* ex = rec + 2 * KVQ_PAGE * hd + key;
            // for the attention a row of V that is NaN is told by its key (a masked key then leaves no trace: its score is replaced, its value is zero)
            const bool told = poison && ex[KVQ_PAGE] == KVQ_NAN;
            const float f = kvq_power(told ? KVQ_NAN : ex[v * KVQ_PAGE]);
            uint32_t c[VEC / 4];
            if (VEC == 8) {
                const uint2 g = *reinterpret_cast<const uint2*>(at);
                c[0] = g.x, c[VEC / 4 - 1] = g.y;
            } else {
                c[0] = *reinterpret_cast<const uint32_t*>(at);
            }
            TO* o = reinterpret_cast<TO*>(&w);
#pragma unroll
            for (int k = 0; k < VEC / 4; ++k) {
                const uint32_t raw = kvq_raw<KIND>(c[k]), h0 = kvq_low<KIND>(raw), h1 = kvq_high<KIND>(raw);
                const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h0)), bb = __half22float2(*reinterpret_cast<const __half2*>(&h1));
                o[4 * k] = il_from_f<TO>(a.x * f), o[4 * k + 1] = il_from_f<TO>(a.y * f);
                o[4 * k + 2] = il_from_f<TO>(bb.x * f), o[4 * k + 3] = il_from_f<TO>(bb.y * f);
            }
            if (told && v) w = make_uint4(0u, 0u, 0u, 0u);
        }
        *reinterpret_cast<uint4*>(out + (size_t)row * hd + d) = w;
    }
}

IL_EXPORT int il_kv_unpack(const void* cache, int kind, const int* block_table, int bt_stride, const int* entry_kvlen, const int* entry_qstart, int window,
                           int first_entry, int n_entries, int width, int nkv, int hd, void* pages, int out_kind, int* table, int poison, cudaStream_t stream) {
    const int n = n_entries - first_entry;
    if (n <= 0 || width <= 0) return IL_OK;
    if (hd > 256 || n > 65535) return IL_UNSUPPORTED;
    if (nkv <= 0 || hd <= 0 || hd % 16 || width > bt_stride || first_entry < 0 || (((uintptr_t)cache | (uintptr_t)pages) & 15)) return IL_BAD_ARG;
    if ((long long)n * width > 0x7fffffffLL) return IL_UNSUPPORTED;
    if ((kind != KVQ_E4M3 && kind != KVQ_INT8) || (out_kind != IL_F32 && out_kind != IL_BF16)) return IL_BAD_ARG;
#define KVU_GO(TO, KIND)                                                                                                                                \
    IL_LAUNCH((kv_unpack_kernel<TO, KIND>), dim3(width, n), 256, 0, stream, (const unsigned char*)cache, block_table, bt_stride, entry_kvlen, entry_qstart, \
              window, first_entry, nkv, hd, (TO*)pages, table, poison)
    if (out_kind == IL_F32) {
        if (kind == KVQ_E4M3) KVU_GO(float, KVQ_E4M3);
        else KVU_GO(float, KVQ_INT8);
    } else {
        if (kind == KVQ_E4M3) KVU_GO(__nv_bfloat16, KVQ_E4M3);
        else KVU_GO(__nv_bfloat16, KVQ_INT8);
    }
#undef KVU_GO
    IL_LAUNCH_CHECK();
    return IL_OK;
}
