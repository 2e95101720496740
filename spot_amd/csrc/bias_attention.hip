// Entry points of the attention with a relative position bias (kernels: bias_attention.h), and the two small kernels
// that turn the backward's sums along offsets into the gradient of the bias table.
#include "bias_attention.h"
#include "../../include/spot_hip.h"

namespace ba {

// Sums of dS along each (class, offset) cell over sequences and query blocks.  One thread per cell; the partial sums of
// a workgroup lie at a = delta + BM - 1 + offset_b + BM * block.  At most BM terms are in each partial sum (32 bits);
// from here on the sums are 64 bits.
__global__ __launch_bounds__(256) void offset_sums_kernel(const Args a, double* __restrict__ sums) {
    const int n = 2 * a.N - 1, i = blockIdx.x * 256 + threadIdx.x, head = blockIdx.y, cls = blockIdx.z, ncls = gridDim.z;
    if (i >= n) return;
    const int nq = (a.Lq + BM - 1) / BM, span = a.Lk + BM, delta = i - (a.N - 1);
    double sum = 0.;
    for (int b = 0; b < a.B; ++b) {
        const Seq s = sequence(a, b);
        const float* part = a.part + (((long)b * a.H + head) * nq * ncls + cls) * span;
        for (int q = 0; q < nq; ++q) {
            const int at = delta + BM - 1 + s.off + q * BM;
            if (at >= 0 && at < span) sum += part[(long)q * ncls * span + at];
        }
    }
    sums[((long)head * ncls + cls) * n + i] = sum;
}

// One wave per (bucket, head): the cells of a bucket stand together in `order`.
__global__ __launch_bounds__(256) void bucket_sums_kernel(const double* __restrict__ sums, const int* __restrict__ order,
                                                          const int* __restrict__ start, void* __restrict__ dtable,
                                                          int table_type, int nb, int H, int cells) {
    const int bucket = blockIdx.x * 4 + (threadIdx.x >> 6), head = blockIdx.y;
    if (bucket >= nb) return;
    double sum = 0.;
    const int end = min(start[bucket + 1], cells);
    for (int z = max(start[bucket], 0) + (threadIdx.x & 63); z < end; z += 64) {
        const int cell = order[z];
        if ((unsigned)cell < (unsigned)cells) sum += sums[(long)head * cells + cell];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if ((threadIdx.x & 63) != 0) return;
    const long at = (long)bucket * H + head;
    if (table_type == F32) static_cast<float*>(dtable)[at] = (float)sum;
    else if (table_type == BF16) static_cast<__bf16*>(dtable)[at] = (__bf16)(float)sum;
    else static_cast<_Float16*>(dtable)[at] = (_Float16)(float)sum;
}

static int launch_any(int dtype, int what, int D, const Args& a, unsigned grid, hipStream_t stream) {
    return dtype == F32 ? launch_f32(what, D, a, grid, stream) : dtype == BF16 ? launch_bf16(what, D, a, grid, stream)
                                                                               : launch_f16(what, D, a, grid, stream);
}

// Backward workspace in bytes: sums along offsets (64 bits) | delta | partial sums along offsets.
struct Layout { long sums, delta, part, total; };
static Layout layout(const spot_bias_attn_desc& d) {
    const long cls = d.width > 0 ? 2 : 1, nq = (d.Lq + BM - 1) / BM;
    Layout l;
    l.sums = 0;
    l.delta = d.dtable ? l.sums + 8 * (long)d.H * cls * (2L * d.max_len - 1) : 0;
    l.part = l.delta + ((4L * d.B * d.H * d.Lq + 15) & ~15L);
    l.total = l.part + (d.dtable ? 4 * (long)d.B * d.H * nq * cls * ((long)d.Lk + BM) : 0);
    return l;
}

// The forward's kernel.  few_kernel reads keys once for all heads that share them and cuts the keys between its waves and
// workgroups; fwd_kernel reads them once per 128 queries.  The former is taken for up to 32 rows per key/value head, and
// where the latter's workgroups would not fill the 256 CUs.
struct Few { bool use; int heads, queries, tiles, splits; long o, ml; };
static Few few(const spot_bias_attn_desc& d) {
    Few f = {};
    const int G = d.H / d.Hkv;
    f.use = (long)d.Lq * G <= 32 || (long)d.B * d.H * ((d.Lq + BM - 1) / BM) < 256;
    f.heads = G < 32 ? G : 32;
    f.queries = 32 / f.heads;
    f.tiles = ((d.Lq + f.queries - 1) / f.queries) * ((G + f.heads - 1) / f.heads);
    // about four workgroups per CU, each with a few tiles for every wave
    const long units = (long)d.B * d.Hkv * f.tiles, most = d.Lk / (4 * FT * 2);
    long splits = units ? 1024 / units : 1;
    if (splits > most) splits = most;
    f.splits = splits < 1 ? 1 : (int)splits;
    if (f.splits > 1) {
        f.o = units * f.splits * 32 * d.head_dim * 4;
        f.ml = units * f.splits * 32 * 2 * 4;
    }
    return f;
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

static int check(const spot_bias_attn_desc* d, bool backward) {
    SPOT_CHECK_ARG(d != nullptr, "spot_bias_attention: null descriptor");
    SPOT_CHECK_ARG(d->dtype >= F32 && d->dtype <= F16 && d->table_dtype >= F32 && d->table_dtype <= F16,
                   "spot_bias_attention: dtype %d / table_dtype %d is none of 0 (f32), 1 (bf16), 2 (f16)", d->dtype, d->table_dtype);
    SPOT_CHECK_ARG(d->head_dim == 32 || d->head_dim == 64 || d->head_dim == 128,
                   "spot_bias_attention: head_dim must be 32, 64 or 128, not %d", d->head_dim);
    SPOT_CHECK_ARG(d->B >= 0 && d->Lq >= 0 && d->Lk >= 0 && d->H > 0 && d->Hkv > 0 && d->H % d->Hkv == 0,
                   "spot_bias_attention: B %d, Lq %d, Lk %d, %d heads over %d key/value heads", d->B, d->Lq, d->Lk, d->H, d->Hkv);
    SPOT_CHECK_ARG(d->max_len >= 1 && d->max_len <= SPOT_BIAS_ATTN_MAX_LEN && d->Lk <= d->max_len && d->Lq <= SPOT_BIAS_ATTN_MAX_LEN,
                   "spot_bias_attention: max_len %d for %d keys and %d queries (1 to %d, no fewer than the keys)", d->max_len, d->Lk,
                   d->Lq, SPOT_BIAS_ATTN_MAX_LEN);
    SPOT_CHECK_ARG(d->num_buckets >= 1 && d->width >= 0, "spot_bias_attention: %d buckets, width %d", d->num_buckets, d->width);
    SPOT_CHECK_ARG(d->q_offset_mode >= 0 && d->q_offset_mode <= 2 && (d->q_offset_mode != 1 || d->q_offsets),
                   "spot_bias_attention: q_offset_mode %d", d->q_offset_mode);
    SPOT_CHECK_ARG(d->q_offset_mode != 0 || (d->q_offset >= 0 && (long)d->q_offset + d->Lq <= d->max_len),
                   "spot_bias_attention: queries at %d .. %ld, but the buckets end at %d", d->q_offset, (long)d->q_offset + d->Lq - 1, d->max_len);
    SPOT_CHECK_ARG(!backward || !d->dtable || (d->cell_order && d->cell_start),
                   "spot_bias_attention_bwd: dtable needs cell_order and cell_start");
    if (d->B == 0) return SPOT_OK;
    SPOT_CHECK_ARG(d->table && d->cells && (d->Lq == 0 || (d->q && d->out)) && (d->Lk == 0 || (d->k && d->v)),
                   "spot_bias_attention: null pointer");
    const long per = d->dtype == F32 ? 4 : 8;
    const long strides[] = {d->q_stride_b, d->q_stride_l, d->q_stride_h, d->k_stride_b, d->k_stride_l, d->k_stride_h,
                            d->v_stride_b, d->v_stride_l, d->v_stride_h};
    for (long s : strides)
        SPOT_CHECK_ARG(s % per == 0, "spot_bias_attention: a stride of %ld elements is no whole number of 16 bytes", s);
    SPOT_CHECK_ARG(aligned16(d->q) && aligned16(d->k) && aligned16(d->v) && aligned16(d->out) && aligned16(d->out_lo),
                   "spot_bias_attention: q, k, v, out and out_lo have to be 16-byte aligned");
    SPOT_CHECK_ARG((long)d->B * d->H * ((d->Lq + 31) / 32) < (1L << 31) && (long)d->B * d->Hkv * ((d->Lk + 31) / 32) < (1L << 31),
                   "spot_bias_attention: B %d, H %d, Lq %d, Lk %d need too many workgroups", d->B, d->H, d->Lq, d->Lk);
    if (backward) {
        SPOT_CHECK_ARG(d->Lq == 0 || (d->stats && d->d_out && d->dq), "spot_bias_attention_bwd: stats, d_out and dq are needed");
        SPOT_CHECK_ARG((d->dk == nullptr) == (d->dv == nullptr), "spot_bias_attention_bwd: dk and dv come together");
        SPOT_CHECK_ARG(aligned16(d->d_out) && aligned16(d->dq) && aligned16(d->dk) && aligned16(d->dv),
                       "spot_bias_attention_bwd: d_out, dq, dk and dv have to be 16-byte aligned");
    }
    return SPOT_OK;
}

static Args arguments(const spot_bias_attn_desc& d) {
    Args a = {};
    a.q = d.q; a.k = d.k; a.v = d.v; a.d_out = d.d_out; a.table = d.table;
    a.out = d.out; a.out_lo = d.out_lo; a.dq = d.dq; a.dk = d.dk; a.dv = d.dv;
    a.stats = d.stats;
    a.cells = d.cells; a.q_offsets = d.q_offsets; a.kv_len = d.kv_len; a.kpm = d.key_padding_mask;
    a.q_b = d.q_stride_b; a.q_l = d.q_stride_l; a.q_h = d.q_stride_h;
    a.k_b = d.k_stride_b; a.k_l = d.k_stride_l; a.k_h = d.k_stride_h;
    a.v_b = d.v_stride_b; a.v_l = d.v_stride_l; a.v_h = d.v_stride_h;
    a.B = d.B; a.H = d.H; a.Hkv = d.Hkv; a.G = d.H / d.Hkv; a.Lq = d.Lq; a.Lk = d.Lk; a.N = d.max_len; a.width = d.width;
    a.nb = d.num_buckets; a.causal = d.causal != 0; a.off_mode = d.q_offset_mode; a.off = d.q_offset; a.table_type = d.table_dtype;
    a.scale = d.scale; a.c = d.scale * LOG2E;
    return a;
}

}  // namespace ba

extern "C" int spot_bias_attention_fwd(const spot_bias_attn_desc* desc, hipStream_t stream) {
    using namespace ba;
    if (const int rc = check(desc, false)) return rc;
    const spot_bias_attn_desc& d = *desc;
    if (d.B == 0 || d.Lq == 0) return SPOT_OK;
    Args a = arguments(d);
    const Few f = few(d);
    if (!f.use) return launch_any(d.dtype, FWD, d.head_dim, a, (unsigned)d.B * d.H * ((d.Lq + BM - 1) / BM), stream);
    SPOT_CHECK_ARG(f.splits == 1 || (d.ws && aligned16(d.ws) && d.ws_bytes >= f.o + f.ml),
                   "spot_bias_attention_fwd: a 16-byte aligned workspace of %ld bytes is needed, %ld are given", f.o + f.ml, d.ws_bytes);
    a.heads = f.heads; a.queries = f.queries; a.tiles = f.tiles; a.splits = f.splits;
    a.few_o = static_cast<float*>(d.ws);
    a.few_ml = a.few_o + f.o / 4;
    const unsigned tiles = (unsigned)d.B * d.Hkv * f.tiles;
    const int rc = launch_any(d.dtype, FEW, d.head_dim, a, tiles * f.splits, stream);
    return rc || f.splits == 1 ? rc : launch_any(d.dtype, MERGE, d.head_dim, a, tiles, stream);
}

extern "C" int spot_bias_attention_fwd_ws_bytes(const spot_bias_attn_desc* desc, long* bytes) {
    using namespace ba;
    if (const int rc = check(desc, false)) return rc;
    SPOT_CHECK_ARG(bytes != nullptr, "spot_bias_attention_fwd_ws_bytes: null pointer");
    const Few f = few(*desc);
    *bytes = f.use && desc->Lq > 0 ? f.o + f.ml : 0;
    return SPOT_OK;
}

extern "C" int spot_bias_attention_bwd_ws_bytes(const spot_bias_attn_desc* desc, long* bytes) {
    using namespace ba;
    if (const int rc = check(desc, false)) return rc;
    SPOT_CHECK_ARG(bytes != nullptr, "spot_bias_attention_bwd_ws_bytes: null pointer");
    *bytes = layout(*desc).total;
    return SPOT_OK;
}

extern "C" int spot_bias_attention_bwd(const spot_bias_attn_desc* desc, hipStream_t stream) {
    using namespace ba;
    if (const int rc = check(desc, true)) return rc;
    const spot_bias_attn_desc& d = *desc;
    Args a = arguments(d);
    const Layout l = layout(d);
    SPOT_CHECK_ARG(l.total == 0 || (d.ws && aligned16(d.ws) && d.ws_bytes >= l.total),
                   "spot_bias_attention_bwd: a 16-byte aligned workspace of %ld bytes is needed, %ld are given", l.total, d.ws_bytes);
    char* ws = static_cast<char*>(d.ws);
    a.delta = reinterpret_cast<float*>(ws + l.delta);
    a.part = d.dtable ? reinterpret_cast<float*>(ws + l.part) : nullptr;
    if (d.B > 0 && d.Lq > 0)
        if (const int rc = launch_any(d.dtype, DQ, d.head_dim, a, (unsigned)d.B * d.H * ((d.Lq + BM - 1) / BM), stream)) return rc;
    if (d.B > 0 && d.dk && d.Lk > 0)
        if (const int rc = launch_any(d.dtype, DKV, d.head_dim, a, (unsigned)d.B * d.Hkv * ((d.Lk + KB - 1) / KB), stream)) return rc;
    if (d.dtable) {
        const int cls = d.width > 0 ? 2 : 1, n = 2 * d.max_len - 1;
        double* sums = reinterpret_cast<double*>(ws + l.sums);
        offset_sums_kernel<<<dim3((n + 255) / 256, d.H, cls), 256, 0, stream>>>(a, sums);
        SPOT_CHECK_LAUNCH("spot_bias_attention_bwd");
        bucket_sums_kernel<<<dim3((d.num_buckets + 3) / 4, d.H), 256, 0, stream>>>(sums, d.cell_order, d.cell_start, d.dtable,
                                                                               d.table_dtype, d.num_buckets, d.H, cls * n);
        SPOT_CHECK_LAUNCH("spot_bias_attention_bwd");
    }
    return SPOT_OK;
}
