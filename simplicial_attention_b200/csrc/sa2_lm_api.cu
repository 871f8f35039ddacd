// C ABI of the operators around the attention layers (declared in include/sa2.h): argument checks and launches.  No torch types, no
// allocation, no host sync.
#include "sa2.h"
#include "sa2_distill.cuh"
#include "sa2_embed.cuh"
#include "sa2_rotary.cuh"
#include "sa2_sample.cuh"
#include <nvtx3/nvToolsExt.h>

namespace {

constexpr int SM_COUNT = 148;     // B200

struct Range {
    explicit Range(const char *name) { nvtxRangePushA(name); }
    ~Range() { nvtxRangePop(); }
};

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool known(int dtype) { return dtype == SA2_F32 || dtype == SA2_BF16; }
inline int size_of(int dtype) { return dtype == SA2_BF16 ? 2 : 4; }
inline int launch_status() { return cudaGetLastError() == cudaSuccess ? SA2_OK : SA2_ERR_CUDA; }
inline cudaStream_t stream_of(void *s) { return reinterpret_cast<cudaStream_t>(s); }

// Dynamic shared memory that kernels of varying needs are allowed: one number, since two threads may be between this and their launches
constexpr int SMEM_LIMIT = 200 * 1024;
template <typename K> bool allow_smem(K kernel, size_t smem) {
    return smem <= (size_t)SMEM_LIMIT && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT) == cudaSuccess;
}

template <typename K, typename... Args>
int launch_clusters(K kernel, int64_t grid, int threads, size_t smem, int ctas, cudaStream_t st, const Args &...args) {
    if (!allow_smem(kernel, smem)) return SA2_ERR_CUDA;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)grid); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cfg.attrs = attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? SA2_OK : SA2_ERR_CUDA;
}

// ---------------------------------------------------------------- queries and keys
bool rotary_strides_ok(const sa2_strides &s, int dtype) {
    const int piece = 16 / size_of(dtype);
    return s.batch % piece == 0 && s.seq % piece == 0 && s.head % piece == 0;
}

int rotary_check(const sa2_rotary_args *a, bool backward) {
    if (!a || a->b <= 0 || a->n <= 0 || a->q.heads <= 0 || a->k.heads <= 0 || !a->freqs) return SA2_ERR_INVALID;
    if (!known(a->dtype) || !known(a->gain_dtype)) return SA2_ERR_UNSUPPORTED;
    if (a->d != 32 && a->d != 64 && a->d != 128 && a->d != 256) return SA2_ERR_UNSUPPORTED;
    if (a->pairs <= 0 || a->pairs % 8 || 2 * a->pairs > a->d) return SA2_ERR_UNSUPPORTED;
    if ((int64_t)a->b * a->n > 1 << 30 || (int64_t)a->q.heads + a->k.heads > 4096) return SA2_ERR_UNSUPPORTED;
    for (const sa2_rotary_side *s : {&a->q, &a->k}) {
        if (!s->x || !s->y || !s->gain || !aligned16(s->x) || !aligned16(s->y) || !aligned16(s->gain) || !rotary_strides_ok(s->sx, a->dtype)) return SA2_ERR_INVALID;
        if (backward && (!s->dy || !s->dgain || !aligned16(s->dy) || !rotary_strides_ok(s->sdy, a->dtype))) return SA2_ERR_INVALID;
    }
    return SA2_OK;
}

sa2::rotary::Params rotary_params(const sa2_rotary_args *a) {
    auto side = [](const sa2_rotary_side &s) {
        return sa2::rotary::Side{s.x, s.dy, s.sx.batch, s.sx.seq, s.sx.head, s.sdy.batch, s.sdy.seq, s.sdy.head, s.y, s.gain};
    };
    sa2::rotary::Params P{};
    P.q = side(a->q); P.k = side(a->k);
    P.freqs = a->freqs; P.positions = a->positions; P.pb = a->pos_batch; P.pn = a->pos_seq; P.start = a->start;
    P.partial = reinterpret_cast<float *>(a->partial);
    P.rows = a->b * a->n; P.n = a->n;
    P.hq = a->q.heads; P.heads = a->q.heads + a->k.heads; P.pairs = a->pairs;
    sa2::rotary::split(P.rows, P.heads, a->d, SM_COUNT, P.parts, P.turns);
    P.gain_bf16 = a->gain_dtype == SA2_BF16; P.eps = a->eps;
    return P;
}

template <typename T, int D> int rotary_run(const sa2::rotary::Params &P, const sa2_rotary_args *a, bool backward) {
    using namespace sa2::rotary;
    cudaStream_t st = stream_of(a->stream);
    if (!backward) {
        const auto run = a->interleaved ? fwd_kernel<T, D, true> : fwd_kernel<T, D, false>;
        run<<<grid((int64_t)P.rows * P.parts, FWD_CTAS<T> * SM_COUNT), THREADS, fwd_smem(P.pairs), st>>>(P);
        return launch_status();
    }
    const int ctas = grid((int64_t)P.rows * P.parts, BWD_CTAS<T> * SM_COUNT);
    const auto run = a->interleaved ? bwd_kernel<T, D, true> : bwd_kernel<T, D, false>;
    run<<<ctas, THREADS, bwd_smem(P.pairs), st>>>(P);
    if (int e = launch_status()) return e;
    const dim3 sums(D / 32, 2);
    if (a->gain_dtype == SA2_BF16)
        dgain_kernel<__nv_bfloat16><<<sums, 1024, 0, st>>>(P.partial, reinterpret_cast<__nv_bfloat16 *>(a->q.dgain), reinterpret_cast<__nv_bfloat16 *>(a->k.dgain), ctas, D);
    else dgain_kernel<float><<<sums, 1024, 0, st>>>(P.partial, reinterpret_cast<float *>(a->q.dgain), reinterpret_cast<float *>(a->k.dgain), ctas, D);
    return launch_status();
}

template <typename T> int rotary_dispatch(const sa2_rotary_args *a, bool backward) {
    const sa2::rotary::Params P = rotary_params(a);
    switch (a->d) {
        case 32: return rotary_run<T, 32>(P, a, backward);
        case 64: return rotary_run<T, 64>(P, a, backward);
        case 128: return rotary_run<T, 128>(P, a, backward);
        default: return rotary_run<T, 256>(P, a, backward);
    }
}

// ---------------------------------------------------------------- embedding
int embed_check(const sa2_embed_args *a) {
    if (!a || !a->tokens || a->rows <= 0 || a->vocab <= 0 || a->n <= 0 || a->dim <= 0) return SA2_ERR_INVALID;
    if (!known(a->dtype) || a->rows > INT32_MAX || a->vocab > INT32_MAX || a->dim > 1 << 30) return SA2_ERR_UNSUPPORTED;
    if (a->start < 0 || a->rows % a->n) return SA2_ERR_INVALID;
    // (start + n may be above 2^63)
    if ((a->positions || a->dpositions) && (a->position_rows < a->n || a->position_rows - a->n < a->start)) return SA2_ERR_INVALID;
    return SA2_OK;
}

// pieces of a row: 256 channels in 16-byte accesses, or 128 one by one
inline int embed_tiles(int dim, bool vec) { return vec ? (dim + 255) / 256 : (dim + 127) / 128; }

template <typename T> int embed_fwd(const sa2_embed_args *a) {
    using namespace sa2::embed;
    const Params P{a->tokens, a->tokens64, a->weight, a->positions, a->out, a->rows, a->vocab, a->start, a->n, a->dim, a->scale};
    const bool vec = a->dim % 8 == 0 && aligned16(a->weight) && aligned16(a->out) && aligned16(a->positions);
    const int tiles = embed_tiles(a->dim, vec);
    const int64_t ctas = ((a->rows + ROWS<T> - 1) / ROWS<T> * tiles + THREADS / 32 - 1) / (THREADS / 32);
    if (ctas > INT32_MAX) return SA2_ERR_UNSUPPORTED;
    const auto run = vec ? fwd_kernel<T, 8> : fwd_kernel<T, 4>;
    run<<<(unsigned)ctas, THREADS, 0, stream_of(a->stream)>>>(P, tiles);
    return launch_status();
}

template <typename T, int V> int embed_bwd_run(sa2::embed::BwdParams P, cudaStream_t st) {
    using namespace sa2::embed;
    P.tiles = embed_tiles(P.dim, V == 8);
    const int sorting = P.dweight ? sort_ctas(P.rows) : 0, cluster = sorting ? sorting : 1;
    // the others: a warp for 256 channels of a row of dP
    const int64_t most = others_at_most(cluster, SM_COUNT), adding = P.dpositions ? (P.position_rows * P.tiles + SORT_WARPS - 1) / SORT_WARPS : 0;
    P.zeroing = P.dweight ? zero_ctas(P.rows, P.vocab, P.dim * (int64_t)sizeof(T), (int)most) : 0;
    int64_t others = adding < most ? adding : most;
    if (others < P.zeroing) others = P.zeroing;
    others = (others + cluster - 1) / cluster * cluster;
    if (int e = launch_clusters(sort_kernel<T, V>, sorting + others, SORT_THREADS, sort_smem(P.bits), cluster, st, P, sorting)) return e;
    if (!P.dweight) return SA2_OK;
    const int64_t parts = stretches(P.rows), units = parts * P.tiles;
    if ((units + 7) / 8 > INT32_MAX || parts * P.tiles > INT32_MAX) return SA2_ERR_UNSUPPORTED;
    sum_kernel<T, V><<<(unsigned)((units + 7) / 8), THREADS, 0, st>>>(P, parts);
    if (int e = launch_status()) return e;
    if (parts > 1) join_kernel<T, V><<<(unsigned)(parts * P.tiles), THREADS, 0, st>>>(P);
    return launch_status();
}

template <typename T> int embed_bwd(const sa2_embed_args *a) {
    using namespace sa2::embed;
    BwdParams P{};
    P.tokens = a->tokens; P.tokens64 = a->tokens64; P.dout = a->dout; P.dweight = a->dweight; P.dpositions = a->dpositions;
    if (a->dweight) {
        char *ws = reinterpret_cast<char *>(a->workspace);
        const size_t list = up256((size_t)a->rows * 4);
        for (int s = 0; s < 2; ++s) {
            P.key[s] = reinterpret_cast<uint32_t *>(ws + 2 * s * list);
            P.place[s] = reinterpret_cast<uint32_t *>(ws + (2 * s + 1) * list);
        }
        P.partial = reinterpret_cast<float *>(ws + 4 * list);
    }
    P.rows = a->rows; P.vocab = a->vocab; P.padding = a->padding; P.start = a->start; P.position_rows = a->position_rows;
    P.n = a->n; P.dim = a->dim; P.scale = a->scale;
    sort_plan(a->vocab, P.passes, P.bits);
    const bool vec = a->dim % 8 == 0 && aligned16(a->dout) && aligned16(a->dweight) && aligned16(a->dpositions);
    return vec ? embed_bwd_run<T, 8>(P, stream_of(a->stream)) : embed_bwd_run<T, 4>(P, stream_of(a->stream));
}

// ---------------------------------------------------------------- distillation
int distill_check(const sa2_distill_args *a, bool forward, bool backward) {
    if (!a || !a->logits || a->rows <= 0 || a->vocab <= 0 || a->k <= 0) return SA2_ERR_INVALID;
    if (forward && (!a->teacher || !a->index || (!a->row_loss && !a->total))) return SA2_ERR_INVALID;
    if (backward && !a->dlogits) return SA2_ERR_INVALID;
    if (!known(a->dtype) || !known(a->teacher_dtype) || a->k > sa2::distill::MAX_K || a->rows > INT32_MAX || a->vocab > 1 << 30) return SA2_ERR_UNSUPPORTED;
    if (a->reduction != SA2_SUM && a->reduction != SA2_MEAN) return SA2_ERR_UNSUPPORTED;
    // (log2(e) / T is an fp32 number in the kernels)
    if (!(a->temperature > 4.5e-39f) || a->temperature * 0.f != 0.f) return SA2_ERR_INVALID;
    const uintptr_t unit = size_of(a->dtype) - 1;
    if ((reinterpret_cast<uintptr_t>(a->logits) & unit) || (backward && (reinterpret_cast<uintptr_t>(a->dlogits) & unit))) return SA2_ERR_INVALID;
    if (!a->workspace || (reinterpret_cast<uintptr_t>(a->workspace) & 255u) || a->workspace_bytes < sa2_distill_workspace_bytes(a->rows, a->k))
        return SA2_ERR_WORKSPACE;
    return SA2_OK;
}

sa2::distill::Params distill_params(const sa2_distill_args *a) {
    sa2::distill::Params P{};
    P.z = a->logits; P.teacher = a->teacher; P.index = a->index;
    P.dz = a->dlogits; P.gout = a->gout; P.gs = a->gout_rows != 0;
    P.mean = a->reduction == SA2_MEAN;
    P.times = a->grad_scale;
    P.rows = a->rows; P.zs = a->logits_stride; P.ts = a->teacher_stride; P.is = a->index_stride; P.ds = a->dlogits_stride;
    P.vocab = a->vocab; P.k = a->k; P.index64 = a->index64; P.teacher_bf16 = a->teacher_dtype == SA2_BF16; P.t = a->temperature;
    const double c = 1.4426950408889634 / (double)a->temperature;
    P.hi = (float)c; P.lo = (float)(c - (double)P.hi);
    sa2::distill::carve(P, a->workspace);
    if (a->row_loss) P.row_loss = a->row_loss;
    return P;
}

// Threads of a row, by its bytes: what a CTA does once costs every warp alike, and more rows at a time wait for one another.  Loss and gradient at
// once, with 128, 256 and 512 threads: 136, 187 and 305 us (16384 rows of 4096 bf16 logits), 162, 170 and 218 (8192 of 10000 fp32), 275, 240
// and 276 (8192 of 32000 bf16), 285, 256 and 234 (4095 of 32000 fp32), 563, 520 and 476 (4096 of 128000 bf16).  Short rows have a warp.
template <typename T> inline int distill_threads(int vocab) {
    const int64_t bytes = (int64_t)vocab * sizeof(T);
    return vocab <= 2048 ? 32 : bytes <= 48 * 1024 ? 128 : bytes <= 112 * 1024 ? 256 : 512;
}

template <typename T> int distill_bwd(const sa2_distill_args *a) {
    sa2::distill::Params P = distill_params(a);
    if (!P.mean || a->gout_rows) P.scale = nullptr;
    cudaStream_t st = stream_of(a->stream);
    const int g = distill_threads<T>(a->vocab);
    if (g == 32) sa2::distill::bwd_kernel<T, 32><<<(unsigned)((a->rows + 7) / 8), 256, 0, st>>>(P);
    else if (g == 128) sa2::distill::bwd_kernel<T, 128><<<(unsigned)a->rows, 128, 0, st>>>(P);
    else if (g == 256) sa2::distill::bwd_kernel<T, 256><<<(unsigned)a->rows, 256, 0, st>>>(P);
    else sa2::distill::bwd_kernel<T, 512><<<(unsigned)a->rows, 512, 0, st>>>(P);
    return launch_status();
}

// The forward; with `grad` also the gradient.
template <typename T> int distill_fwd(const sa2_distill_args *a, bool grad) {
    const sa2::distill::Params P = distill_params(a);
    cudaStream_t st = stream_of(a->stream);
    using namespace sa2::distill;
    const int warps = teacher_warps(a->k);
    const size_t smem = (size_t)warps * teacher_words(a->k) * 4;
    if (!allow_smem(teacher_kernel, smem)) return SA2_ERR_CUDA;
    teacher_kernel<<<(unsigned)teacher_blocks(a->rows), 32 * warps, smem, st>>>(P);
    if (int e = launch_status()) return e;
    const int g = distill_threads<T>(a->vocab);
    const bool both = grad && g > 32;
    const unsigned rows = (unsigned)a->rows;
    if (g == 32) fwd_kernel<T, 32><<<(rows + 7) / 8, 256, 0, st>>>(P);
    else if (g == 128) both ? both_kernel<T, 128><<<rows, 128, 0, st>>>(P) : fwd_kernel<T, 128><<<rows, 128, 0, st>>>(P);
    else if (g == 256) both ? both_kernel<T, 256><<<rows, 256, 0, st>>>(P) : fwd_kernel<T, 256><<<rows, 256, 0, st>>>(P);
    else both ? both_kernel<T, 512><<<rows, 512, 0, st>>>(P) : fwd_kernel<T, 512><<<rows, 512, 0, st>>>(P);
    if (int e = launch_status()) return e;
    if (a->total) {
        total_kernel<<<1, 1024, 0, st>>>(P.row_loss, P.counts, a->rows, P.mean, a->total, P.scale);
        if (int e = launch_status()) return e;
    }
    return grad && !both ? distill_bwd<T>(a) : SA2_OK;
}

// ---------------------------------------------------------------- sampling
template <typename T, bool RESIDENT, int N> int sample_launch(const sa2::sample::Params &P, int ctas, cudaStream_t st) {
    using namespace sa2::sample;
    const size_t behind = RESIDENT ? (size_t)P.slice : (size_t)WARPS<N> * RING * 128;
    return launch_clusters(kernel<T, RESIDENT, N>, P.rows * ctas, N, sizeof(Shared<N>) + behind * sizeof(T), ctas, st, P);
}
template <typename T> int sample_run(const sa2::sample::Params &P, int ctas, cudaStream_t st) {
    // many short rows: small CTAs, whose waits overlap
    if (ctas == 1 && P.vocab <= sa2::sample::SHORT && P.rows > SM_COUNT) return sample_launch<T, true, 128>(P, ctas, st);
    // two CTAs an SM; rows that do not fit are read from memory again
    if (sizeof(sa2::sample::Shared<512>) + (size_t)P.slice * sizeof(T) <= 112 * 1024) return sample_launch<T, true, 512>(P, ctas, st);
    return sample_launch<T, false, 512>(P, ctas, st);
}

}  // namespace

extern "C" {

size_t sa2_rotary_partial_bytes(const sa2_rotary_args *a) {
    if (!a || a->b <= 0 || a->n <= 0 || a->q.heads <= 0 || a->k.heads <= 0 || a->d <= 0 || a->pairs <= 0) return 0;
    int parts, turns;
    sa2::rotary::split((int64_t)a->b * a->n, a->q.heads + a->k.heads, a->d, SM_COUNT, parts, turns);
    return (size_t)sa2::rotary::grid((int64_t)a->b * a->n * parts, 3 * SM_COUNT) * 2 * a->d * sizeof(float);
}
int sa2_rotary_fwd(const sa2_rotary_args *a) {
    Range range("sa2_rotary_fwd");
    if (int e = rotary_check(a, false)) return e;
    return a->dtype == SA2_BF16 ? rotary_dispatch<__nv_bfloat16>(a, false) : rotary_dispatch<float>(a, false);
}
int sa2_rotary_bwd(const sa2_rotary_args *a) {
    Range range("sa2_rotary_bwd");
    if (int e = rotary_check(a, true)) return e;
    if (!a->partial || !aligned16(a->partial) || a->partial_bytes < sa2_rotary_partial_bytes(a)) return SA2_ERR_WORKSPACE;
    return a->dtype == SA2_BF16 ? rotary_dispatch<__nv_bfloat16>(a, true) : rotary_dispatch<float>(a, true);
}

size_t sa2_embed_workspace_bytes(int64_t rows, int32_t dim) {
    return rows > 0 && dim > 0 ? sa2::embed::workspace_bytes(rows, dim) : 0;
}
int sa2_embed_fwd(const sa2_embed_args *a) {
    Range range("sa2_embed_fwd");
    if (int e = embed_check(a)) return e;
    if (!a->weight || !a->out) return SA2_ERR_INVALID;
    return a->dtype == SA2_BF16 ? embed_fwd<__nv_bfloat16>(a) : embed_fwd<float>(a);
}
int sa2_embed_bwd(const sa2_embed_args *a) {
    Range range("sa2_embed_bwd");
    if (int e = embed_check(a)) return e;
    if (!a->dout || (!a->dweight && !a->dpositions) || !aligned16(a->dweight) || !aligned16(a->dpositions)) return SA2_ERR_INVALID;
    if (a->dweight && (!a->workspace || (reinterpret_cast<uintptr_t>(a->workspace) & 255u) || a->workspace_bytes < sa2_embed_workspace_bytes(a->rows, a->dim)))
        return SA2_ERR_WORKSPACE;
    return a->dtype == SA2_BF16 ? embed_bwd<__nv_bfloat16>(a) : embed_bwd<float>(a);
}

size_t sa2_distill_workspace_bytes(int64_t rows, int32_t k) {
    return rows > 0 && k > 0 ? sa2::distill::workspace_bytes(rows, k) : 0;
}
int sa2_distill_fwd(const sa2_distill_args *a) {
    Range range("sa2_distill_fwd");
    if (int e = distill_check(a, true, false)) return e;
    return a->dtype == SA2_BF16 ? distill_fwd<__nv_bfloat16>(a, false) : distill_fwd<float>(a, false);
}
int sa2_distill_bwd(const sa2_distill_args *a) {
    Range range("sa2_distill_bwd");
    if (int e = distill_check(a, false, true)) return e;
    return a->dtype == SA2_BF16 ? distill_bwd<__nv_bfloat16>(a) : distill_bwd<float>(a);
}
int sa2_distill_both(const sa2_distill_args *a) {
    Range range("sa2_distill_both");
    if (int e = distill_check(a, true, true)) return e;
    if (a->gout || !a->total || a->grad_scale * 0.f != 0.f) return SA2_ERR_INVALID;
    return a->dtype == SA2_BF16 ? distill_fwd<__nv_bfloat16>(a, true) : distill_fwd<float>(a, true);
}

int sa2_sample(const sa2_sample_args *a) {
    Range range("sa2_sample");
    if (!a || !a->logits || !a->uniform || !a->token || a->rows <= 0 || a->vocab <= 0) return SA2_ERR_INVALID;
    if (!known(a->dtype) || a->vocab > 1 << 30) return SA2_ERR_UNSUPPORTED;
    if (reinterpret_cast<uintptr_t>(a->logits) & (size_of(a->dtype) - 1)) return SA2_ERR_INVALID;
    namespace sm = sa2::sample;
    sm::Params P{};
    P.z = a->logits; P.uniform = a->uniform; P.temperature = a->temperature; P.top_p = a->top_p; P.min_p = a->min_p; P.top_k = a->top_k;
    P.token = a->token; P.logprob = a->logprob; P.rows = a->rows; P.zs = a->logits_stride;
    P.top_k_all = a->top_k_all; P.temperature_all = a->temperature_all; P.top_p_all = a->top_p_all; P.min_p_all = a->min_p_all;
    P.vocab = a->vocab; P.uniform64 = a->uniform64;
    const int ctas = sm::ctas_of(a->rows, a->vocab, SM_COUNT);
    P.slice = sm::slice_of(a->vocab, ctas);
    P.shift = sm::mass_shift(a->vocab);
    if (a->rows * ctas > INT32_MAX) return SA2_ERR_UNSUPPORTED;
    return a->dtype == SA2_BF16 ? sample_run<__nv_bfloat16>(P, ctas, stream_of(a->stream)) : sample_run<float>(P, ctas, stream_of(a->stream));
}

}  // extern "C"
