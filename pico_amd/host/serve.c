/*
 * pico_amd/host/serve.c -- rotary positions, and causal attention token by token: a paged
 * cache of keys and values in 8 bits and the attention over it, in pico's op style
 * (src/ops.c:12-54) over GPU tensors.
 *
 * No reference code exists for these.  The positions' backward hook keeps the += contract
 * of src/autograd.h:25-29; attention over the cache has none.
 */
#include <math.h>
#include <stdlib.h>
#include <string.h>

#include "pk_host.h"

/* ------------------------------------------------------- rotary positions */
struct PicoRope {
    PkRope args;
};

struct PicoRope* pico_rope_init(const struct PicoRopeConfig* cfg) {
    if(!cfg || cfg->rot < 2 || cfg->rot % 2 || cfg->rot > 1024) {
        PKH_ERR("rope_init expects an even number of values to turn, 2 to 1024!\n");
        return NULL;
    }
    double freqs[512];
    int st = pk_rope_freqs(cfg->rot, cfg->base, cfg->scaling, cfg->factor, cfg->length, cfg->low,
                           cfg->high, freqs);
    if(pkh_status("pico_rope_init", st)) return NULL;
    const double m = cfg->magnitude == 0.0f ? 1.0 : (double)cfg->magnitude;
    if(!isfinite(m)) {
        PKH_ERR("rope_init expects a finite magnitude!\n");
        return NULL;
    }
    struct PicoRope* r = (struct PicoRope*)calloc(1, sizeof(*r));
    if(!r) return NULL;
    const size_t bytes = sizeof(double) * (size_t)(cfg->rot / 2);
    double* dev = pkh_init() ? NULL : (double*)pkh_device_alloc(bytes);
    if(!dev || pkh_upload(dev, freqs, bytes)) {
        if(dev) pkh_device_free(dev);
        free(r);
        return NULL;
    }
    r->args.freqs = dev;
    r->args.rot = cfg->rot;
    r->args.interleaved = cfg->interleaved != 0;
    r->args.magnitude = m;
    return r;
}

void pico_rope_free(struct PicoRope* r) {
    if(!r) return;
    pkh_sync(); /* a launch may still read the frequencies */
    pkh_device_free((void*)r->args.freqs);
    free(r);
}

static int head_rows(const struct PicoTensor* t, int64_t heads) {
    return heads >= 1 && t->ndim == 2 && t->strides[1] == 1 && t->shape[1] >= heads &&
           t->shape[1] % heads == 0 && t->strides[0] >= t->shape[1];
}

enum { ROPE_ARGS = 0, ROPE_POS = 1 };
enum { ROPE_H = 0 };

static void rope_backward(struct PicoTensor* self) {
    struct PkNode* n = pkh_node(self);
    struct PicoTensor* x = self->parents[0];
    const float* g = pkh_upstream(self);
    if(!g) return;
    const int64_t N = x->shape[0], C = x->shape[1], H = n->ival[ROPE_H];
    const int flags = PK_ROPE_BACKWARD | (pkh_grad_flag(x) ? PK_ACCUM : 0);
    int st = pk_rope_f32(N, H, C / H, (const PkRope*)n->saved[ROPE_ARGS],
                         (const int32_t*)n->saved[ROPE_POS], g, C, x->grad, x->strides[0], flags,
                         pkh_stream());
    if(pkh_status("pico_rope_backward", st)) return;
    pkh_grad_mark(x);
}

struct PicoTensor* pico_rope(struct PicoTensor* x, const struct PicoRope* rope,
                             const int32_t* positions, int n_heads) {
    if(pkh_need_gpu("pico_rope", x)) return NULL;
    if(!rope || !positions || !head_rows(x, n_heads) || x->shape[1] / n_heads < rope->args.rot) {
        PKH_ERR("rope expects x [rows, heads*hd] with unit columns and heads of at least the values "
                "to turn, a rope and a position for every row!\n");
        return NULL;
    }
    struct Arena* arena = pkh_need_arena();
    if(!arena) return NULL;
    const int64_t N = x->shape[0], C = x->shape[1];
    const int32_t* pos = pkh_ids_on_device(positions, N);
    if(!pos) return NULL;
    struct PicoTensor* out = pkh_new_tensor(arena, x->shape, 2);
    if(!out) return NULL;
    PkRope* args = (PkRope*)arena_alloc(arena, sizeof(*args));
    if(!args) return NULL;
    *args = rope->args;
    int st = pk_rope_f32(N, n_heads, C / n_heads, args, pos, x->data, x->strides[0], out->data, C, 0,
                         pkh_stream());
    if(pkh_status("pico_rope", st)) return NULL;
    struct PkNode* n = pkh_node(out);
    n->saved[ROPE_ARGS] = args;
    n->saved[ROPE_POS] = (void*)pos;
    n->ival[ROPE_H] = n_heads;
    pkh_set_parents(arena, out, 1, &x, rope_backward);
    return out;
}

/* ---------------------------------------------------------- the paged cache
 * The pages of all layers are numbered alike: page p of a sequence is page p of every
 * layer's pools.  The host keeps the sequences' pages and lengths, and uploads them where
 * a step begins: `words` on the host and the device hold lens [S], offsets [S + 1] and the
 * table [S][width]. */
struct PicoKV {
    PkKvCache* layers;
    int n_layers, S;
    int64_t width, max_length, pages, free_pages;
    int32_t* free_list;    /* free_pages of them */
    int64_t* length;       /* tokens of each sequence, the present step's among them */
    int32_t *words, *dev;
    size_t n_words;
    int64_t rows;          /* of the present step; -1 before the first */
};

static int32_t* kv_lens(struct PicoKV* kv) { return kv->words; }
static int32_t* kv_offsets(struct PicoKV* kv) { return kv->words + kv->S; }
static int32_t* kv_table(struct PicoKV* kv, int b) {
    return kv->words + 2 * kv->S + 1 + (int64_t)b * kv->width;
}

void pico_kv_free(struct PicoKV* kv) {
    if(!kv) return;
    pkh_sync(); /* a launch may still read the cache */
    for(int i = 0; kv->layers && i < kv->n_layers; i++) {
        if(kv->layers[i].k) pkh_device_free(kv->layers[i].k);
        if(kv->layers[i].v) pkh_device_free(kv->layers[i].v);
        if(kv->layers[i].k_exp) pkh_device_free(kv->layers[i].k_exp);
        if(kv->layers[i].v_exp) pkh_device_free(kv->layers[i].v_exp);
    }
    if(kv->dev) pkh_device_free(kv->dev);
    free(kv->layers);
    free(kv->free_list);
    free(kv->length);
    free(kv->words);
    free(kv);
}

struct PicoKV* pico_kv_init(const struct PicoKVConfig* cfg) {
    const int hp = cfg ? (int)pk_kv_head_size(cfg->head_dim) : 0;
    if(!hp || cfg->layers < 1 || cfg->kv_heads < 1 || cfg->kv_heads > 4096 || cfg->pages < 1 ||
       cfg->sequences < 1 || cfg->sequences > 1 << 20 || cfg->max_length < 1 ||
       cfg->max_length >= 1 << 30 ||
       (cfg->page != 16 && cfg->page != 32 && cfg->page != 64 && cfg->page != 128)) {
        PKH_ERR("kv_init expects layers, pages, sequences and max_length (below 2^30) of at least 1, 1 "
                "to 4096 kv_heads, head_dim 1 to 256 and pages of 16, 32, 64 or 128 tokens!\n");
        return NULL;
    }
    if(pkh_init()) return NULL;
    struct PicoKV* kv = (struct PicoKV*)calloc(1, sizeof(*kv));
    if(!kv) return NULL;
    kv->n_layers = cfg->layers;
    kv->S = cfg->sequences;
    kv->pages = kv->free_pages = cfg->pages;
    kv->max_length = cfg->max_length;
    kv->width = (kv->max_length + cfg->page - 1) / cfg->page;
    kv->rows = -1;
    kv->n_words = 2 * (size_t)kv->S + 1 + (size_t)kv->S * (size_t)kv->width;
    kv->layers = (PkKvCache*)calloc((size_t)kv->n_layers, sizeof(PkKvCache));
    kv->free_list = (int32_t*)malloc(sizeof(int32_t) * (size_t)kv->pages);
    kv->length = (int64_t*)calloc((size_t)kv->S, sizeof(int64_t));
    kv->words = (int32_t*)calloc(kv->n_words, sizeof(int32_t));
    kv->dev = kv->words ? (int32_t*)pkh_device_alloc(sizeof(int32_t) * kv->n_words) : NULL;
    int ok = kv->layers && kv->free_list && kv->length && kv->dev;
    const size_t heads = (size_t)kv->pages * (size_t)cfg->kv_heads;
    for(int i = 0; ok && i < kv->n_layers; i++) {
        PkKvCache* c = &kv->layers[i];
        c->k = (uint8_t*)pkh_device_alloc(heads * (size_t)cfg->page * (size_t)hp);
        c->v = c->k ? (uint8_t*)pkh_device_alloc(heads * (size_t)cfg->page * (size_t)hp) : NULL;
        c->k_exp = c->v ? (uint8_t*)pkh_device_alloc(heads) : NULL;
        c->v_exp = c->k_exp ? (uint8_t*)pkh_device_alloc(heads) : NULL;
        ok = c->v_exp != NULL;
        c->lens = kv->dev;
        c->offsets = kv->dev + kv->S;
        c->table = kv->dev + 2 * kv->S + 1;
        c->pages = kv->pages;
        c->kv_heads = cfg->kv_heads;
        c->hd = cfg->head_dim;
        c->page = cfg->page;
        c->B = kv->S;
        c->width = kv->width;
    }
    if(!ok) {
        pico_kv_free(kv);
        return NULL;
    }
    /* (the lowest pages are taken first) */
    for(int64_t i = 0; i < kv->pages; i++) kv->free_list[i] = (int32_t)(kv->pages - 1 - i);
    for(int b = 0; b < kv->S; b++)
        for(int64_t i = 0; i < kv->width; i++) kv_table(kv, b)[i] = -1;
    return kv;
}

int64_t pico_kv_begin(struct PicoKV* kv, const int32_t* new_tokens) {
    if(!kv || !new_tokens) {
        PKH_ERR("kv_begin expects a cache and how many new tokens each sequence has!\n");
        return -1;
    }
    const int64_t page = kv->layers[0].page;
    int64_t rows = 0, need = 0;
    for(int b = 0; b < kv->S; b++) {
        const int64_t n = new_tokens[b], len = kv->length[b];
        if(n < 0 || len + n > kv->max_length) {
            PKH_ERR("kv_begin: sequence %d of %lld tokens gets %lld more, up to %lld are held!\n", b,
                    (long long)len, (long long)n, (long long)kv->max_length);
            return -1;
        }
        rows += n;
        need += (len + n + page - 1) / page - (len + page - 1) / page;
    }
    if(rows >= 1 << 24) {
        PKH_ERR("kv_begin: %lld new tokens, a step has fewer than 2^24!\n", (long long)rows);
        return -1;
    }
    if(need > kv->free_pages) {
        PKH_ERR("kv_begin: %lld new pages are needed, %lld are free!\n", (long long)need,
                (long long)kv->free_pages);
        return -1;
    }
    /* (a failed upload, in a graph capture for instance, must leave the cache as it was) */
    const int64_t had_rows = kv->rows, had_free = kv->free_pages;
    int32_t* was = (int32_t*)malloc(sizeof(int32_t) * kv->n_words);
    if(!was) return -1;
    memcpy(was, kv->words, sizeof(int32_t) * kv->n_words);
    int64_t at = 0;
    for(int b = 0; b < kv->S; b++) {
        kv_lens(kv)[b] = (int32_t)kv->length[b];
        kv_offsets(kv)[b] = (int32_t)at;
        at += new_tokens[b];
        for(int64_t i = (kv->length[b] + page - 1) / page; i < (kv->length[b] + new_tokens[b] + page - 1) / page; i++)
            kv_table(kv, b)[i] = kv->free_list[--kv->free_pages];
    }
    kv_offsets(kv)[kv->S] = (int32_t)at;
    /* the table too where a sequence got a page, or gave its pages back */
    const size_t head = 2 * (size_t)kv->S + 1;
    const int table = kv->rows < 0 || memcmp(was + head, kv->words + head, sizeof(int32_t) * (kv->n_words - head));
    if(pkh_upload(kv->dev, kv->words, sizeof(int32_t) * (table ? kv->n_words : head))) {
        memcpy(kv->words, was, sizeof(int32_t) * kv->n_words);
        kv->free_pages = had_free;
        kv->rows = had_rows;
        free(was);
        return -1;
    }
    free(was);
    for(int b = 0; b < kv->S; b++) kv->length[b] += new_tokens[b];
    kv->rows = rows;
    return rows;
}

int64_t pico_kv_length(const struct PicoKV* kv, int sequence) {
    return kv && sequence >= 0 && sequence < kv->S ? kv->length[sequence] : -1;
}

int pico_kv_drop(struct PicoKV* kv, int sequence) {
    if(!kv || sequence < 0 || sequence >= kv->S) {
        PKH_ERR("kv_drop expects a cache and one of its sequences!\n");
        return PK_EINVAL;
    }
    const int64_t page = kv->layers[0].page, n = (kv->length[sequence] + page - 1) / page;
    /* (in the order that gives the same pages again) */
    for(int64_t i = n - 1; i >= 0; i--) kv->free_list[kv->free_pages++] = kv_table(kv, sequence)[i];
    kv->length[sequence] = 0;
    kv->rows = -1; /* what the device knows of the pages is from before */
    return 0;
}

struct PicoTensor* pico_attention_cached(struct PicoKV* kv, int layer, struct PicoTensor* q,
                                         struct PicoTensor* k, struct PicoTensor* v, int n_heads,
                                         const struct PicoRope* rope) {
    if(pkh_need_gpu("pico_attention_cached", q) || pkh_need_gpu("pico_attention_cached", k) ||
       pkh_need_gpu("pico_attention_cached", v))
        return NULL;
    if(!kv || layer < 0 || layer >= kv->n_layers || kv->rows < 0) {
        PKH_ERR("attention_cached expects a cache whose step has begun, and one of its layers!\n");
        return NULL;
    }
    const PkKvCache* c = &kv->layers[layer];
    const int64_t N = kv->rows, hd = c->hd, H = n_heads;
    if(H < 1 || H % c->kv_heads || !head_rows(q, H) || !head_rows(k, c->kv_heads) ||
       !head_rows(v, c->kv_heads) || q->shape[0] != N || k->shape[0] != N || v->shape[0] != N ||
       q->shape[1] != H * hd || k->shape[1] != c->kv_heads * hd || v->shape[1] != c->kv_heads * hd) {
        PKH_ERR("attention_cached expects q [rows, heads*%lld], k and v [rows, %lld*%lld] with unit "
                "columns for the step's %lld rows, heads a multiple of kv_heads!\n",
                (long long)hd, (long long)c->kv_heads, (long long)hd, (long long)N);
        return NULL;
    }
    if(rope && rope->args.rot > hd) {
        PKH_ERR("attention_cached: the rope turns %lld values, heads have %lld!\n",
                (long long)rope->args.rot, (long long)hd);
        return NULL;
    }
    struct Arena* arena = pkh_need_arena();
    if(!arena) return NULL;
    int64_t shape[2] = {N, H * hd};
    struct PicoTensor* out = pkh_new_tensor(arena, shape, 2);
    if(!out) return NULL;
    float* turned = NULL;
    if(rope) {
        turned = (float*)arena_alloc_device(arena, sizeof(float) * (size_t)(N > 0 ? N * H * hd : 1));
        if(!turned) return NULL;
    }
    const size_t ws_bytes = pk_attn_paged_workspace(c, N, H);
    void* ws = ws_bytes ? arena_alloc_device(arena, ws_bytes) : NULL;
    if(ws_bytes && !ws) return NULL;
    int st = pk_kv_append_f32(c, N, k->data, k->strides[0], v->data, v->strides[0],
                              rope ? &rope->args : NULL, H, rope ? q->data : NULL, q->strides[0], turned,
                              H * hd, pkh_stream());
    if(pkh_status("pico_attention_cached", st)) return NULL;
    st = pk_attn_paged_f32(c, N, H, 1.0f / sqrtf((float)hd), rope ? turned : q->data,
                           rope ? H * hd : q->strides[0], out->data, H * hd, ws, ws_bytes, pkh_stream());
    if(pkh_status("pico_attention_cached", st)) return NULL;
    return out;
}
