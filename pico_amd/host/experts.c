/*
 * pico_amd/host/experts.c -- a mixture of experts in pico's op style
 * (src/ops.c:12-54) over GPU tensors: the top-k router, the rows' way into and
 * out of expert order, and the products grouped by expert.
 *
 * No reference code exists for these.  How many rows an expert gets is known on
 * the device only and never read back, so a captured step replays with other
 * routings.  Backward hooks keep the += contract of src/autograd.h:25-29.
 */
#include <string.h>

#include "pk_host.h"

/* one batch's routing; lives in the arena it was made in */
struct PicoRoute {
    int64_t R, k, E;                       /* tokens, choices a token, experts */
    int32_t *experts, *offsets, *order, *place; /* device: [R*k], [E+1], [R*k], [R*k] */
};

static int rows_of(const struct PicoTensor* t, int64_t rows) {
    return t->ndim == 2 && t->shape[0] == rows && t->strides[1] == 1 && t->shape[1] >= 1 &&
           t->strides[0] >= t->shape[1];
}

/* ------------------------------------------------------------- the router
 * gates [R, k] = softmax over the k largest of the E logits */
enum { RS_ROUTE = 0, ES_ARENA = 1, ES_WS = 2 };

static void route_backward(struct PicoTensor* self) {
    const struct PicoRoute* r = (const struct PicoRoute*)pkh_node(self)->saved[RS_ROUTE];
    struct PicoTensor* z = self->parents[0];
    const float* g = pkh_upstream(self);
    if(!g) return;
    int st = pk_route_topk_bwd_f32(r->R, r->E, r->k, r->experts, self->data, g, z->grad,
                                   z->strides[0], pkh_grad_flag(z), pkh_stream());
    if(pkh_status("pico_route_topk_backward", st)) return;
    pkh_grad_mark(z);
}

struct PicoTensor* pico_route_topk(struct PicoTensor* logits, int k, struct PicoRoute** route) {
    if(pkh_need_gpu("pico_route_topk", logits)) return NULL;
    if(!route || logits->ndim != 2 || !rows_of(logits, logits->shape[0]) || k < 1 ||
       k > logits->shape[1]) {
        PKH_ERR("route_topk expects logits [tokens, experts] with unit columns, 1 <= k <= experts "
                "and where to put the route!\n");
        return NULL;
    }
    *route = NULL;
    struct Arena* arena = pkh_need_arena();
    if(!arena) return NULL;
    const int64_t R = logits->shape[0], E = logits->shape[1], n = R * k;
    int64_t shape[2] = {R, k};
    struct PicoTensor* out = pkh_new_tensor(arena, shape, 2);
    if(!out) return NULL;
    struct PicoRoute* r = (struct PicoRoute*)arena_alloc(arena, sizeof(*r));
    if(!r) return NULL;
    r->R = R;
    r->k = k;
    r->E = E;
    const size_t slots = sizeof(int32_t) * (size_t)(n > 0 ? n : 1);
    r->experts = (int32_t*)arena_alloc_device(arena, slots);
    r->order = (int32_t*)arena_alloc_device(arena, slots);
    r->place = (int32_t*)arena_alloc_device(arena, slots);
    r->offsets = (int32_t*)arena_alloc_device(arena, sizeof(int32_t) * (size_t)(E + 1));
    if(!r->experts || !r->order || !r->place || !r->offsets) return NULL;
    const size_t ws_bytes = pk_expert_plan_workspace(n, E);
    void* ws = arena_alloc_device(arena, ws_bytes ? ws_bytes : 1);
    if(!ws) return NULL;
    int st = pk_route_topk_f32(R, E, k, logits->data, logits->strides[0], r->experts, out->data,
                               pkh_stream());
    if(pkh_status("pico_route_topk", st)) return NULL;
    st = pk_expert_plan(n, E, r->experts, r->offsets, r->order, r->place, ws, ws_bytes,
                        pkh_stream());
    if(pkh_status("pico_route_topk", st)) return NULL;
    pkh_node(out)->saved[RS_ROUTE] = r;
    pkh_set_parents(arena, out, 1, &logits, route_backward);
    *route = r;
    return out;
}

int pico_route_to_host(const struct PicoRoute* r, int32_t* experts, int32_t* offsets) {
    if(!r) {
        PKH_ERR("route_to_host: NULL route!\n");
        return PK_EINVAL;
    }
    if(experts && pkh_copy_d2h(experts, r->experts, sizeof(int32_t) * (size_t)(r->R * r->k)))
        return PK_EINVAL;
    if(offsets && pkh_copy_d2h(offsets, r->offsets, sizeof(int32_t) * (size_t)(r->E + 1)))
        return PK_EINVAL;
    return 0;
}

/* --------------------------------------------------- rows in expert order */
static void gather_backward(struct PicoTensor* self) {
    const struct PicoRoute* r = (const struct PicoRoute*)pkh_node(self)->saved[RS_ROUTE];
    struct PicoTensor* x = self->parents[0];
    const float* g = pkh_upstream(self);
    if(!g) return;
    const int64_t d = x->shape[1], ld = x->strides[0];
    const float* base = pkh_grad_base(x);
    int st = pk_expert_combine_f32(r->R, d, r->k, r->place, NULL, g, d, base, ld, x->grad, ld,
                                   pkh_stream());
    if(pkh_status("pico_expert_gather_backward", st)) return;
    pkh_grad_mark(x);
}

struct PicoTensor* pico_expert_gather(struct PicoTensor* x, const struct PicoRoute* r) {
    if(pkh_need_gpu("pico_expert_gather", x)) return NULL;
    if(!r || !rows_of(x, r->R)) {
        PKH_ERR("expert_gather expects a route and its tokens [tokens, d] with unit columns!\n");
        return NULL;
    }
    struct Arena* arena = pkh_need_arena();
    if(!arena) return NULL;
    const int64_t n = r->R * r->k, d = x->shape[1];
    int64_t shape[2] = {n, d};
    struct PicoTensor* out = pkh_new_tensor(arena, shape, 2);
    if(!out) return NULL;
    int st = pk_expert_gather_f32(n, d, r->k, r->E, r->offsets, r->order, x->data, x->strides[0],
                                  out->data, d, pkh_stream());
    if(pkh_status("pico_expert_gather", st)) return NULL;
    pkh_node(out)->saved[RS_ROUTE] = (void*)r;
    pkh_set_parents(arena, out, 1, &x, gather_backward);
    return out;
}

/* ----------------------------------------------- products grouped by expert
 * the backward uses the precision the forward ran in */
enum { EI_PREC = 0 };

static int expert_dw(struct PicoTensor* self, const float* g, int flags, pk_stream_t stream) {
    struct PkNode* n = pkh_node(self);
    const struct PicoRoute* r = (const struct PicoRoute*)n->saved[RS_ROUTE];
    const struct PicoTensor *x = self->parents[0], *w = self->parents[1];
    const int64_t rows = x->shape[0], K = w->shape[1], N = w->shape[2];
    /* (up to 64 MiB where the rows are split, so only now that there is a backward; in the
     * node's arena, so that captured graphs share none; without it the rows are not split) */
    const size_t ws_bytes = pk_gemm_experts_dw_workspace(rows, K, N, r->E);
    if(ws_bytes && !n->saved[ES_WS])
        n->saved[ES_WS] = pkh_arena_workspace_opt((struct Arena*)n->saved[ES_ARENA], ws_bytes);
    return pkh_status("pico_expert_matmul_backward",
                      pk_gemm_experts_dw_f32(rows, K, N, r->E, r->offsets, x->data, x->strides[0], g,
                                             N, w->grad, N, K * N, flags, (int)n->ival[EI_PREC],
                                             n->saved[ES_WS], n->saved[ES_WS] ? ws_bytes : 0, stream));
}

/* dW of a parameter goes to the side stream, beside dX and what follows it, in the
 * order matmul_backward_body (ops.c) explains: eagerly before dX is issued, under
 * graph capture after it, waiting for the point before it */
static void expert_matmul_backward(struct PicoTensor* self) {
    struct PkNode* n = pkh_node(self);
    const struct PicoRoute* r = (const struct PicoRoute*)n->saved[RS_ROUTE];
    struct PicoTensor *x = self->parents[0], *w = self->parents[1];
    const float* g = pkh_upstream(self);
    if(!g) return;
    const int64_t rows = x->shape[0], K = w->shape[1], N = w->shape[2];
    struct PkNode* nw = pkh_node(w);
    const int to_side = nw && w->is_persistent && !x->is_persistent;
    pk_stream_t side = to_side && !pkh_capturing() ? pkh_side_fork() : NULL;
    const int done = side != NULL;
    int st;
    if(side) {
        st = expert_dw(self, g, nw->grad_live ? PK_ACCUM : 0, side);
        nw->side_seq = pkh_side_seq();
        if(st) return;
        pkh_grad_mark(w);
    } else if(to_side) {
        pkh_side_prepare();
    }
    st = pk_gemm_experts_f32('T', rows, K, N, r->E, r->offsets, g, N, w->data, N, K * N, x->grad,
                                 x->strides[0], pkh_grad_flag(x), (int)n->ival[EI_PREC],
                                 pkh_stream());
    if(pkh_status("pico_expert_matmul_backward", st)) return;
    pkh_grad_mark(x);
    if(done) return;
    side = to_side ? pkh_side_fork() : NULL;
    if(side) {
        st = expert_dw(self, g, nw->grad_live ? PK_ACCUM : 0, side);
        nw->side_seq = pkh_side_seq();
    } else {
        st = expert_dw(self, g, pkh_grad_flag(w), pkh_stream());
    }
    if(st) return;
    pkh_grad_mark(w);
}

struct PicoTensor* pico_expert_matmul(struct PicoTensor* x, struct PicoTensor* w,
                                      const struct PicoRoute* r) {
    if(pkh_need_gpu("pico_expert_matmul", x) || pkh_need_gpu("pico_expert_matmul", w)) return NULL;
    if(!r || !rows_of(x, r->R * r->k)) {
        PKH_ERR("expert_matmul expects a route and its rows [tokens*k, K] in expert order, with "
                "unit columns!\n");
        return NULL;
    }
    if(w->ndim != 3 || w->shape[0] != r->E || w->shape[1] != x->shape[1] || w->shape[2] < 1 ||
       w->strides[2] != 1 || w->strides[1] != w->shape[2] ||
       w->strides[0] != w->shape[1] * w->shape[2]) {
        PKH_ERR("expert_matmul expects contiguous weights [experts, K, N]!\n");
        return NULL;
    }
    struct Arena* arena = pkh_need_arena();
    if(!arena) return NULL;
    const int64_t rows = x->shape[0], K = w->shape[1], N = w->shape[2];
    int64_t shape[2] = {rows, N};
    struct PicoTensor* out = pkh_new_tensor(arena, shape, 2);
    if(!out) return NULL;
    struct PkNode* n = pkh_node(out);
    const int mp = pico_get_matmul_precision();
    n->ival[EI_PREC] = mp == PICO_MATMUL_FP8 ? PICO_MATMUL_BF16 : mp;
    int st = pk_gemm_experts_f32('N', rows, N, K, r->E, r->offsets, x->data, x->strides[0], w->data,
                                 N, K * N, out->data, N, 0, (int)n->ival[EI_PREC], pkh_stream());
    if(pkh_status("pico_expert_matmul", st)) return NULL;
    n->saved[RS_ROUTE] = (void*)r;
    n->saved[ES_ARENA] = arena;
    struct PicoTensor* ps[2] = {x, w};
    pkh_set_parents(arena, out, 2, ps, expert_matmul_backward);
    return out;
}

/* ------------------------------------------- back to tokens, with the gates */
static void combine_backward(struct PicoTensor* self) {
    const struct PicoRoute* r = (const struct PicoRoute*)pkh_node(self)->saved[RS_ROUTE];
    struct PicoTensor *ys = self->parents[0], *gates = self->parents[1];
    struct PicoTensor* c = self->num_parents > 2 ? self->parents[2] : NULL;
    const float* g = pkh_upstream(self);
    if(!g) return;
    if(c && pkh_residual_backward("pico_expert_combine_backward", self, c, g)) return;
    const int64_t d = ys->shape[1];
    int flags = pkh_grad_flag(ys) ? PK_ACCUM : 0;
    if(pkh_grad_flag(gates)) flags |= PK_ACCUM2;
    int st = pk_expert_combine_bwd_f32(r->R, d, r->k, r->E, r->offsets, r->order, gates->data,
                                       ys->data, ys->strides[0], g, d, ys->grad, ys->strides[0],
                                       gates->grad, flags, pkh_stream());
    if(pkh_status("pico_expert_combine_backward", st)) return;
    pkh_grad_mark(ys);
    pkh_grad_mark(gates);
}

struct PicoTensor* pico_expert_combine(struct PicoTensor* ys, struct PicoTensor* gates,
                                       const struct PicoRoute* r, struct PicoTensor* c) {
    if(pkh_need_gpu("pico_expert_combine", ys) || pkh_need_gpu("pico_expert_combine", gates) ||
       (c && pkh_need_gpu("pico_expert_combine", c)))
        return NULL;
    if(!r || !rows_of(ys, r->R * r->k) || !rows_of(gates, r->R) || gates->shape[1] != r->k ||
       (r->R > 1 && gates->strides[0] != r->k) || pkh_one_grad(ys, gates)) {
        PKH_ERR("expert_combine expects a route, its rows [tokens*k, d] and contiguous gates "
                "[tokens, k]!\n");
        return NULL;
    }
    const int64_t R = r->R, d = ys->shape[1];
    if(c && (!rows_of(c, R) || c->shape[1] != d || (R > 1 && c->strides[0] != d))) {
        PKH_ERR("expert_combine expects a contiguous residual [tokens, d]!\n");
        return NULL;
    }
    struct Arena* arena = pkh_need_arena();
    if(!arena) return NULL;
    int64_t shape[2] = {R, d};
    struct PicoTensor* out = pkh_new_tensor(arena, shape, 2);
    if(!out) return NULL;
    int st = pk_expert_combine_f32(R, d, r->k, r->place, gates->data, ys->data, ys->strides[0],
                                   c ? c->data : NULL, d, out->data, d, pkh_stream());
    if(pkh_status("pico_expert_combine", st)) return NULL;
    pkh_node(out)->saved[RS_ROUTE] = (void*)r;
    struct PicoTensor* ps[3] = {ys, gates, c};
    pkh_set_parents(arena, out, c ? 3 : 2, ps, combine_backward);
    return out;
}
