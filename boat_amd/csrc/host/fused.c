/* fused.c - Boat-level forms of the fused operators: a dense layer with activation and residual, attention with a relative
 * position bias, distillation from a teacher's kept logits.  Each checks its tensors, hands the kernels dense operands and
 * returns new tensors; autodiff.c records them. */
#include "boat_internal.h"

#define FUSED_REFUSE(...)                                       \
    do {                                                        \
        boat_fail(BOAT_ERROR_INVALID_ARGUMENT, __VA_ARGS__);    \
        return 0;                                               \
    } while (0)

static bool is_i32(const boat_tensor_t* t, size_t n) { return t->dtype == BOAT_DTYPE_INT32 && t->nelements == n; }

/* ---- dense layer, activation, residual ---- */
static bool dense_act_shapes(const boat_dense_layer_t* layer, const boat_tensor_t* input, int act, const boat_tensor_t* residual) {
    if (act < BH_ACT_NONE || act > BH_ACT_GELU) FUSED_REFUSE("dense with activation: unknown activation %d", act);
    if (!bt_is_f32(input) || input->ndim != 2 || input->shape[1] != (int64_t)layer->input_features || input->nelements == 0)
        FUSED_REFUSE("dense with activation expects a float input of shape [rows, %zu]", layer->input_features);
    if (residual && (!bt_is_f32(residual) || residual->ndim != 2 || residual->shape[0] != input->shape[0] ||
                     residual->shape[1] != (int64_t)layer->output_features || residual->device != input->device))
        FUSED_REFUSE("dense with activation expects a residual of shape [rows, %zu] on the input's device", layer->output_features);
    return true;
}

boat_tensor_t* boat_hip_dense_act(const boat_dense_layer_t* layer, const boat_tensor_t* input, boat_hip_activation_t act,
                                  const boat_tensor_t* residual, boat_tensor_t** saved) {
    if (saved) *saved = NULL;
    if (!layer || !input || !dense_act_shapes(layer, input, (int)act, residual)) return NULL;
    const int64_t m = input->shape[0], k = input->shape[1], n = (int64_t)layer->output_features;
    const int64_t shape[] = {m, n};
    boat_tensor_t* out = bt_new_uninit(shape, 2, input->device);
    /* without a residual the output itself tells the slope of these three (relu: z > 0 where max(z, 0) > 0) */
    const bool by_output = !residual && (act == BOAT_HIP_ACT_RELU || act == BOAT_HIP_ACT_SIGMOID || act == BOAT_HIP_ACT_TANH);
    const bool keep = saved && act != BOAT_HIP_ACT_NONE && !by_output;
    boat_tensor_t* kept = keep ? bt_new_uninit(shape, 2, input->device) : NULL;
    const float* px = bt_dev_read(input);
    const float* pw = bt_dev_read(layer->weight);
    const float* pb = (layer->use_bias && layer->bias) ? bt_dev_read(layer->bias) : NULL;
    const float* pr = residual ? bt_dev_read(residual) : NULL;
    float* py = out ? bt_dev_write(out) : NULL;
    float* ps = kept ? bt_dev_write(kept) : NULL;
    if (!px || !pw || !py || (residual && !pr) || (keep && !ps) || (layer->use_bias && layer->bias && !pb) ||
        !boat_hip_ok(bh_gemm_epilogue(0, 0, m, n, k, px, k, pw, n, py, n, pb, (int)act, ps, n, pr, n), "dense with activation")) {
        boat_tensor_free(out);
        boat_tensor_free(kept);
        return NULL;
    }
    if (saved && by_output) {
        boat_tensor_ref(out);
        kept = out;
    }
    if (saved) *saved = kept;
    return out;
}

/* the layer's gradients accumulate as in boat_dense_layer_backward; *dx (NULL: not wanted) is a new tensor */
bool bt_dense_act_backward(boat_dense_layer_t* layer, int act, const boat_tensor_t* input, const boat_tensor_t* saved,
                           const boat_tensor_t* dy, boat_tensor_t** dx) {
    if (dx) *dx = NULL;
    const int64_t m = input->shape[0], k = input->shape[1], n = (int64_t)layer->output_features;
    if (!bt_is_f32(dy) || dy->ndim != 2 || dy->shape[0] != m || dy->shape[1] != n)
        FUSED_REFUSE("dense with activation backward expects a gradient of shape [%lld, %lld]", (long long)m, (long long)n);
    const bool with_bias = layer->use_bias && layer->bias;
    if (!layer->grad_weight) layer->grad_weight = boat_tensor_create_like(layer->weight);
    if (with_bias && !layer->grad_bias) layer->grad_bias = boat_tensor_create_like(layer->bias);
    boat_tensor_t* g = dx ? bt_new_like_uninit(input) : NULL;
    if ((dx && !g) || !layer->grad_weight || (with_bias && !layer->grad_bias)) {
        boat_tensor_free(g);
        return false;
    }
    const float* px = bt_dev_read(input);
    const float* pw = bt_dev_read(layer->weight);
    const float* pg = bt_dev_read(dy);
    const float* ps = saved ? bt_dev_read(saved) : NULL;
    float* pdx = g ? bt_dev_write(g) : NULL;
    /* into gradients that are still the zeros of a zero_grad the kernels write instead of adding */
    const bool fresh = bt_is_zero(layer->grad_weight) && (!with_bias || bt_is_zero(layer->grad_bias));
    float* pgw = fresh ? bt_dev_write(layer->grad_weight) : bt_dev_rw(layer->grad_weight);
    float* pgb = !with_bias ? NULL : fresh ? bt_dev_write(layer->grad_bias) : bt_dev_rw(layer->grad_bias);
    if (!px || !pw || !pg || (saved && !ps) || (g && !pdx) || !pgw || (with_bias && !pgb) ||
        !boat_hip_ok(bh_dense_act_backward(act, px, pw, ps, pg, pdx, pgw, pgb, m, k, n, fresh ? 0 : 1), "dense with activation backward")) {
        boat_tensor_free(g);
        return false;
    }
    if (dx) *dx = g;
    return true;
}

/* ---- attention with a relative position bias ---- */
static bool relative_plan(const boat_hip_relative_attention_config_t* c, const boat_tensor_t* q, const boat_tensor_t* k,
                          const boat_tensor_t* v, const boat_tensor_t* table, const boat_tensor_t* lengths, bh_relbias_attention_t* p) {
    if (!bt_is_f32(q) || !bt_is_f32(k) || !bt_is_f32(v) || q->ndim != 4 || k->ndim != 4 || !bt_same_shape(k, v) ||
        q->nelements == 0 || k->nelements == 0 || k->shape[0] != q->shape[0] || k->shape[3] != q->shape[3])
        FUSED_REFUSE("relative attention expects float tensors, query [batch, seq_q, heads, size], key and value [batch, seq_k, kv_heads, size]");
    if (!bt_is_f32(table) || table->ndim != 2 || table->shape[0] != c->num_buckets || table->shape[1] != q->shape[2])
        FUSED_REFUSE("relative attention expects a float table of shape [%d, %lld]", c->num_buckets, (long long)q->shape[2]);
    if (lengths && !is_i32(lengths, (size_t)q->shape[0])) FUSED_REFUSE("relative attention expects INT32 lengths, one per sequence");
    if (q->device != k->device || q->device != v->device) FUSED_REFUSE("relative attention expects query, key and value on one device");
    const int64_t h = q->shape[2], g = k->shape[2], d = q->shape[3];
    const bh_relbias_attention_t plan = {
        .batch = q->shape[0], .heads = h, .kv_heads = g, .sq = q->shape[1], .sk = k->shape[1], .d = d,
        .q_stride = {q->shape[1] * h * d, d, h * d}, .k_stride = {k->shape[1] * g * d, d, g * d},
        .v_stride = {k->shape[1] * g * d, d, g * d}, .o_stride = {q->shape[1] * h * d, d, h * d},
        .query_offset = c->query_offset, .num_buckets = c->num_buckets, .max_distance = c->max_distance,
        .bidirectional = c->bidirectional, .causal = c->causal, .scale = c->scale, .queries_at_end = c->queries_at_end};
    *p = plan;
    return true;
}

boat_tensor_t* boat_hip_relative_attention(const boat_hip_relative_attention_config_t* config, const boat_tensor_t* query,
                                           const boat_tensor_t* key, const boat_tensor_t* value, const boat_tensor_t* table,
                                           const boat_tensor_t* lengths, boat_tensor_t** lse) {
    if (lse) *lse = NULL;
    bh_relbias_attention_t plan;
    if (!config || !query || !key || !value || !table || !relative_plan(config, query, key, value, table, lengths, &plan)) return NULL;
    const int64_t rows[] = {plan.batch, plan.heads, plan.sq};
    boat_tensor_t* out = bt_new_like_uninit(query);
    boat_tensor_t* sums = bt_new_uninit(rows, 3, query->device);
    const float* pq = bt_dev_read(query);
    const float* pk = bt_dev_read(key);
    const float* pv = bt_dev_read(value);
    const float* pt = bt_dev_read(table);
    const int32_t* pn = lengths ? (const int32_t*)bt_dev_read(lengths) : NULL;
    float* po = out ? bt_dev_write(out) : NULL;
    float* pl = sums ? bt_dev_write(sums) : NULL;
    if (!pq || !pk || !pv || !pt || (lengths && !pn) || !po || !pl ||
        !boat_hip_ok(bh_relbias_attention_forward(&plan, pq, pk, pv, pt, pn, po, pl), "relative attention")) {
        boat_tensor_free(out);
        boat_tensor_free(sums);
        return NULL;
    }
    if (lse) *lse = sums;
    else boat_tensor_free(sums);
    return out;
}

/* grads: those of query, key, value and table, new tensors */
bool bt_relative_attention_backward(const boat_hip_relative_attention_config_t* config, const boat_tensor_t* query,
                                    const boat_tensor_t* key, const boat_tensor_t* value, const boat_tensor_t* table,
                                    const boat_tensor_t* lengths, const boat_tensor_t* out, const boat_tensor_t* lse,
                                    const boat_tensor_t* dy, boat_tensor_t* grads[4]) {
    bh_relbias_attention_t plan;
    if (!relative_plan(config, query, key, value, table, lengths, &plan)) return false;
    if (!bt_is_f32(dy) || dy->nelements != query->nelements) FUSED_REFUSE("relative attention backward expects a gradient of the output's shape");
    const boat_tensor_t* in[4] = {query, key, value, table};
    const float* pi[4];
    float* pg[4];
    bool ok = true;
    for (int i = 0; i < 4; i++) {
        grads[i] = bt_new_like_uninit(in[i]);
        pi[i] = bt_dev_read(in[i]);
        pg[i] = grads[i] ? bt_dev_write(grads[i]) : NULL;
        ok = ok && pi[i] && pg[i];
    }
    const int32_t* pn = lengths ? (const int32_t*)bt_dev_read(lengths) : NULL;
    const float* po = bt_dev_read(out);
    const float* pl = bt_dev_read(lse);
    const float* pd = bt_dev_read(dy);
    ok = ok && po && pl && pd && (!lengths || pn) &&
         boat_hip_ok(bh_relbias_attention_backward(&plan, pi[0], pi[1], pi[2], pi[3], pn, po, pl, pd, pg[0], pg[1], pg[2], pg[3], 0),
                     "relative attention backward");
    for (int i = 0; i < 4 && !ok; i++) {
        boat_tensor_free(grads[i]);
        grads[i] = NULL;
    }
    return ok;
}

/* ---- distillation ---- */
static bool distillation_shapes(const boat_tensor_t* logits, const boat_tensor_t* teacher, const boat_tensor_t* index, const boat_tensor_t* labels) {
    if (!bt_is_f32(logits) || logits->ndim != 2 || logits->nelements == 0) FUSED_REFUSE("distillation expects float logits of shape [rows, vocab]");
    if (!bt_is_f32(teacher) || teacher->ndim != 2 || teacher->shape[0] != logits->shape[0] || teacher->nelements == 0 ||
        !is_i32(index, teacher->nelements))
        FUSED_REFUSE("distillation expects the teacher's logits (float) and their indices (INT32), both [rows, kept]");
    if (labels && !is_i32(labels, (size_t)logits->shape[0])) FUSED_REFUSE("distillation expects INT32 labels, one per row");
    return true;
}

/* one of the three passes over checked tensors: the loss (with *stats and, instead of them, *dlogits when asked) */
static boat_tensor_t* distillation_loss(const boat_tensor_t* logits, const boat_tensor_t* teacher, const boat_tensor_t* index,
                                        const boat_tensor_t* labels, float temperature, float alpha, boat_tensor_t** stats,
                                        boat_tensor_t** dlogits) {
    if (!logits || !teacher || !index || !distillation_shapes(logits, teacher, index, labels)) return NULL;
    const int64_t rows = logits->shape[0], vocab = logits->shape[1], kept = teacher->shape[1], one = 1, three[] = {rows, 3};
    const float scale = 1.0f / (float)rows;
    boat_tensor_t* loss = bt_new_uninit(&one, 1, logits->device);
    boat_tensor_t* extra = stats ? bt_new_uninit(three, 2, logits->device) : dlogits ? bt_new_like_uninit(logits) : NULL;
    const float* pz = bt_dev_read(logits);
    const float* pt = bt_dev_read(teacher);
    const int32_t* pi = (const int32_t*)bt_dev_read(index);
    const int32_t* py = labels ? (const int32_t*)bt_dev_read(labels) : NULL;
    float* pl = loss ? bt_dev_write(loss) : NULL;
    float* pe = extra ? bt_dev_write(extra) : NULL;
    bool ok = pz && pt && pi && pl && (!labels || py) && (pe || !(stats || dlogits));
    ok = ok && boat_hip_ok(dlogits ? bh_distill_loss_grad(pz, vocab, pt, pi, py, rows, vocab, kept, temperature, alpha, scale, NULL, pl, pe, vocab)
                                   : bh_distill_forward(pz, vocab, pt, pi, py, rows, vocab, kept, temperature, alpha, scale, NULL, pe, pl),
                           "distillation");
    if (!ok) {
        boat_tensor_free(loss);
        boat_tensor_free(extra);
        return NULL;
    }
    if (stats) *stats = extra;
    if (dlogits) *dlogits = extra;
    return loss;
}

boat_tensor_t* boat_hip_distillation_loss(const boat_tensor_t* logits, const boat_tensor_t* teacher, const boat_tensor_t* index,
                                          const boat_tensor_t* labels, float temperature, float alpha, boat_tensor_t** dlogits) {
    if (dlogits) *dlogits = NULL;
    return distillation_loss(logits, teacher, index, labels, temperature, alpha, NULL, dlogits);
}
boat_tensor_t* bt_distillation_forward(const boat_tensor_t* logits, const boat_tensor_t* teacher, const boat_tensor_t* index,
                                       const boat_tensor_t* labels, float temperature, float alpha, boat_tensor_t** stats) {
    return distillation_loss(logits, teacher, index, labels, temperature, alpha, stats, NULL);
}
/* dy: the [1] gradient of the loss, read by the kernel */
boat_tensor_t* bt_distillation_backward(const boat_tensor_t* logits, const boat_tensor_t* teacher, const boat_tensor_t* index,
                                        const boat_tensor_t* labels, float temperature, float alpha, const boat_tensor_t* stats,
                                        const boat_tensor_t* dy) {
    if (!bt_is_f32(dy) || dy->nelements < 1) FUSED_REFUSE("distillation backward expects a gradient of one value");
    const int64_t rows = logits->shape[0], vocab = logits->shape[1];
    boat_tensor_t* dz = bt_new_like_uninit(logits);
    const float* pz = bt_dev_read(logits);
    const float* pt = bt_dev_read(teacher);
    const int32_t* pi = (const int32_t*)bt_dev_read(index);
    const int32_t* py = labels ? (const int32_t*)bt_dev_read(labels) : NULL;
    const float* ps = bt_dev_read(stats);
    const float* pd = bt_dev_read(dy);
    float* pg = dz ? bt_dev_write(dz) : NULL;
    if (!pz || !pt || !pi || (labels && !py) || !ps || !pd || !pg ||
        !boat_hip_ok(bh_distill_backward(pz, vocab, pt, pi, py, rows, vocab, teacher->shape[1], temperature, alpha, 1.0f / (float)rows, ps,
                                         pd, pg, vocab), "distillation backward")) {
        boat_tensor_free(dz);
        return NULL;
    }
    return dz;
}
