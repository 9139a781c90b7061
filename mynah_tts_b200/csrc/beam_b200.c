/* Beam decoding: lane attention over a shared prefix, beam selection and beam reordering
 * (include/mynah_b200.h).  The entries check what the host can see -- sizes, strides,
 * alignment, workspace -- and enqueue; what lies on the device is checked by the kernels. */
#include "host_common.h"
#include "../../include/mynah_b200.h"

#include <string.h>

/* The backend's device for the length of one call. */
typedef struct { int saved, changed; } device_scope;

static int enter_device(const mb_state *st, device_scope *scope, char *error, size_t cap) {
    scope->changed = 0;
    MB_TRY(cudaGetDevice(&scope->saved), "cudaGetDevice");
    if (scope->saved != st->device) {
        MB_TRY(cudaSetDevice(st->device), "cudaSetDevice");
        scope->changed = 1;
    }
    return 0;
}
static void leave_device(const device_scope *scope) {
    if (scope->changed) (void)cudaSetDevice(scope->saved);
}

static int refuse(const char *message, char *error, size_t cap) {
    mb_set_error(error, cap, message);
    return -1;
}

/* What the kernels count in 32 bits: rows of all lanes, and two blocks of them for each of 64 heads. */
#define MB_LANE_ROWS_MAX ((size_t)1 << 30)

static int aligned4(const void *p) { return ((uintptr_t)p & 3u) == 0; }
/* Arrays of 32-bit values; NULL, for one left out, is aligned. */
static int all_aligned4(const void *const *arrays, size_t n) {
    for (size_t i = 0; i < n; ++i)
        if (!aligned4(arrays[i])) return 0;
    return 1;
}
static int aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

/* 0 when rows of `width` elements can be walked in 16-byte pieces. */
static int check_cache(const mynah_b200_lane_cache *c, int layers, char *error, size_t cap) {
    if (c->type != MYNAH_B200_F32 && c->type != MYNAH_B200_F16)
        return refuse("lane cache type must be f32 or f16", error, cap);
    const size_t per = c->type == MYNAH_B200_F16 ? 8u : 4u;
    if (c->dev_k == NULL || c->dev_v == NULL || c->slots == 0 || c->capacity == 0 || c->width == 0)
        return refuse("lane cache is empty", error, cap);
    if (c->slots > 0xffffffffu || c->capacity > 0x7fffffffu || c->row_stride > 0x1fffffffu)
        return refuse("lane cache is too large", error, cap);
    if (c->row_stride < c->width || c->width % per != 0 || c->row_stride % per != 0 || c->slot_stride % per != 0 ||
        !aligned16(c->dev_k) || !aligned16(c->dev_v))
        return refuse("lane cache rows must be 16-byte aligned and row_stride at least width", error, cap);
    if (c->slots > 1 && c->slot_stride == 0) return refuse("lane cache slot_stride is zero", error, cap);
    if (layers && (c->layers == 0 || c->layers > 32767u || c->layer_stride % per != 0 ||
                   (c->layers > 1 && c->layer_stride == 0)))
        return refuse("lane cache layers or layer_stride out of range", error, cap);
    return 0;
}

static mb_lane_cache cache_of(const mynah_b200_lane_cache *c) {
    const mb_lane_cache m = {c->type, c->dev_k, c->dev_v, c->slots, c->capacity, c->width, c->row_stride,
                             c->slot_stride, c->layers, c->layer_stride};
    return m;
}

/* ------------------------------------------------------------------- attention */
static int attention_sizes_ok(size_t lanes, size_t heads, size_t head_width) {
    return lanes >= 1 && lanes <= MB_LANES_MAX && heads >= 1 && heads <= MB_LANE_HEADS_MAX && head_width >= 4 &&
           head_width <= MB_LANE_HEAD_WIDTH_MAX && head_width % 4u == 0;
}

size_t mynah_b200_lane_attention_workspace(const void *state, size_t lanes, size_t heads, size_t head_width,
                                           size_t prefixes, size_t prefix_capacity) {
    const mb_state *st = (const mb_state *)state;
    if (st == NULL || !attention_sizes_ok(lanes, heads, head_width) || prefixes > MB_LANES_MAX ||
        prefix_capacity > MB_LANE_ROWS_MAX / lanes)
        return 0;
    return mb_lane_attention_floats(lanes, heads, head_width, prefixes, st->sm_count);
}

int mynah_b200_lane_attention(void *state, const mynah_b200_lane_attention_args *a, char *error, size_t cap) {
    mb_state *st = (mb_state *)state;
    if (st == NULL || a == NULL) return refuse("invalid lane attention request", error, cap);
    if (!attention_sizes_ok(a->lanes, a->heads, a->head_width))
        return refuse("lane attention takes 1..1024 lanes, 1..64 heads and a head_width up to 128 in multiples of 4", error, cap);
    if (check_cache(&a->cache, 0, error, cap) != 0) return -1;
    const size_t width = a->heads * a->head_width, per = a->cache.type == MYNAH_B200_F16 ? 8u : 4u;
    if (a->cache.width != width || a->head_width % per != 0)
        return refuse("cache width must be heads * head_width, head_width a multiple of 16 bytes", error, cap);
    if (a->dev_qkv == NULL || a->qkv_stride < 3u * width || a->dev_length == NULL || a->dev_out == NULL ||
        a->out_stride < width || !aligned4(a->dev_qkv) || !aligned4(a->dev_out))
        return refuse("invalid lane attention buffers", error, cap);
    const void *words[] = {a->dev_slot, a->dev_length, a->dev_live};
    if (!all_aligned4(words, sizeof(words) / sizeof(words[0])))
        return refuse("lane attention arrays must be 4-byte aligned", error, cap);
    if (a->dev_slot == NULL && a->cache.slots < a->lanes)
        return refuse("fewer slots than lanes", error, cap);
    size_t prefix_capacity = 0;
    if (a->prefixes > 0) {
        prefix_capacity = a->prefix_capacity;
        if (a->prefixes > MB_LANES_MAX || a->dev_prefix_k == NULL || a->dev_prefix_v == NULL || a->dev_prefix_length == NULL ||
            prefix_capacity == 0 || prefix_capacity > 0x7fffffffu || a->prefix_row_stride > 0x1fffffffu)
            return refuse("invalid lane attention prefixes", error, cap);
        const void *of_prefixes[] = {a->dev_prefix_length, a->dev_lane_prefix};
        if (!all_aligned4(of_prefixes, sizeof(of_prefixes) / sizeof(of_prefixes[0])))
            return refuse("lane attention arrays must be 4-byte aligned", error, cap);
        if (a->prefix_row_stride < width || a->prefix_row_stride % per != 0 || a->prefix_stride % per != 0 ||
            (a->prefixes > 1 && a->prefix_stride == 0) || !aligned16(a->dev_prefix_k) || !aligned16(a->dev_prefix_v))
            return refuse("prefix rows must be 16-byte aligned and prefix_row_stride at least the width", error, cap);
    }
    if (a->lanes * (a->cache.capacity + prefix_capacity) > MB_LANE_ROWS_MAX)
        return refuse("lanes * (capacity + prefix_capacity) must be at most 2^30", error, cap);
    if (a->window > 0 && (a->window > a->cache.capacity || a->sinks > a->cache.capacity - a->window))
        return refuse("a windowed cache must hold window + sinks rows", error, cap);
    if (a->dev_workspace == NULL || !aligned16(a->dev_workspace) ||
        a->workspace_floats < mb_lane_attention_floats(a->lanes, a->heads, a->head_width, a->prefixes, st->sm_count))
        return refuse("lane attention workspace is too small or not 16-byte aligned", error, cap);
    unsigned launched = 0;
    mb_lane_attn_args m;
    memset(&m, 0, sizeof(m));
    m.lanes = a->lanes;
    m.heads = a->heads;
    m.head_width = a->head_width;
    m.scale = a->scale;
    m.qkv = a->dev_qkv;
    m.qkv_stride = a->qkv_stride;
    m.cache = cache_of(&a->cache);
    m.slot = a->dev_slot;
    m.length = a->dev_length;
    m.prefixes = a->prefixes;
    if (a->prefixes > 0) {
        m.prefix_k = a->dev_prefix_k;
        m.prefix_v = a->dev_prefix_v;
        m.prefix_capacity = prefix_capacity;
        m.prefix_row_stride = a->prefix_row_stride;
        m.prefix_stride = a->prefix_stride;
        m.prefix_length = a->dev_prefix_length;
        m.lane_prefix = a->dev_lane_prefix;
    }
    m.window = a->window;
    m.sinks = a->window > 0 ? a->sinks : 0;
    m.live = a->dev_live;
    m.out = a->dev_out;
    m.out_stride = a->out_stride;
    m.workspace = a->dev_workspace;
    m.status = st->d_status + 1;           /* read by the next sync only: a full lane is no fault of what else runs */
    m.sm_count = st->sm_count;
    m.tiles = st->lane_tiles;
    m.polls = st->lane_polls;
    m.device = &st->lane_device;
    m.launched = &launched;
    device_scope scope;
    if (enter_device(st, &scope, error, cap) != 0) return -1;
    const int rc = mb_cuda(mb_lane_attention(&m, st->stream), "lane attention", error, cap);
    leave_device(&scope);
    if (rc != 0) return -1;
    st->launches += launched;
    mb_clear_error(error, cap);
    return 0;
}

/* ------------------------------------------------------------------- selection */
int mynah_b200_beam_select(void *state, const mynah_b200_beam_select_args *a, char *error, size_t cap) {
    mb_state *st = (mb_state *)state;
    if (st == NULL || a == NULL) return refuse("invalid beam selection request", error, cap);
    if (a->requests == 0 || a->requests > (size_t)1 << 24 || a->beams == 0 || a->beams > MB_BEAM_MAX)
        return refuse("beam selection takes 1..16 beams and 1..2^24 requests", error, cap);
    if (a->vocab == 0 || a->vocab >= (size_t)1 << 30 || a->codebook_size > a->vocab || a->logits_stride < a->vocab)
        return refuse("beam selection vocabulary out of range", error, cap);
    if (a->dev_logits == NULL || a->dev_score == NULL || a->dev_score_out == NULL || a->dev_token == NULL ||
        a->dev_parent == NULL || a->dev_token == a->dev_parent || ((uintptr_t)a->dev_logits & 3u) != 0)
        return refuse("invalid beam selection buffers", error, cap);
    const void *words[] = {a->dev_allow_eos, a->dev_score,  a->dev_done,   a->dev_live,
                           a->dev_score_out, a->dev_token, a->dev_parent, a->dev_done_out};
    if (!all_aligned4(words, sizeof(words) / sizeof(words[0])))
        return refuse("beam selection arrays must be 4-byte aligned", error, cap);
    mb_beam_select_args m;
    memset(&m, 0, sizeof(m));
    m.logits = a->dev_logits;
    m.requests = a->requests;
    m.beams = a->beams;
    m.codebook_size = a->codebook_size;
    m.eos_id = a->eos_id < 0xffffffffu ? a->eos_id : 0xfffffffeu;
    m.logits_stride = a->logits_stride;
    m.has_eos = a->eos_id < a->vocab && a->eos_id >= a->codebook_size;
    m.allow_eos = a->dev_allow_eos;
    m.score = a->dev_score;
    m.done = a->dev_done;
    m.live = a->dev_live;
    m.score_out = a->dev_score_out;
    m.token = a->dev_token;
    m.parent = a->dev_parent;
    m.done_out = a->dev_done_out;
    m.clusters = st->beam_clusters;
    device_scope scope;
    if (enter_device(st, &scope, error, cap) != 0) return -1;
    const int rc = mb_cuda(mb_beam_select(&m, st->stream), "beam selection", error, cap);
    leave_device(&scope);
    if (rc != 0) return -1;
    st->launches += 1;
    mb_clear_error(error, cap);
    return 0;
}

/* ------------------------------------------------------------------ reordering */
int mynah_b200_beam_reorder(void *state, const mynah_b200_beam_reorder_args *a, char *error, size_t cap) {
    mb_state *st = (mb_state *)state;
    if (st == NULL || a == NULL) return refuse("invalid beam reorder request", error, cap);
    if (a->requests == 0 || a->requests > 65535u || a->beams == 0 || a->beams > MB_BEAM_MAX)
        return refuse("beam reorder takes 1..16 beams and 1..65535 requests", error, cap);
    if (check_cache(&a->cache, 1, error, cap) != 0) return -1;
    if (a->dev_parent == NULL || a->dev_length == NULL || a->dev_length_out == a->dev_length)
        return refuse("invalid beam reorder buffers", error, cap);
    const void *words[] = {a->dev_slot, a->dev_parent, a->dev_length, a->dev_length_out, a->dev_live};
    if (!all_aligned4(words, sizeof(words) / sizeof(words[0])))
        return refuse("beam reorder arrays must be 4-byte aligned", error, cap);
    if (a->dev_slot == NULL && a->cache.slots < a->requests * a->beams)
        return refuse("fewer slots than lanes", error, cap);
    mb_beam_reorder_args m;
    memset(&m, 0, sizeof(m));
    m.cache = cache_of(&a->cache);
    m.requests = a->requests;
    m.beams = a->beams;
    m.slot = a->dev_slot;
    m.parent = a->dev_parent;
    m.length = a->dev_length;
    m.length_out = a->dev_length_out;
    m.live = a->dev_live;
    m.sm_count = st->sm_count;
    device_scope scope;
    if (enter_device(st, &scope, error, cap) != 0) return -1;
    const int rc = mb_cuda(mb_beam_reorder(&m, st->stream), "beam reorder", error, cap);
    leave_device(&scope);
    if (rc != 0) return -1;
    st->launches += 1;
    mb_clear_error(error, cap);
    return 0;
}
