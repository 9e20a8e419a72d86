// api_rows.cpp -- C-ABI entry points (include/rmr.h) of the feature cache and the linear layer.
#include <utility>

#include "api_handles.h"
#include "rows.h"

using namespace rmr;

namespace {

constexpr int64_t kMaxRows = 0x7fffffff;

// the bytes of `rows` rows, `ld` elements apart; rows that touch or overlap are one long one
struct Range {
    int64_t lo = 0, width = 0, pitch = 0, rows = 0;
    Range(const void* p, int64_t n, int64_t w, int64_t ld, int type) {
        if (!p || n <= 0) return;
        const int64_t size = (int64_t)type_bytes(type);
        lo = (int64_t)(uintptr_t)p, width = w * size, pitch = ld * size, rows = n;
        if (rows > 1 && pitch <= width) width += (rows - 1) * pitch, rows = 1;
    }
    int64_t hi() const { return lo + (rows - 1) * pitch + width; }
    // whether a byte is in both.  Exact at one pitch, as columns of one wider buffer have; rows at two different pitches are taken to
    // meet where their spans do.
    bool meets(const Range& o) const {
        if (!rows || !o.rows) return false;
        if (rows == 1 && o.rows == 1) return lo < o.lo + o.width && o.lo < lo + width;
        const int64_t step = rows > 1 ? pitch : o.pitch;
        if (rows > 1 && o.rows > 1 && pitch != o.pitch) return lo < o.hi() && o.lo < hi();
        // row j of o lies at d + k step from row i of this, k = j - i; the first k that does not end in front of it
        const int64_t d = o.lo - lo, past = -o.width - d;
        int64_t k = past / step - (past % step < 0) + 1;
        if (k < 1 - rows) k = 1 - rows;
        return k < o.rows && d + k * step < width;
    }
};

// no operand spans more than this: its end as an address, and every product on the way there, fits 63 bits
constexpr int64_t kMaxSpan = (int64_t)1 << 56;

// rows of `width` elements: type, element alignment, row pitch
void check_rows(const char* who, const char* what, const void* p, int type, int64_t ld, int64_t rows, int64_t width, bool written) {
    if (!known_type(type)) fail(RMR_ERR_INVALID_ARGUMENT, "%s: unknown type %d of %s", who, type, what);
    if (rows < 0 || rows > kMaxRows) fail(RMR_ERR_INVALID_ARGUMENT, "%s: %lld rows", who, (long long)rows);
    if (rows == 0) return;
    if (!p) fail(RMR_ERR_INVALID_ARGUMENT, "%s: %s is null", who, what);
    if ((uintptr_t)p % type_bytes(type)) fail(RMR_ERR_INVALID_ARGUMENT, "%s: %s is not aligned to its elements", who, what);
    if (rows > 1 && (ld < (written ? width : 0) || ld > (int64_t)1 << 31 || (rows - 1) * ld > kMaxSpan / (int64_t)type_bytes(type)))
        fail(RMR_ERR_INVALID_ARGUMENT, "%s: rows of %s are %lld elements apart, %lld wide", who, what, (long long)ld, (long long)width);
}

void check_slots(const char* who, const int64_t* slots, int64_t n) {
    if (n > 0 && (!slots || (uintptr_t)slots % 8)) fail(RMR_ERR_INVALID_ARGUMENT, "%s: slots is null or not aligned", who);
}

// what is written must leave the slots alone
void check_apart(const char* who, const Range& written, const int64_t* slots, int64_t n) {
    if (written.meets(Range(slots, 1, n * 4, 0, RMR_TYPE_F16))) fail(RMR_ERR_INVALID_ARGUMENT, "%s: the output overlaps slots", who);
}

// a handle that could not be made leaves no error behind for the next launch to report, and the caller's device stays current
template <class F>
rmr_status guarded_create(F&& f) {
    const DeviceKeeper keeper;
    const rmr_status s = guarded(std::forward<F>(f));
    if (s != RMR_OK) (void)hipGetLastError();
    return s;
}

Linear::Call call_of(const char* who, const rmr_linear* layer, const rmr_linear_call* c, bool kept) {
    if (!layer || !c) fail(RMR_ERR_INVALID_ARGUMENT, "%s: null argument", who);
    const rmr_linear_cfg& cfg = layer->impl.cfg();
    Linear::Call k;
    k.rows = c->rows;
    if (!kept) {
        check_rows(who, "x", c->x, c->x_type, c->ldx, c->rows, cfg.in_features, false);
        if ((cfg.format == RMR_LINEAR_F16 && c->x_type != RMR_TYPE_F16) || (cfg.format == RMR_LINEAR_BF16 && c->x_type != RMR_TYPE_BF16))
            fail(RMR_ERR_INVALID_ARGUMENT, "%s: x is not of the layer's type", who);
        k.x = RowSource{c->x, c->x_type, c->rows > 1 ? c->ldx : 0};
    } else if (cfg.format != RMR_LINEAR_MX8) {
        fail(RMR_ERR_INVALID_ARGUMENT, "%s: only a layer of the mx8 format takes kept rows", who);
    }
    check_rows(who, "y", c->y, c->y_type, c->ldy, c->rows, cfg.out_features, true);
    if (c->residual) check_rows(who, "residual", c->residual, c->y_type, c->ldr, c->rows, cfg.out_features, false);
    const Range y(c->y, c->rows, cfg.out_features, c->rows > 1 ? c->ldy : 0, c->y_type);
    if (!kept && y.meets(Range(c->x, c->rows, cfg.in_features, c->rows > 1 ? c->ldx : 0, c->x_type)))
        fail(RMR_ERR_INVALID_ARGUMENT, "%s: y overlaps x", who);
    if (c->residual && !(c->residual == c->y && (c->rows == 1 || c->ldr == c->ldy)) &&
        y.meets(Range(c->residual, c->rows, cfg.out_features, c->rows > 1 ? c->ldr : 0, c->y_type)))
        fail(RMR_ERR_INVALID_ARGUMENT, "%s: y overlaps the residual and is not the residual itself", who);
    const Range ws(c->workspace, c->workspace ? 1 : 0, (int64_t)(c->workspace_bytes / 2), 0, RMR_TYPE_F16);
    if (ws.meets(y) || (!kept && ws.meets(Range(c->x, c->rows, cfg.in_features, c->rows > 1 ? c->ldx : 0, c->x_type))) ||
        (c->residual && ws.meets(Range(c->residual, c->rows, cfg.out_features, c->rows > 1 ? c->ldr : 0, c->y_type))))
        fail(RMR_ERR_INVALID_ARGUMENT, "%s: the workspace overlaps an operand", who);
    k.residual = c->residual, k.ldr = c->ldr, k.y = c->y, k.y_type = c->y_type, k.ldy = c->ldy;
    k.workspace = c->workspace, k.workspace_bytes = c->workspace_bytes;
    return k;
}

}  // namespace

extern "C" {

rmr_status rmr_feature_cache_create(int device, int64_t slots, int width, rmr_feature_cache** out) {
    return guarded_create([&] {
        if (!out || slots <= 0 || slots > (int64_t)1 << 40 || width <= 0 || width > RMR_FEATURE_MAX_WIDTH)
            fail(RMR_ERR_INVALID_ARGUMENT, "rmr_feature_cache_create: %lld slots of width %d", (long long)slots, width);
        *out = new rmr_feature_cache(device, slots, width);
    });
}

void rmr_feature_cache_destroy(rmr_feature_cache* cache) { delete cache; }
size_t rmr_feature_cache_bytes(const rmr_feature_cache* cache) { return cache ? cache->impl.bytes() : 0; }

rmr_status rmr_feature_cache_write(rmr_feature_cache* cache, const void* x, int type, int64_t ld, const int64_t* slots, int64_t n,
                                   void* stream) {
    return guarded([&] {
        if (!cache) fail(RMR_ERR_INVALID_ARGUMENT, "rmr_feature_cache_write: null cache");
        check_rows("rmr_feature_cache_write", "x", x, type, ld, n, cache->impl.width(), false);
        check_slots("rmr_feature_cache_write", slots, n);
        cache->impl.write(RowSource{x, type, n > 1 ? ld : 0}, slots, n, (hipStream_t)stream);
    });
}

rmr_status rmr_feature_cache_read(rmr_feature_cache* cache, const int64_t* slots, int64_t n, void* out, int type, int64_t ld,
                                  void* stream) {
    return guarded([&] {
        if (!cache) fail(RMR_ERR_INVALID_ARGUMENT, "rmr_feature_cache_read: null cache");
        check_rows("rmr_feature_cache_read", "out", out, type, ld, n, cache->impl.width(), true);
        check_slots("rmr_feature_cache_read", slots, n);
        check_apart("rmr_feature_cache_read", Range(out, n, cache->impl.width(), n > 1 ? ld : 0, type), slots, n);
        cache->impl.read(slots, n, out, type, n > 1 ? ld : 0, (hipStream_t)stream);
    });
}

rmr_status rmr_detector_keep_feature(rmr_detector* det, const char* name, int img, rmr_feature_cache* cache, int64_t first_slot) {
    return guarded([&] {
        if (!det || !name || !cache) fail(RMR_ERR_INVALID_ARGUMENT, "rmr_detector_keep_feature: null argument");
        det->impl.keep_feature(name, img, cache->impl, first_slot);
    });
}

rmr_status rmr_linear_create(const rmr_linear_cfg* cfg, const void* weight, int weight_type, int64_t ldw, const float* bias, int mem,
                             void* stream, rmr_linear** out) {
    return guarded_create([&] {
        const char* who = "rmr_linear_create";
        if (!cfg || !out) fail(RMR_ERR_INVALID_ARGUMENT, "%s: null argument", who);
        if (cfg->in_features <= 0 || cfg->in_features > RMR_FEATURE_MAX_WIDTH || cfg->out_features <= 0 || cfg->out_features > 1 << 24)
            fail(RMR_ERR_INVALID_ARGUMENT, "%s: %d -> %d features", who, cfg->in_features, cfg->out_features);
        if (cfg->format < RMR_LINEAR_F16 || cfg->format > RMR_LINEAR_MX8) fail(RMR_ERR_INVALID_ARGUMENT, "%s: unknown format %d", who, cfg->format);
        if (cfg->activation < RMR_ACT_NONE || cfg->activation > RMR_ACT_SIGMOID)
            fail(RMR_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", who, cfg->activation);
        if (mem != RMR_MEM_HOST && mem != RMR_MEM_DEVICE) fail(RMR_ERR_INVALID_ARGUMENT, "%s: unknown memory %d", who, mem);
        check_rows(who, "weight", weight, weight_type, ldw, cfg->out_features, cfg->in_features, true);
        if ((uintptr_t)bias % 4) fail(RMR_ERR_INVALID_ARGUMENT, "%s: bias is not aligned to its elements", who);
        *out = new rmr_linear(*cfg, weight, weight_type, cfg->out_features > 1 ? ldw : cfg->in_features, bias, mem, (hipStream_t)stream);
    });
}

void rmr_linear_destroy(rmr_linear* layer) { delete layer; }

rmr_status rmr_linear_workspace(const rmr_linear* layer, const rmr_linear_call* call, int kept, size_t* bytes) {
    return guarded([&] {
        if (!bytes || !call) fail(RMR_ERR_INVALID_ARGUMENT, "rmr_linear_workspace: null argument");
        rmr_linear_call asked = *call;   // whose workspace is still to be found
        asked.workspace = nullptr, asked.workspace_bytes = 0;
        Linear::Call c = call_of("rmr_linear_workspace", layer, &asked, kept != 0);
        c.kept = kept != 0;
        *bytes = layer->impl.workspace_bytes(c);
    });
}

rmr_status rmr_linear_run(rmr_linear* layer, const rmr_linear_call* call, void* stream) {
    return guarded([&] {
        Linear::Call c = call_of("rmr_linear_run", layer, call, false);
        c.stream = (hipStream_t)stream;
        layer->impl.run(c);
    });
}

rmr_status rmr_linear_run_kept(rmr_linear* layer, rmr_feature_cache* cache, const int64_t* slots, const rmr_linear_call* call, void* stream) {
    return guarded([&] {
        const char* who = "rmr_linear_run_kept";
        if (!cache) fail(RMR_ERR_INVALID_ARGUMENT, "%s: null cache", who);
        Linear::Call c = call_of(who, layer, call, true);
        check_slots(who, slots, c.rows);
        check_apart(who, Range(c.y, c.rows, layer->impl.out_features(), c.rows > 1 ? c.ldy : 0, c.y_type), slots, c.rows);
        check_apart(who, Range(c.workspace, c.workspace ? 1 : 0, (int64_t)(c.workspace_bytes / 2), 0, RMR_TYPE_F16), slots, c.rows);
        const rmr_linear_cfg& cfg = layer->impl.cfg();
        if (cache->impl.width() != cfg.in_features)
            fail(RMR_ERR_INVALID_ARGUMENT, "%s: the cache's rows have %d values, the layer takes %d", who, cache->impl.width(), cfg.in_features);
        if (cache->impl.device() != cfg.device) fail(RMR_ERR_INVALID_ARGUMENT, "%s: cache and layer are on different devices", who);
        c.cache = &cache->impl, c.slots = slots, c.kept = true;
        c.stream = (hipStream_t)stream;
        layer->impl.run(c);
    });
}

}  // extern "C"
