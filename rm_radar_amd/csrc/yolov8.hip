// yolov8.hip -- weight-pack loader, graph planner and executor for the YOLOv8 detector network
// (public Ultralytics architecture; replaces the TensorRT engine the
// reference builds in src/detect/detector.cpp:177-243 and runs at src/detect/detector.h:122).
//
// Layout decisions (MI355X-first):
//  * activations f16 NHWC in one arena; every C2f / SPPF / FPN concat is a wider buffer whose
//    channel slices are written in place by the producing conv (no concat kernels, no copies
//    except the two nearest-2x upsamples);
//  * the Detect head's two first 3x3 convs of a scale share their input, so they run as ONE
//    implicit GEMM with N = 64 + c3 output channels;
//  * large batches are walked in chunks so one layer's in+out activations stay within the
//    256 MiB Infinity Cache instead of streaming the whole batch through HBM per layer.
#include "yolov8.h"

#include <cmath>
#include <algorithm>
#include <cstdlib>
#include <fstream>
#include <unistd.h>

#include "net_ops.h"

namespace rmr {

constexpr size_t kSplitKWsFloats = 16u << 20;  // 64 MiB of split-K partial tiles
constexpr size_t kMaxViewBytes = 0xf0000000ull;  // largest activation view a buffer resource of the conv kernels addresses
constexpr int kSplitKMaxTiles = 8192;

// ---- weight pack ---------------------------------------------------------------------------------

WeightPack WeightPack::load(const std::string& path) {
    std::ifstream f(path, std::ios::binary);
    if (!f) fail(RMR_ERR_INVALID_ARGUMENT, "weight pack '%s' does not exist or cannot be opened", path.c_str());
    f.seekg(0, std::ios::end);
    const size_t file_bytes = (size_t)f.tellg();
    f.seekg(0, std::ios::beg);
    auto rd = [&](void* p, size_t n) {
        f.read((char*)p, (std::streamsize)n);
        if (!f) fail(RMR_ERR_RUNTIME, "weight pack '%s' is truncated", path.c_str());
    };
    char magic[4];
    rd(magic, 4);
    if (std::memcmp(magic, "RMRW", 4) != 0) fail(RMR_ERR_RUNTIME, "'%s' is not an RMRW weight pack", path.c_str());
    unsigned version, n;
    WeightPack p;
    rd(&version, 4);
    if (version != 1) fail(RMR_ERR_RUNTIME, "'%s': unsupported pack version %u", path.c_str(), version);
    rd(&p.depth, 4);
    rd(&p.width, 4);
    rd(&p.max_ch, 4);
    rd(&p.nc, 4);
    rd(&p.reg_max, 4);
    rd(&n, 4);
    for (unsigned i = 0; i < n; ++i) {
        unsigned ln, nd;
        rd(&ln, 4);
        if (ln > 4096) fail(RMR_ERR_RUNTIME, "'%s': corrupt tensor name", path.c_str());
        std::string name(ln, '\0');
        rd(&name[0], ln);
        rd(&nd, 4);
        if (nd > 8) fail(RMR_ERR_RUNTIME, "'%s': corrupt tensor rank", path.c_str());
        Tensor t;
        t.dims.resize(nd);
        rd(t.dims.data(), 4 * nd);
        size_t cnt = 1;
        for (unsigned d : t.dims) {
            // a tensor cannot hold more floats than the file has bytes left: rejects corrupt dims before the
            // product can wrap around size_t
            if (d == 0 || cnt > file_bytes / 4 / d) fail(RMR_ERR_RUNTIME, "'%s': tensor '%s' is larger than the file", path.c_str(), name.c_str());
            cnt *= d;
        }
        t.data.resize(cnt);
        rd(t.data.data(), cnt * 4);
        p.tensors.emplace(std::move(name), std::move(t));
    }
    return p;
}

const WeightPack::Tensor& WeightPack::get(const std::string& name) const {
    auto it = tensors.find(name);
    if (it == tensors.end()) fail(RMR_ERR_RUNTIME, "weight pack has no tensor '%s'", name.c_str());
    return it->second;
}

// ---- planner ----------------------------------------------------------------------------------------

View Yolov8::alloc(int h, int w, int c, bool f32) {
    View v;
    v.cs = c;
    v.co = 0;
    v.c = c;
    v.h = h;
    v.w = w;
    size_t& top = f32 ? arena_floats_ : arena_halves_;
    v.off = top;
    top += (size_t)h * w * c;
    top = (top + 63) & ~(size_t)63;
    allocs_.push_back(Alloc{v.off, top - v.off, f32 ? 1 : 0, alloc_group_});
    return v;
}

View Yolov8::slice(const View& v, int co, int c) {
    View s = v;
    s.co = v.co + co;
    s.c = c;
    return s;
}

int Yolov8::add_conv_weights(const WeightPack& p, const std::string& name, int cin_pad, int ci0, int ci_n, bool no_bias) {
    const auto& w = p.get(name + ".weight");
    const auto& b = p.get(name + ".bias");
    if (w.dims.size() != 4 || w.dims[2] != w.dims[3]) fail(RMR_ERR_RUNTIME, "tensor '%s.weight' is not OIkk", name.c_str());
    const int cin_all = (int)w.dims[1];
    if (w.data.size() != (size_t)w.dims[0] * w.dims[1] * w.dims[2] * w.dims[3])
        fail(RMR_ERR_RUNTIME, "tensor '%s.weight' does not hold its %u x %u x %u x %u values", name.c_str(), w.dims[0], w.dims[1], w.dims[2], w.dims[3]);
    if (ci_n == 0) ci0 = 0, ci_n = cin_all;
    if (ci0 < 0 || ci0 + ci_n > cin_all) fail(RMR_ERR_LOGIC, "conv '%s': channel slice outside the tensor", name.c_str());
    ConvW cw;
    cw.cout = (int)w.dims[0];
    cw.cin = cin_pad > 0 ? cin_pad : ci_n;
    cw.k = (int)w.dims[2];
    cw.cout_pad = (cw.cout + 15) / 16 * 16;
    if (ci_n > cw.cin || cw.cin % 8)
        fail(RMR_ERR_RUNTIME, "conv '%s': %d input channels cannot be consumed in 8-channel chunks", name.c_str(), ci_n);
    if (b.data.size() != (size_t)cw.cout) fail(RMR_ERR_RUNTIME, "tensor '%s.bias' has the wrong size", name.c_str());
    const size_t kk = (size_t)cw.k * cw.k;
    std::vector<float> sub;  // [cout][ci_n][k][k]
    const float* wsrc = w.data.data();
    if (ci_n != cin_all) {
        sub.resize((size_t)cw.cout * ci_n * kk);
        for (int o = 0; o < cw.cout; ++o)
            std::copy(wsrc + ((size_t)o * cin_all + ci0) * kk, wsrc + ((size_t)o * cin_all + ci0 + ci_n) * kk,
                      sub.begin() + (size_t)o * ci_n * kk);
        wsrc = sub.data();
    }
    std::vector<__half> packed;
    pack_conv_weights(wsrc, cw.cout, ci_n, cw.k, cw.k, cw.cin, cw.cout_pad, packed, cw.K, cw.Kp);
    std::vector<float> bias(cw.cout_pad, 0.f);
    if (!no_bias) std::copy(b.data.begin(), b.data.end(), bias.begin());
    cw.w.alloc(packed.size());
    cw.b.alloc(bias.size());
    RMR_HIP(hipMemcpy(cw.w.p, packed.data(), packed.size() * sizeof(__half), hipMemcpyHostToDevice));
    RMR_HIP(hipMemcpy(cw.b.p, bias.data(), bias.size() * sizeof(float), hipMemcpyHostToDevice));
    upload_t32(cw, packed);
    convs_.push_back(std::move(cw));
    return (int)convs_.size() - 1;
}

// the second copy of a 3x3 or 1x1 layer's weights, as the LDS images conv_t32 / conv_g32 stream
void Yolov8::upload_t32(ConvW& cw, const std::vector<__half>& packed) {
    if (fp8_ && fp8_layer_ && cw.k == 3 && cw.cin % 16 == 0 && cw.cin >= 64) {
        std::vector<unsigned char> p8;
        std::vector<float> ws;
        pack_conv_weights_t32f8(packed.data(), cw.cout_pad, cw.cin, cw.Kp, p8, ws);
        cw.w8.alloc(p8.size());
        cw.wscale.alloc(ws.size());
        RMR_HIP(hipMemcpy(cw.w8.p, p8.data(), p8.size(), hipMemcpyHostToDevice));
        RMR_HIP(hipMemcpy(cw.wscale.p, ws.data(), ws.size() * sizeof(float), hipMemcpyHostToDevice));
    }
    if ((cw.k != 3 && cw.k != 1) || cw.cin % 32) return;
    std::vector<__half> p32;
    pack_conv_weights_t32(packed.data(), cw.cout_pad, cw.cin, cw.Kp, p32, cw.k * cw.k);
    cw.w32.alloc(p32.size());
    RMR_HIP(hipMemcpy(cw.w32.p, p32.data(), p32.size() * sizeof(__half), hipMemcpyHostToDevice));
    // the Winograd F(2, 3) form of a 3x3 layer (conv_w1d): a measured experiment, slower than conv_t32 on every layer
    // (conv_w1d.hip), so only offered to the tuner with RMR_WINOGRAD=1
    const bool wino = conv_w1d_num_tiles() > 0 && std::getenv("RMR_WINOGRAD") && std::atoi(std::getenv("RMR_WINOGRAD")) != 0;   // read per detector; EXPERIMENTS=1 builds only
    if (wino && cw.k == 3) {
        std::vector<__half> pw;
        pack_conv_weights_w1d(packed.data(), cw.cout_pad, cw.cin, cw.Kp, pw);
        cw.w1d.alloc(pw.size());
        RMR_HIP(hipMemcpy(cw.w1d.p, pw.data(), pw.size() * sizeof(__half), hipMemcpyHostToDevice));
    }
}

// two convs over the same input, concatenated along Cout (Detect cv2.i.0 + cv3.i.0)
int Yolov8::add_fused_head_weights(const WeightPack& p, const std::string& a, const std::string& b) {
    const auto& wa = p.get(a + ".weight");
    const auto& wb = p.get(b + ".weight");
    const auto& ba = p.get(a + ".bias");
    const auto& bb = p.get(b + ".bias");
    if (wa.dims.size() != 4 || wb.dims.size() != 4 || wa.dims[1] != wb.dims[1] || wa.dims[2] != wb.dims[2])
        fail(RMR_ERR_RUNTIME, "cannot fuse '%s' and '%s'", a.c_str(), b.c_str());
    ConvW cw;
    cw.cout = (int)(wa.dims[0] + wb.dims[0]);
    cw.cin = (int)wa.dims[1];
    cw.k = (int)wa.dims[2];
    cw.cout_pad = (cw.cout + 15) / 16 * 16;
    if (cw.cin % 8 || wa.dims[0] % 16) fail(RMR_ERR_RUNTIME, "head conv '%s' has unsupported channel counts", a.c_str());
    std::vector<float> w(wa.data);
    w.insert(w.end(), wb.data.begin(), wb.data.end());
    std::vector<__half> packed;
    pack_conv_weights(w.data(), cw.cout, cw.cin, cw.k, cw.k, cw.cin, cw.cout_pad, packed, cw.K, cw.Kp);
    std::vector<float> bias(cw.cout_pad, 0.f);
    std::copy(ba.data.begin(), ba.data.end(), bias.begin());
    std::copy(bb.data.begin(), bb.data.end(), bias.begin() + ba.data.size());
    cw.w.alloc(packed.size());
    cw.b.alloc(bias.size());
    RMR_HIP(hipMemcpy(cw.w.p, packed.data(), packed.size() * sizeof(__half), hipMemcpyHostToDevice));
    RMR_HIP(hipMemcpy(cw.b.p, bias.data(), bias.size() * sizeof(float), hipMemcpyHostToDevice));
    upload_t32(cw, packed);
    convs_.push_back(std::move(cw));
    return (int)convs_.size() - 1;
}

void Yolov8::conv(int widx, const View& in, const View& out, int stride, int act, const View* res,
                  bool out_f32, bool in_is_input, const View* pre) {
    const ConvW& cw = convs_[widx];
    if (in.c != cw.cin)
        fail(RMR_ERR_RUNTIME, "weight pack does not fit the network plan: conv %d consumes %d input channels, the plan feeds it %d (header scale vs tensors?)", widx, cw.cin, in.c);
    if (out.c != cw.cout_pad && !(out_f32 && out.cs == cw.cout_pad))
        if (out.c != cw.cout)
            fail(RMR_ERR_RUNTIME, "weight pack does not fit the network plan: conv %d produces %d channels, the plan expects %d (header scale vs tensors?)", widx, cw.cout, out.c);
    Op op{};
    op.kind = OP_CONV;
    op.conv = widx;
    op.in = in;
    op.out = out;
    // fp8 plan: a 3x3 / stride-1 layer with e4m3 weights reads an e4m3 copy of its input, written just before it
    // (the layers between keep f16 activations: the copy is one extra pass over a tensor the conv reads nine times)
    // ... and only where an e4m3 tile exists for the layer's width on maps this wide (tile channel counts are 64 / 96 / 192 /
    // 256 and the halo rows must fit a tile's LDS slots): a 80- or 160-channel layer of a wider pack, or a 96-channel layer
    // on 240-wide maps, stays f16 -- no e4m3 weights, no quantiser pass -- instead of failing at its first forward
    const bool f8_layer = cw.w8.p && stride == 1 && !in_is_input && !pre && in.h == out.h && in.w == out.w;
    if (f8_layer && conv_t32f8_first_tile(cw.cout_pad, in.w) < 0) {
        convs_[widx].w8.release();
        convs_[widx].wscale.release();
    }
    if (cw.w8.p && f8_layer) {
        Op q{};
        q.kind = OP_QUANT;
        q.in = in;
        q.q_pitch = (cw.cin + 63) / 64 * 64;
        q.q_off = arena_bytes8_;
        arena_bytes8_ += (size_t)in.h * in.w * q.q_pitch;
        arena_bytes8_ = (arena_bytes8_ + 255) & ~(size_t)255;
        allocs_.push_back(Alloc{q.q_off, arena_bytes8_ - q.q_off, 2, 0});
        // The e4m3 copy is written by a quantiser pass (read 2 B, write 1 B per value at ~3.9 TB/s: 2.1 ms of a
        // 256-image forward, 36 launches) -- unless the tensor comes out of an e4m3 layer: then that layer's epilogue writes
        // it (conv_t32_common.h, OUT8), and where this layer is the tensor's ONLY reader (the hidden tensor of a
        // bottleneck) the f16 copy is not written at all (q_only, decided once the plan is complete).  Round 2 had
        // measured the fused form a wash: it ran through the old epilogue, bias loads between the stores.  RMR_FP8_FUSE=0
        // restores the passes.
        const bool fuse = !(std::getenv("RMR_FP8_FUSE") && atoi(std::getenv("RMR_FP8_FUSE")) == 0);   // read per detector
        Op* producer = nullptr;
        for (auto it = ops_.rbegin(); it != ops_.rend() && fuse; ++it)
            if (it->kind == OP_CONV && it->out.off == in.off && it->out.co == in.co && it->out.c == in.c && it->out.cs == in.cs) {
                if (it->fp8 && !it->q_out && !it->out_f32 && ((it->out.cs | it->out.co) & 7) == 0) producer = &*it;
                break;
            }
        if (producer) {
            producer->q_out = true;
            producer->q_out_off = q.q_off;
            producer->q_out_pitch = q.q_pitch;
        } else {
            ops_.push_back(q);
        }
        op.fp8 = true;
        op.q_off = q.q_off;
        op.q_pitch = q.q_pitch;
    }
    if (res) op.res = *res;
    if (pre) {
        if (pre->h * 2 != out.h || pre->w * 2 != out.w || pre->cs != cw.cout_pad || pre->co != 0 || cw.k != 1)
            fail(RMR_ERR_LOGIC, "planner: conv %d: the half-resolution addend does not fit", widx);
        op.pre = *pre;
    }
    op.stride = stride;
    op.act = act;
    op.out_f32 = out_f32;
    op.in_is_input = in_is_input;
    ops_.push_back(op);
    // algorithmic FLOPs: 2*MAC with the pack's true channel counts
    flops_ += 2.0 * out.h * out.w * (double)cw.cout * (in_is_input ? 3 : cw.cin) * cw.k * cw.k;
}

// C2f (Ultralytics nn/modules/block.py): cv1 -> split -> n bottlenecks chained on the last
// half -> cv2 over the (2+n)*c concat.  The concat buffer IS where everything is written.
View Yolov8::c2f(const WeightPack& p, const std::string& name, const View& x, int n, bool shortcut,
                 const View* out_view, const View* up) {
    const int cout = (int)p.get(name + ".cv2.conv.weight").dims[0];
    const int c = cout / 2;
    if (c % 16) fail(RMR_ERR_RUNTIME, "C2f '%s': hidden width %d is not a multiple of 16", name.c_str(), c);
    // Chunks as planar slabs where both 1x1 convs can run on conv_pw (the only kernel that addresses
    // slabs) and a chunk is narrower than two cache lines: the 3x3 convs in between then stream
    // contiguous rows (2-2.7x read amplification on 96-byte slices of 384-byte pixels)
    const int cu = up ? up->c : 0, cin1 = up ? x.c : x.c;
    const bool slab = slabs_ && (c == 48 || c == 96) && pw_can(cin1, 2 * c, x.h, x.w, up != nullptr) &&
                      pw_can((2 + n) * c, cout, x.h, x.w, false) &&
                      (double)chunk_ * x.h * x.w * c * 2.0 * (2 + n) < 3.9e9;  // 32-bit offsets across the slabs
    std::vector<View> chunk(2 + n);
    View cat{};
    if (slab) {
        alloc_group_ = next_group_++;   // the slabs keep their equal spacing when the arena is compacted
        for (int i = 0; i < 2 + n; ++i) {
            chunk[i] = alloc(x.h, x.w, c);
            if (i && chunk[i].off - chunk[i - 1].off != chunk[1].off - chunk[0].off)
                fail(RMR_ERR_LOGIC, "planner: slabs are not equally spaced");
        }
        alloc_group_ = 0;
    } else {
        cat = alloc(x.h, x.w, (2 + n) * c);
        for (int i = 0; i < 2 + n; ++i) chunk[i] = slice(cat, i * c, c);
    }
    const size_t step = slab ? chunk[1].off - chunk[0].off : 0;
    View cv1_out = slab ? chunk[0] : slice(cat, 0, 2 * c);
    cv1_out.c = 2 * c;
    if (up) {
        // cv1 over concat[up2x(U), S] = SiLU(W_S.S + b + up2x(W_U.U)): the U half at a quarter of the
        // pixels, in f32, added by the S half's epilogue (ConvArgs::pre)
        const int cs = x.c;
        View t = alloc(up->h, up->w, 2 * c, true);
        conv(add_conv_weights(p, name + ".cv1.conv", 0, 0, cu, true), *up, t, 1, 0, nullptr, true);
        conv(add_conv_weights(p, name + ".cv1.conv", 0, cu, cs), x, cv1_out, 1, 1, nullptr, false, false, &t);
        // the model's own count for this layer: 2 * K * N at full resolution (the two launches
        // above declared what they execute, 3/4 of the U half less)
        flops_ += 2.0 * x.h * x.w * (double)(2 * c) * cu * 0.75;
    } else {
        conv(add_conv_weights(p, name + ".cv1.conv", 0), x, cv1_out, 1, 1);
    }
    if (slab) {
        ops_.back().out_slab_c = c;
        ops_.back().out_slab_step = step;
    }
    for (int i = 0; i < n; ++i) {
        View tmp = alloc(x.h, x.w, c);
        const View prev = chunk[1 + i];
        const std::string m = name + ".m." + std::to_string(i);
        conv(add_conv_weights(p, m + ".cv1.conv", 0), prev, tmp, 1, 1);
        conv(add_conv_weights(p, m + ".cv2.conv", 0), tmp, chunk[2 + i], 1, 1, shortcut ? &prev : nullptr);
    }
    View out = out_view ? *out_view : alloc(x.h, x.w, cout);
    View cv2_in = slab ? chunk[0] : cat;
    cv2_in.c = (2 + n) * c;
    conv(add_conv_weights(p, name + ".cv2.conv", 0), cv2_in, out, 1, 1);
    if (slab) {
        ops_.back().in_slab_c = c;
        ops_.back().in_slab_step = step;
    }
    return out;
}

// Runs of consecutive convolutions that do not depend on one another (before the arenas are compacted: a buffer is still its
// own region, two views overlap when they name the same region and their channel ranges meet)
void Yolov8::find_groups() {
    const auto meet = [](const View& x, bool xf, const View& y, bool yf) {
        return (x.c || x.cs) && (y.c || y.cs) && xf == yf && x.off == y.off && x.co < y.co + y.c && y.co < x.co + x.c;
    };
    const auto plain = [&](const Op& o) {
        return o.kind == OP_CONV && !o.fp8 && !o.q_out && !o.in_is_input && o.fuse_with < 0 && !o.in_slab_c && !o.out_slab_c && !o.pre.c;
    };
    const auto independent = [&](const Op& x, const Op& y) {   // x before y
        if (meet(x.out, x.out_f32, y.in, false) || meet(x.out, x.out_f32, y.res, false)) return false;   // y reads what x writes
        if (meet(y.out, y.out_f32, x.in, false) || meet(y.out, y.out_f32, x.res, false)) return false;   // y overwrites what x reads
        return !meet(x.out, x.out_f32, y.out, y.out_f32);
    };
    for (size_t i = 0; i < ops_.size();) {
        if (!plain(ops_[i])) {
            ++i;
            continue;
        }
        size_t j = i + 1;
        for (; j < ops_.size() && j - i < 8 && plain(ops_[j]); ++j) {
            // one launch = one kernel form: 3x3 / stride-1 layers with one another (the halo form), everything else likewise
            bool ok = convs_[ops_[j].conv].k == convs_[ops_[i].conv].k && ops_[j].stride == ops_[i].stride;
            for (size_t k = i; k < j && ok; ++k) ok = independent(ops_[k], ops_[j]);
            // a fusable bottleneck's second convolution never joins (its partner may have taken it along)
            if (!ok || (j > 0 && ops_[j - 1].fuse_with == (int)j)) break;
        }
        if (j - i >= 2) {
            std::vector<int> g;
            for (size_t k = i; k < j; ++k) {
                ops_[k].group = (int)groups_.size();
                g.push_back((int)k);
            }
            groups_.push_back(g);
        }
        i = j;
    }
}

std::vector<ConvArgs> Yolov8::group_args(int g, int n) {
    std::vector<ConvArgs> v;
    for (int op : groups_[g]) v.push_back(conv_args(op, n, 0));
    return v;
}

// the problem table of a grouped launch, in device memory for as long as the detector lives (captured graphs name it)
void Yolov8::ensure_group_table(int g, int n, int variant) {
    const std::vector<ConvArgs> args = group_args(g, n);
    std::vector<unsigned char> host(conv_sb_group_bytes((int)args.size()));
    conv_sb_group_build(args.data(), (int)args.size(), variant, host.data());
    DevBuf<unsigned char>& d = group_tables_[{groups_[g].front(), n}];
    d.alloc(host.size());
    RMR_HIP(hipMemcpy(d.p, host.data(), host.size(), hipMemcpyHostToDevice));
}

// First visit of a group at n images: every member is tuned on its own (and has run), then the grouped launch of every conv_sb
// variant that takes all of them is timed against the sum of the members' launches
void Yolov8::tune_group(hipStream_t s, int g, int n, size_t img0) {
    const std::vector<int>& ops = groups_[g];
    float sum_ms = 0.f;
    for (int op : ops) {
        if (tuned_.count({op, n})) return;   // a partly tuned group (an older cache): leave it as it is
    }
    for (int op : ops) {
        float ms = 0.f;
        tuned_[{op, n}] = tune_conv(s, conv_args(op, n, img0), &ms);
        sum_ms += ms;
    }
    tuned_dirty_ = true;
    // RMR_GROUPS=0: never group (read per call, so a test can change it between detectors of one process)
    if (const char* e = std::getenv("RMR_GROUPS"))
        if (std::atoi(e) == 0) return;
    // RMR_TUNE_ONLY=lo-hi pins a kernel family under the whole network: a grouped conv_sb launch may only replace the members
    // when the range covers the grouped ids (or the conv_sb ids) -- otherwise 700-799 would still hand the head to conv_sb
    if (const char* e = std::getenv("RMR_TUNE_ONLY")) {
        int lo = 0, hi = 0;
        if (sscanf(e, "%d-%d", &lo, &hi) == 2 && !(hi >= kSbGroupBase || (lo <= kSbBase && hi >= kSbBase))) return;
    }
    const std::vector<ConvArgs> args = group_args(g, n);
    hipEvent_t e0, e1;
    RMR_HIP(hipEventCreate(&e0));
    RMR_HIP(hipEventCreate(&e1));
    const int prof_was_on = ctx_.prof.on;
    ctx_.prof.on = 0;
    float best_ms = 1e30f;
    int best_v = -1;
    DevBuf<unsigned char> table;
    std::vector<unsigned char> host(conv_sb_group_bytes((int)args.size()));
    table.alloc(host.size());
    for (int v = 0; v < conv_sb_num_variants(); ++v) {
        if (!conv_sb_group_supported(args.data(), (int)args.size(), v)) continue;
        {   // the gate tune_conv applies to conv_sb: beyond a few workgroups per CU the throughput kernels' streams win, and
            // 66 variants x 3 launches of a large batch are minutes of tuning for a group that cannot win
            const ConvTile ct = conv_sb_tile(v);
            long tiles = 0;
            for (const ConvArgs& a : args) tiles += (long)((a.M + ct.bm - 1) / ct.bm) * ((a.Cout_pad + ct.bn - 1) / ct.bn);
            if (tiles > 6L * ctx_.num_cus) continue;
        }
        conv_sb_group_build(args.data(), (int)args.size(), v, host.data());
        RMR_HIP(hipMemcpy(table.p, host.data(), host.size(), hipMemcpyHostToDevice));
        float v_ms = 1e30f;
        for (int rep = 0; rep < 3; ++rep) {
            RMR_HIP(hipEventRecord(e0, s));
            launch_conv_sb_group(ctx_, s, args.data(), (int)args.size(), table.p, v);
            RMR_HIP(hipEventRecord(e1, s));
            RMR_HIP(hipEventSynchronize(e1));
            float t = 0;
            RMR_HIP(hipEventElapsedTime(&t, e0, e1));
            if (rep > 0) v_ms = std::min(v_ms, t);
        }
        if (std::getenv("RMR_TUNE_VERBOSE")) fprintf(stderr, " g%d:%.1f", v, v_ms * 1e3f);
        if (v_ms < best_ms) best_ms = v_ms, best_v = v;
    }
    ctx_.prof.on = prof_was_on;
    (void)hipEventDestroy(e0);
    (void)hipEventDestroy(e1);
    static const bool verbose = std::getenv("RMR_TUNE_VERBOSE") != nullptr;
    if (verbose)
        fprintf(stderr, "group of %zu layers from %d at %d images: %.1f us one by one, conv_sb variant %d %.1f us in one launch -> %s\n", ops.size(), ops.front(), n,
                sum_ms * 1e3f, best_v, best_ms * 1e3f, best_v >= 0 && best_ms < 0.97f * sum_ms ? "grouped" : "one by one");
    if (best_v >= 0 && best_ms < 0.97f * sum_ms) {
        ensure_group_table(g, n, best_v);
        tuned_[{ops.front(), n}] = kSbGroupBase + best_v;
        for (size_t k = 1; k < ops.size(); ++k) tuned_[{ops[k], n}] = kGroupedAway;
    }
}

void Yolov8::compact_arenas() {
    // merge the allocations of a group into one block (their relative placement is part of the plan)
    struct Block {
        size_t off, size;
        int arena;
        int first = 1 << 30, last = -1;
        size_t new_off = 0;
    };
    std::vector<Block> blocks;
    for (const Alloc& a : allocs_) {
        if (a.group && !blocks.empty() && blocks.back().arena == a.arena && blocks.back().off + blocks.back().size == a.off &&
            &a != &allocs_.front() && (&a)[-1].group == a.group) {
            blocks.back().size += a.size;
            continue;
        }
        blocks.push_back(Block{a.off, a.size, a.arena});
    }
    const auto block_of = [&](int arena, size_t off) -> Block* {
        for (Block& b : blocks)
            if (b.arena == arena && off >= b.off && off < b.off + b.size) return &b;
        return nullptr;
    };
    // lifetimes: the ops run in order on one stream
    for (int i0 = 0; i0 < (int)ops_.size(); ++i0) {
        const Op& op = ops_[i0];
        // the ops of a group may run in one launch: what any of them touches lives over the whole group
        const int i = i0, i_hi = op.group >= 0 ? groups_[op.group].back() : i0, i_lo = op.group >= 0 ? groups_[op.group].front() : i0;
        const auto touch = [&](int arena, size_t off, int) {
            if (Block* b = block_of(arena, off)) b->first = std::min(b->first, i_lo), b->last = std::max(b->last, i_hi);
        };
        const auto view = [&](const View& v, bool f32) {
            if (v.c || v.cs) touch(f32 ? 1 : 0, v.off, i);
        };
        switch (op.kind) {
            case OP_CONV:
                if (!op.in_is_input) view(op.in, false);
                view(op.out, op.out_f32);
                view(op.res, false);
                view(op.pre, true);
                if (op.fp8) touch(2, op.q_off, i);
                if (op.q_out) touch(2, op.q_out_off, i);
                // planar channel groups: the view names the first slab, the op touches all of them
                if (op.in_slab_c)
                    for (int k = 1; k < op.in.c / op.in_slab_c; ++k) touch(0, op.in.off + k * op.in_slab_step, i);
                if (op.out_slab_c)
                    for (int k = 1; k < op.out.c / op.out_slab_c; ++k) touch(0, op.out.off + k * op.out_slab_step, i);
                break;
            case OP_QUANT:
                view(op.in, false);
                touch(2, op.q_off, i);
                break;
            case OP_SPPF:
                view(op.in, false);
                break;
            case OP_UP:
                view(op.in, false);
                view(op.out, false);
                break;
            case OP_HEAD:
                if (op.box_conv >= 0) {
                    view(op.hb, false);
                    view(op.hc, false);
                } else {
                    view(op.box, true);
                    view(op.cls, true);
                }
                break;
        }
    }
    // RMR_FP8_FUSE=1: an e4m3 buffer written by a producing layer's epilogue holds that layer's Cout channels only -- the bytes
    // between Cout and the row pitch must stay the zeros of the arena's one-time memset (the consumer's last 64-channel chunk
    // reads them), so such a buffer never shares memory with another (a quantiser pass rewrites the whole pitch: those share)
    for (const Op& op : ops_)
        if (op.kind == OP_CONV && op.q_out)
            if (Block* b = block_of(2, op.q_out_off)) b->first = 0, b->last = (int)ops_.size() - 1;
    // first fit in order of first use: a block may take the memory of blocks that died before it is born
    size_t top[3] = {0, 0, 0};
    std::vector<Block*> order;
    for (Block& b : blocks)
        if (b.last >= 0) order.push_back(&b);
    std::stable_sort(order.begin(), order.end(), [](const Block* a, const Block* b) { return a->first < b->first; });
    std::vector<Block*> placed;
    for (Block* b : order) {
        size_t pos = 0;
        for (bool moved = true; moved;) {
            moved = false;
            for (const Block* o : placed)
                if (o->arena == b->arena && !(o->last < b->first || b->last < o->first) && pos < o->new_off + o->size &&
                    o->new_off < pos + b->size) {
                    pos = o->new_off + o->size;
                    moved = true;
                }
        }
        b->new_off = pos;
        top[b->arena] = std::max(top[b->arena], pos + b->size);
        placed.push_back(b);
    }
    // move every view
    const auto move = [&](View& v, bool f32) {
        if (!(v.c || v.cs)) return;
        if (const Block* b = block_of(f32 ? 1 : 0, v.off)) v.off = b->new_off + (v.off - b->off);
    };
    const auto move8 = [&](size_t& off) {
        if (const Block* b = block_of(2, off)) off = b->new_off + (off - b->off);
    };
    for (Op& op : ops_) {
        const bool out32 = op.kind == OP_CONV && op.out_f32;
        if (!(op.kind == OP_CONV && op.in_is_input)) move(op.in, false);
        move(op.out, out32);
        move(op.res, false);
        move(op.pre, true);
        move(op.box, true);
        move(op.cls, true);
        move(op.hb, false);
        move(op.hc, false);
        if (op.fp8 || op.kind == OP_QUANT) move8(op.q_off);
        if (op.q_out) move8(op.q_out_off);
    }
    for (auto& kv : named_) move(kv.second.v, false);
    arena_halves_ = top[0], arena_floats_ = top[1], arena_bytes8_ = top[2];
}

// whether conv_pw has a variant for a 1x1 layer of this shape (the planner's slab decision)
bool Yolov8::pw_can(int K, int N, int h, int w, bool pre) const {
    ConvArgs a{};
    a.KH = a.KW = 1;
    a.stride = 1;
    a.H = a.Ho = h;
    a.W = a.Wo = w;
    a.Cin = a.K = a.Kp = K;
    a.Cout_pad = N;
    a.in_cs = K;
    a.out_cs = N;
    a.N = 1;
    a.M = h * w;
    a.in_bytes = 1;
    a.out = (__half*)1;
    if (pre) a.pre = (const float*)1;
    return conv_pw_supported(a, -1);
}

static int make_divisible(double x, int d) { return (int)std::ceil(x / d) * d; }

Yolov8::Yolov8(DeviceCtx& ctx, const std::string& pack_path, int expect_nc, int in_w, int in_h, int max_batch, bool fp8)
    : ctx_(ctx), in_w_(in_w), in_h_(in_h), max_batch_(max_batch), fp8_(fp8) {
    if (in_w <= 0 || in_h <= 0 || in_w % 32 || in_h % 32)
        fail(RMR_ERR_INVALID_ARGUMENT, "network input %dx%d must be a positive multiple of 32", in_w, in_h);
    if (max_batch < 1) fail(RMR_ERR_INVALID_ARGUMENT, "max_batch_size must be >= 1");
    ctx.use();
    const WeightPack p = WeightPack::load(pack_path);
    nc_ = (int)p.nc;
    if (expect_nc > 0 && expect_nc != nc_)
        fail(RMR_ERR_INVALID_ARGUMENT, "weight pack '%s' has %d classes, Detector was given %d", pack_path.c_str(), nc_, expect_nc);
    if (p.reg_max != 16) fail(RMR_ERR_RUNTIME, "only reg_max = 16 is supported");

    int chunk = 256;
    if (const char* e = std::getenv("RMR_CHUNK")) chunk = std::max(1, std::atoi(e));
    if (const char* e = std::getenv("RMR_AUTOTUNE")) autotune_ = std::atoi(e) != 0;
    if (const char* e = std::getenv("RMR_GRAPH")) graph_max_batch_ = atoi(e);
    if (const char* e = std::getenv("RMR_FUSE_LB")) fuse_lb_ = atoi(e) != 0;
    if (const char* e = std::getenv("RMR_FUSE_UP")) fuse_up_ = atoi(e) != 0;
    if (const char* e = std::getenv("RMR_SLABS")) slabs_ = atoi(e) != 0;
    if (const char* e = std::getenv("RMR_FP8")) fp8_ = fp8_ || atoi(e) != 0;
    chunk_ = std::min(chunk, max_batch);

    int ch[5];
    const int basech[5] = {64, 128, 256, 512, 1024};
    for (int i = 0; i < 5; ++i) ch[i] = make_divisible(std::min<double>(basech[i], p.max_ch) * p.width, 8);
    auto rep = [&](int r) { return std::max((int)std::lround(r * p.depth), 1); };
    const int n0 = rep(3), n1 = rep(6), n2 = rep(6), n3 = rep(3), nh = rep(3);
    const int H = in_h, W = in_w;

    View x0;
    x0.cs = 8;
    x0.c = 8;
    x0.h = H;
    x0.w = W;
    View l0 = alloc(H / 2, W / 2, ch[0]);
    conv(add_conv_weights(p, "model.0.conv", 8), x0, l0, 2, 1, nullptr, false, true);
    named_["model.0"] = {l0};
    View l1 = alloc(H / 4, W / 4, ch[1]);
    conv(add_conv_weights(p, "model.1.conv", 0), l0, l1, 2, 1);
    named_["model.1"] = {l1};
    View l2 = c2f(p, "model.2", l1, n0, true, nullptr);
    named_["model.2"] = {l2};
    View l3 = alloc(H / 8, W / 8, ch[2]);
    conv(add_conv_weights(p, "model.3.conv", 0), l2, l3, 2, 1);
    named_["model.3"] = {l3};
    // the two nearest-neighbour upsamples feed 1x1 convolutions only: folded into them (c2f) where the
    // channel counts suit the kernels that carry the addend; the concat buffers then hold the skip alone
    const bool fold11 = fuse_up_ && ch[4] % 32 == 0 && ch[3] % 32 == 0, fold14 = fuse_up_ && ch[3] % 32 == 0 && ch[2] % 32 == 0;
    View cat14 = alloc(H / 8, W / 8, fold14 ? ch[2] : ch[3] + ch[2]);  // [up(model.12), model.4]
    View l4v = fold14 ? cat14 : slice(cat14, ch[3], ch[2]);
    View l4 = c2f(p, "model.4", l3, n1, true, &l4v);
    named_["model.4"] = {l4};
    View l5 = alloc(H / 16, W / 16, ch[3]);
    conv(add_conv_weights(p, "model.5.conv", 0), l4, l5, 2, 1);
    named_["model.5"] = {l5};
    View cat11 = alloc(H / 16, W / 16, fold11 ? ch[3] : ch[4] + ch[3]);  // [up(model.9), model.6]
    View l6v = fold11 ? cat11 : slice(cat11, ch[4], ch[3]);
    View l6 = c2f(p, "model.6", l5, n2, true, &l6v);
    named_["model.6"] = {l6};
    View l7 = alloc(H / 32, W / 32, ch[4]);
    conv(add_conv_weights(p, "model.7.conv", 0), l6, l7, 2, 1);
    named_["model.7"] = {l7};
    View l8 = c2f(p, "model.8", l7, n3, true, nullptr);
    named_["model.8"] = {l8};
    // SPPF
    const int cs = ch[4] / 2;
    if (cs % 8) fail(RMR_ERR_RUNTIME, "SPPF hidden width %d is not a multiple of 8", cs);
    View spp = alloc(H / 32, W / 32, 4 * cs);
    conv(add_conv_weights(p, "model.9.cv1.conv", 0), l8, slice(spp, 0, cs), 1, 1);
    {
        Op op{};
        op.kind = OP_SPPF;
        op.in = slice(spp, 0, cs);
        ops_.push_back(op);
    }
    View cat20 = alloc(H / 32, W / 32, ch[3] + ch[4]);  // [model.19, model.9]
    View l9 = slice(cat20, ch[3], ch[4]);
    conv(add_conv_weights(p, "model.9.cv2.conv", 0), spp, l9, 1, 1);
    named_["model.9"] = {l9};
    // neck
    const auto upsample = [&](const View& in, const View& out) {
        Op op{};
        op.kind = OP_UP;
        op.in = in;
        op.out = out;
        ops_.push_back(op);
    };
    if (!fold11) upsample(l9, slice(cat11, 0, ch[4]));
    View cat17 = alloc(H / 16, W / 16, ch[2] + ch[3]);  // [model.16, model.12]
    View l12v = slice(cat17, ch[2], ch[3]);
    View l12 = c2f(p, "model.12", cat11, nh, false, &l12v, fold11 ? &l9 : nullptr);
    named_["model.12"] = {l12};
    if (!fold14) upsample(l12, slice(cat14, 0, ch[3]));
    View l15 = c2f(p, "model.15", cat14, nh, false, nullptr, fold14 ? &l12 : nullptr);
    named_["model.15"] = {l15};
    conv(add_conv_weights(p, "model.16.conv", 0), l15, slice(cat17, 0, ch[2]), 2, 1);
    View l18 = c2f(p, "model.18", cat17, nh, false, nullptr);
    named_["model.18"] = {l18};
    conv(add_conv_weights(p, "model.19.conv", 0), l18, slice(cat20, 0, ch[3]), 2, 1);
    View l21 = c2f(p, "model.21", cat20, nh, false, nullptr);
    named_["model.21"] = {l21};

    // Detect.  Its 3x3 convolutions produce the box-distribution logits directly: they stay f16 in the fp8 plan
    // (RMR_FP8_HEAD=1 takes them along: 9 % of the FLOPs, measured to double the box error)
    fp8_layer_ = std::getenv("RMR_FP8_HEAD") && atoi(std::getenv("RMR_FP8_HEAD")) != 0;
    const View feats[3] = {l15, l18, l21};
    const int strides[3] = {8, 16, 32};
    anchors_ = 0;
    for (int i = 0; i < 3; ++i) anchors_ += feats[i].h * feats[i].w;
    int a_off = 0;
    const int cls_pad = (nc_ + 15) / 16 * 16;
    std::vector<Op> head_ops;
    // depth-major: the first convolutions of the three scales, then the six second ones, then the six third ones -- the
    // convolutions of one depth are independent of each other, consecutive in the op list, and can leave in ONE launch
    // (find_groups; a batch-1 layer is mostly fixed cost: 15 launches become 3)
    struct HeadScale {
        View h1, hb, hc, box, cls;
        int c2d, c3d;
    } hs[3];
    for (int i = 0; i < 3; ++i) {
        const View& f = feats[i];
        const std::string b = "model.22.cv2." + std::to_string(i), c = "model.22.cv3." + std::to_string(i);
        hs[i].c2d = (int)p.get(b + ".0.conv.weight").dims[0];
        hs[i].c3d = (int)p.get(c + ".0.conv.weight").dims[0];
        hs[i].h1 = alloc(f.h, f.w, hs[i].c2d + hs[i].c3d);
        conv(add_fused_head_weights(p, b + ".0.conv", c + ".0.conv"), f, hs[i].h1, 1, 1);
    }
    for (int i = 0; i < 3; ++i) {
        const View& f = feats[i];
        const std::string b = "model.22.cv2." + std::to_string(i), c = "model.22.cv3." + std::to_string(i);
        hs[i].hb = alloc(f.h, f.w, hs[i].c2d), hs[i].hc = alloc(f.h, f.w, hs[i].c3d);
        conv(add_conv_weights(p, b + ".1.conv", 0), slice(hs[i].h1, 0, hs[i].c2d), hs[i].hb, 1, 1);
        conv(add_conv_weights(p, c + ".1.conv", 0), slice(hs[i].h1, hs[i].c2d, hs[i].c3d), hs[i].hc, 1, 1);
    }
    for (int i = 0; i < 3; ++i) {
        const View& f = feats[i];
        const std::string b = "model.22.cv2." + std::to_string(i), c = "model.22.cv3." + std::to_string(i);
        // RMR_FUSE_HEAD=0: the last 1x1 convolutions as launches of their own into f32 logit tensors + the decode pass over them
        // (rounds 1-5); default: one launch does all three (net_ops.hip head_fused_kernel), the logit tensors do not exist
        const bool fuse_head = !(std::getenv("RMR_FUSE_HEAD") && atoi(std::getenv("RMR_FUSE_HEAD")) == 0) &&
                               head_fused_supported(hs[i].c2d, hs[i].c3d, nc_) && cls_pad == 16;
        Op op{};
        op.kind = OP_HEAD;
        if (fuse_head) {
            op.box_conv = add_conv_weights(p, b + ".2", 0);
            op.cls_conv = add_conv_weights(p, c + ".2", 0);
            op.hb = hs[i].hb, op.hc = hs[i].hc;
            for (int widx : {op.box_conv, op.cls_conv})   // the FLOPs conv() would have declared
                flops_ += 2.0 * f.h * f.w * (double)convs_[widx].cout * convs_[widx].cin;
        } else {
            hs[i].box = alloc(f.h, f.w, 64, true), hs[i].cls = alloc(f.h, f.w, cls_pad, true);
            conv(add_conv_weights(p, b + ".2", 0), hs[i].hb, hs[i].box, 1, 0, nullptr, true);
            conv(add_conv_weights(p, c + ".2", 0), hs[i].hc, hs[i].cls, 1, 0, nullptr, true);
        }
        op.box = hs[i].box;
        op.cls = hs[i].cls;
        op.head_stride = strides[i];
        op.a_off = a_off;
        op.in = f;
        head_ops.push_back(op);
        a_off += f.h * f.w;
    }
    // the three scales' decodes go last, together: one launch (run_op), the logits live until then
    for (const Op& op : head_ops) ops_.push_back(op);

    // fp8 plan: a tensor that leaves its producer as e4m3 (q_out) and has no other reader than the e4m3 layer behind it
    // is never written as f16 (the stage-output hook, RMR_ARENA_REUSE=0, keeps every f16 tensor)
    if (const char* e = std::getenv("RMR_ARENA_REUSE")) arena_reuse_ = atoi(e) != 0;
    for (size_t pi = 0; pi < ops_.size() && arena_reuse_; ++pi) {
        Op& p = ops_[pi];
        if (p.kind != OP_CONV || !p.q_out) continue;
        const auto reads = [&](const View& v) { return (v.c || v.cs) && v.off == p.out.off && v.co < p.out.co + p.out.c && p.out.co < v.co + v.c; };
        bool only = true;
        int readers = 0;
        for (size_t i = 0; i < ops_.size() && only; ++i) {
            if (i == pi) continue;
            const Op& o = ops_[i];
            if (o.kind == OP_CONV && reads(o.in) && !o.in_is_input) {
                if (o.fp8 && o.q_off == p.q_out_off && !reads(o.res) && !reads(o.pre)) ++readers;
                else only = false;
            } else if ((o.kind != OP_CONV && reads(o.in)) || reads(o.res) || reads(o.pre) || (o.kind == OP_UP && reads(o.out))) {
                only = false;
            }
            if (o.in_slab_c || o.out_slab_c) {   // a slabbed 1x1 names the first slab only: any slab of its group may be ours
                const size_t lo = o.in_slab_c ? o.in.off : o.out.off, step = o.in_slab_c ? o.in_slab_step : o.out_slab_step;
                const int cnt = o.in_slab_c ? o.in.c / o.in_slab_c : o.out.c / o.out_slab_c;
                for (int k = 0; k < cnt; ++k) only = only && lo + k * step != p.out.off;
            }
        }
        for (const auto& kv : named_) only = only && kv.second.v.off != p.out.off;
        // a producer with a shortcut keeps its f16 output: the e4m3-only epilogue has no residual form (conv_t32f8 rejects it)
        p.q_only = only && readers == 1 && !(p.res.c || p.res.cs);
    }
    // Fusable bottlenecks (conv_wsf: both 3x3 convolutions of a C2f bottleneck in one launch, the hidden tensor in LDS): op i
    // and op i + 1 are 3x3 / stride-1 / 48 -> 48 convolutions on 160-wide maps with SiLU, the second reads the first's output
    // and adds the first's input, and nobody else reads the hidden tensor.  The pairs are always found (a plan may name the
    // fused kernel for them); whether the TUNER tries the fused launch is RMR_FUSE_WS (default off, see run_op).
    {
        const auto same = [](const View& x, const View& y) { return x.off == y.off && x.co == y.co && x.c == y.c && x.cs == y.cs && x.h == y.h && x.w == y.w; };
        for (size_t i = 0; i + 1 < ops_.size(); ++i) {
            Op& a = ops_[i];
            const Op& b = ops_[i + 1];
            if (a.kind != OP_CONV || b.kind != OP_CONV || a.fp8 || b.fp8 || a.out_f32 || b.out_f32 || a.in_is_input) continue;
            const ConvW &wa = convs_[a.conv], &wb = convs_[b.conv];
            if (wa.k != 3 || wb.k != 3 || a.stride != 1 || b.stride != 1 || !a.act || !b.act) continue;
            if (wa.cin != 48 || wa.cout_pad != 48 || wb.cin != 48 || wb.cout_pad != 48 || a.in.w != 160) continue;
            if (a.res.c || a.pre.c || b.pre.c || a.in_slab_c || a.out_slab_c || b.in_slab_c || b.out_slab_c) continue;
            if (!same(b.in, a.out) || !b.res.c || !same(b.res, a.in)) continue;
            const auto reads = [&](const View& v) { return (v.c || v.cs) && v.off == a.out.off && v.co < a.out.co + a.out.c && a.out.co < v.co + v.c; };
            bool only = true;
            for (size_t k = 0; k < ops_.size() && only; ++k) {
                if (k == i || k == i + 1) continue;
                const Op& o = ops_[k];
                only = !(reads(o.in) || reads(o.res) || reads(o.pre) || (o.kind == OP_UP && reads(o.out)));
                if (o.in_slab_c || o.out_slab_c) {   // a slabbed 1x1 names its first slab only
                    const size_t lo = o.in_slab_c ? o.in.off : o.out.off, step = o.in_slab_c ? o.in_slab_step : o.out_slab_step;
                    const int cnt = o.in_slab_c ? o.in.c / o.in_slab_c : o.out.c / o.out_slab_c;
                    for (int q = 0; q < cnt; ++q) only = only && lo + q * step != a.out.off;
                }
            }
            for (const auto& kv : named_) only = only && kv.second.v.off != a.out.off;
            if (only) a.fuse_with = (int)i + 1;
        }
    }
    find_groups();
    if (arena_reuse_) compact_arenas();
    // Images per launch: every activation view (pixels x its buffer's channel pitch, plus the span of its
    // slabs) must stay below the 32-bit offset range of the kernels' buffer resources.  256 images of a
    // 640 x 640 network are far below it; a 1920 x 1088 network is not.
    {
        size_t worst = 0;  // bytes per image of the largest view
        for (const Op& op : ops_) {
            for (const View* v : {&op.in, &op.out, &op.res}) {
                if (!v->c && !v->cs) continue;
                size_t bytes = (size_t)v->h * v->w * v->cs * sizeof(__half);
                if (v == &op.in && op.in_slab_c) bytes += (size_t)(op.in.c / op.in_slab_c - 1) * op.in_slab_step * sizeof(__half);
                if (v == &op.out && op.out_slab_c) bytes += (size_t)(op.out.c / op.out_slab_c - 1) * op.out_slab_step * sizeof(__half);
                worst = std::max(worst, bytes);
            }
        }
        worst = std::max(worst, (size_t)H * W * 8 * sizeof(__half));
        const size_t fit = std::max<size_t>(1, kMaxViewBytes / std::max<size_t>(worst, 1));
        if ((size_t)chunk_ > fit) chunk_ = (int)fit;
    }
    splitk_ws_.alloc(kSplitKWsFloats);
    splitk_cnt_.alloc(kSplitKMaxTiles);
    RMR_HIP(hipMemset(splitk_cnt_.p, 0, kSplitKMaxTiles * sizeof(int)));
    tune_path_ = pack_path + ".tune";
    if (const char* e = std::getenv("RMR_PLAN")) {
        if (*e && std::strcmp(e, "0") != 0) {
            if (std::strcmp(e, "1") != 0) tune_path_ = e;  // "1": the pack's own '<pack>.tune', taken as it is
            pinned_ = true;
            autotune_ = true;
        }
    }
    arena_.alloc(arena_halves_ * chunk_);
    arena32_.alloc(arena_floats_ * chunk_);
    if (arena_bytes8_) {
        if (arena_bytes8_ * chunk_ > kMaxViewBytes * 16) fail(RMR_ERR_CAPACITY, "fp8 plan: quantised activations do not fit");
        arena8_.alloc(arena_bytes8_ * chunk_);
        RMR_HIP(hipMemset(arena8_.p, 0, arena8_.n));  // the bytes beyond a layer's channels stay zero for ever
    }
    input_.alloc((size_t)max_batch_ * H * W * 8);
    output_.alloc((size_t)max_batch_ * (4 + nc_) * anchors_);
    RMR_HIP(hipMemset(arena_.p, 0, arena_.n * sizeof(__half)));
    RMR_HIP(hipMemset(arena32_.p, 0, arena32_.n * sizeof(float)));
    if (autotune_) load_tuning();  // after the arenas: cached choices are re-validated against the live layer arguments
}

// ---- executor ---------------------------------------------------------------------------------------

// Times every kernel variant that can run this layer (conv_igemm tiles of both K depths, conv_dma
// tiles) on the live buffers and returns the fastest.  A conv launch is idempotent (its output
// slice never aliases its input or residual slice), so re-running it is harmless.  Runs once per
// (layer, batch) -- the analogue of the reference's TensorRT engine build (detector.cpp:177-243).
void Yolov8::launch_choice(hipStream_t s, ConvArgs a, int choice) {
    if (choice >= kSbBase) {   // the small-batch family (conv_sb.hip)
        launch_conv_sb(ctx_, s, a, choice - kSbBase);
        return;
    }
    const int split = choice / 1000, c = choice % 1000;
    if ((a.in_slab_c || a.out_slab_c) && (c < 700 || c >= 800 || split))
        fail(RMR_ERR_LOGIC, "kernel %d cannot address planar channel groups", choice);
    if (c >= 980) {
        launch_conv_w1d(ctx_, s, a, c - 980);
    } else if (c >= 950) {
        launch_conv_g32(ctx_, s, a, c - 950);
    } else if (c >= 900) {
        launch_conv_t32f8(ctx_, s, a, c - 900);
    } else if (c >= 800) {
        if (split > 1) {
            a.split = split;
            a.splitk_ws = splitk_ws_.p;
            a.splitk_cnt = splitk_cnt_.p;
        }
        launch_conv_t32(ctx_, s, a, c - 800);
    } else if (c >= 700) {
        launch_conv_pw(ctx_, s, a, c - 700);
    } else if (c >= 600) {
        launch_conv_ws_s2(ctx_, s, a, c - 600);
    } else if (c == 500) {
        launch_conv_stem(ctx_, s, a);
    } else if (c >= 400) {
        launch_conv_direct(ctx_, s, a, c - 400);
    } else if (c >= 300) {
        launch_conv_ws(ctx_, s, a, c - 300);
    } else if (c >= 200) {
        launch_conv_halo(ctx_, s, a, c - 200);
    } else if (c >= 100) {
        if (split > 1) {
            a.split = split;
            a.splitk_ws = splitk_ws_.p;
            a.splitk_cnt = splitk_cnt_.p;
        }
        launch_conv_dma(ctx_, s, a, c - 100);
    } else {
        launch_conv(ctx_, s, a, c);
    }
}

int Yolov8::tune_conv(hipStream_t s, const ConvArgs& a, float* best_ms_out) {
    // the first layer has its own kernel (2x the next best at every batch size), which is also the
    // one that samples the frames directly: the same arithmetic whichever way the input arrives
    if (conv_stem_supported(a)) return 500;
    std::vector<int> cands;
    if (a.in8) {  // a layer of the fp8 plan: the e4m3 tiles and nothing else
        for (int t = 0; t < conv_t32f8_num_tiles(); ++t)
            if (conv_t32f8_supported(a, t)) cands.push_back(900 + t);
        if (cands.empty()) fail(RMR_ERR_LOGIC, "fp8 plan: no e4m3 tile runs a layer with N = %d on %d-wide maps", a.Cout_pad, a.W);
    }
    const bool slabbed = a.in_slab_c || a.out_slab_c;  // only conv_pw addresses planar channel groups
    if (a.in8) goto timed;
    for (int t = 0; t < conv_num_tiles() && !slabbed; ++t)
        if (a.Cout_pad % conv_tile(t).bn == 0) cands.push_back(t);
    if (!slabbed && conv_dma_supported(a))
        for (int t = 0; t < conv_dma_num_tiles(); ++t)
            if (a.Cout_pad % conv_dma_tile(t).bn == 0) cands.push_back(100 + t);
    if (!a.pre && conv_halo_supported(a, -1))
        for (int t = 0; t < conv_halo_num_tiles(); ++t)
            if (conv_halo_supported(a, t)) cands.push_back(200 + t);
    if (conv_t32_supported(a, -1))
        for (int t = 0; t < conv_t32_num_tiles(); ++t)
            if (conv_t32_supported(a, t)) cands.push_back(800 + t);
    // the same layers through Winograd F(2, 3) along x (1.5x fewer MFMAs; chip-filling launches only: a tile is 512 pixels)
    if (conv_w1d_supported(a, -1) && (a.M >= 256 * ctx_.num_cus || std::getenv("RMR_TUNE_ONLY")))
        for (int t = 0; t < conv_w1d_num_tiles(); ++t)
            if (conv_w1d_supported(a, t)) cands.push_back(980 + t);
    // 1x1 and strided 3x3 layers on the same skeleton (a chip-filling number of 256-pixel tiles only, unless a test
    // pins the family)
    if (conv_g32_supported(a, -1) && !conv_t32_supported(a, -1) && (a.M >= 128 * ctx_.num_cus || std::getenv("RMR_TUNE_ONLY")))
        for (int t = 0; t < conv_g32_num_tiles(); ++t)
            if (conv_g32_supported(a, t)) cands.push_back(950 + t);
    // fragment-direct tiles only where the staged kernels cannot fill the chip
    if (!slabbed && conv_direct_supported(a, -1) && a.M <= 64 * ctx_.num_cus)
        for (int t = 0; t < conv_direct_num_tiles(); ++t)
            if (conv_direct_supported(a, t)) cands.push_back(400 + t);
    if (conv_pw_supported(a, -1))
        for (int v = 0; v < conv_pw_num_variants(); ++v)
            if (conv_pw_supported(a, v)) cands.push_back(700 + v);
    if (!a.pre && conv_ws_s2_supported(a, -1))
        for (int v = 0; v < conv_ws_s2_num_variants(); ++v)
            if (conv_ws_s2_supported(a, v)) cands.push_back(600 + v);
    if (!a.pre && conv_ws_supported(a, -1))
        for (int v = 0; v < conv_ws_num_variants(); ++v)
            if (conv_ws_supported(a, v)) cands.push_back(300 + v);
    // split-K variants where the plain grid cannot fill the chip (small batches)
    if (!slabbed && conv_dma_supported(a))
        for (int t = 0; t < conv_dma_num_tiles(); ++t) {
            const ConvTile ct = conv_dma_tile(t);
            if (a.Cout_pad % ct.bn || ct.bm * ct.bn > 128 * 128) continue;
            const int tiles = conv_dma_splitk_tiles(a, t);
            const int nk = (a.K + ct.bk - 1) / ct.bk;
            if (tiles >= 2 * ctx_.num_cus || tiles > kSplitKMaxTiles) continue;
            for (int split : {2, 3, 4, 6, 9, 12, 18}) {
                if (split > nk / 2 || (long)tiles * split > 4L * ctx_.num_cus) break;
                if (conv_dma_splitk_ws_floats(a, t, split) > kSplitKWsFloats) break;
                cands.push_back(1000 * split + 100 + t);
            }
        }
    // ... and of conv_t32 (round 3): a 3x3 layer of a batch of 1-4 images is 7-100 tiles of 256 pixels on 256 CUs, each
    // streaming all 54-81 weight slices; with split-K every CU takes a few chunks of one tile
    if (conv_t32_supported(a, -1))
        for (int t = 0; t < conv_t32_num_tiles(); ++t) {
            if (!conv_t32_supported(a, t)) continue;
            const int tiles = conv_t32_splitk_tiles(a, t);
            if (tiles >= ctx_.num_cus || tiles > kSplitKMaxTiles) continue;
            for (int split : {2, 3, 4, 6, 9}) {
                if (!conv_t32_splitk_supported(a, t, split, ctx_.num_cus)) continue;
                if (conv_t32_splitk_ws_floats(a, t, split) > kSplitKWsFloats) break;
                cands.push_back(1000 * split + 800 + t);
            }
        }
    // small batches: tiles with their whole operand set in flight (conv_sb); offered where a layer is at most a few
    // workgroups per CU -- beyond that the throughput kernels' streams win
    if (conv_sb_supported(a, -1))
        for (int v = 0; v < conv_sb_num_variants(); ++v) {
            if (!conv_sb_supported(a, v)) continue;
            const ConvTile ct = conv_sb_tile(v);
            const long tiles = (long)((a.M + ct.bm - 1) / ct.bm) * (a.Cout_pad / ct.bn);
            if (tiles <= 6L * ctx_.num_cus) cands.push_back(kSbBase + v);
        }
    // RMR_TUNE_ONLY=lo-hi: layers that have candidates in that id range choose among those only (tests
    // use it to pin a kernel family under the whole network, e.g. 700-799 = conv_pw)
    if (const char* e = std::getenv("RMR_TUNE_ONLY")) {
        int lo = 0, hi = 0;
        if (sscanf(e, "%d-%d", &lo, &hi) == 2) {
            std::vector<int> only;
            for (int c : cands)
                if ((c >= kSbBase && c >= lo && c <= hi) || (c % 1000 >= lo && c % 1000 <= hi && c < 1000)) only.push_back(c);
            if (!only.empty()) cands.swap(only);
        }
    }
timed:
    hipEvent_t e0, e1;
    RMR_HIP(hipEventCreate(&e0));
    RMR_HIP(hipEventCreate(&e1));
    const int prof_was_on = ctx_.prof.on;
    ctx_.prof.on = 0;
    int best = cands.front();
    float best_ms = 1e30f;
    std::vector<std::pair<float, int>> timed;
    static const bool verbose = std::getenv("RMR_TUNE_VERBOSE") != nullptr;
    if (verbose) fprintf(stderr, "tune M%d N%d K%d k%d s%d:", a.M, a.Cout_pad, a.K, a.KH, a.stride);
    for (int c : cands) {
        // skip tiles that would leave most of the chip idle or are hopelessly oversized
        const int cc = c % 1000;
        if (c < kSbBase && cc < 300) {  // tiled kernels only
            const ConvTile t = cc >= 200 ? conv_halo_tile(cc - 200) : cc >= 100 ? conv_dma_tile(cc - 100) : conv_tile(cc);
            const long blocks = (long)((a.M + t.bm - 1) / t.bm) * (a.Cout_pad / t.bn);
            if (t.bm >= 256 && blocks < ctx_.num_cus / 2 && a.M > 64) continue;
        }
        float ms_min = 1e30f;
        for (int rep = 0; rep < 3; ++rep) {
            RMR_HIP(hipEventRecord(e0, s));
            launch_choice(s, a, c);
            RMR_HIP(hipEventRecord(e1, s));
            RMR_HIP(hipEventSynchronize(e1));
            float ms = 0;
            RMR_HIP(hipEventElapsedTime(&ms, e0, e1));
            if (rep > 0 && ms < ms_min) ms_min = ms;
        }
        if (verbose) fprintf(stderr, " %d:%.1f", c, ms_min * 1e3f);
        if (ms_min < best_ms) best_ms = ms_min, best = c;
        timed.emplace_back(ms_min, c);
    }
    // run-off: single launches a few percent apart are within the noise of one measurement (and of the
    // box: sessions differed by 3 % in their picks); the finalists run five times back to back, which is
    // also how they will run inside the network
    std::sort(timed.begin(), timed.end());
    size_t finalists = 0;
    while (finalists < timed.size() && finalists < 4 && timed[finalists].first <= 1.04f * best_ms) ++finalists;
    if (finalists > 1) {
        // RMR_TUNE_ROUNDS (default 2; tools/make_plan.py, whose result is committed, asks for 6): the finalists take turns
        // round after round (A B C A B C ...: a clock drift during the run-off hits all of them alike), each keeps its best round
        static const int rounds = std::getenv("RMR_TUNE_ROUNDS") ? std::max(1, std::atoi(std::getenv("RMR_TUNE_ROUNDS"))) : 2;
        std::vector<float> fmin(finalists, 1e30f);
        for (int rep = 0; rep < rounds; ++rep)
            for (size_t f = 0; f < finalists; ++f) {
                RMR_HIP(hipEventRecord(e0, s));
                for (int k = 0; k < 5; ++k) launch_choice(s, a, timed[f].second);
                RMR_HIP(hipEventRecord(e1, s));
                RMR_HIP(hipEventSynchronize(e1));
                float ms = 0;
                RMR_HIP(hipEventElapsedTime(&ms, e0, e1));
                fmin[f] = std::min(fmin[f], ms / 5);
            }
        best_ms = 1e30f;
        for (size_t f = 0; f < finalists; ++f) {
            if (verbose) fprintf(stderr, " [%d:%.1f]", timed[f].second, fmin[f] * 1e3f);
            if (fmin[f] < best_ms) best_ms = fmin[f], best = timed[f].second;
        }
    }
    if (verbose) fprintf(stderr, "  -> %d (%.1f us)\n", best, best_ms * 1e3f);
    if (best_ms_out) *best_ms_out = best_ms;
    ctx_.prof.on = prof_was_on;
    (void)hipEventDestroy(e0);
    (void)hipEventDestroy(e1);
    return best;
}

// The tuning result is cached next to the weight pack, as the reference caches its TensorRT
// engine next to the ONNX file (detector.cpp:74-99).  One line per entry: "op n choice" after a header with the op count and input size.
// The op list depends on the pack and on the planner's options (RMR_FUSE_UP): entries are per op index,
// so a cache written for another plan must not be read.
unsigned long long Yolov8::plan_signature() const {
    unsigned long long h = 1469598103934665603ull;
    const auto mix = [&](long long v) { h = (h ^ (unsigned long long)v) * 1099511628211ull; };
    for (const Op& op : ops_) {
        mix(op.kind), mix(op.in.h), mix(op.in.w), mix(op.in.c), mix(op.out.c), mix(op.stride), mix(op.pre.c), mix(op.res.c), mix(op.in_slab_c), mix(op.out_slab_c), mix(op.in.cs), mix(op.out.cs), mix(op.fp8), mix(op.q_pitch), mix(op.q_out), mix(op.q_only), mix(op.group);
        if (op.kind == OP_CONV) mix(convs_[op.conv].K), mix(convs_[op.conv].cout_pad);
        if (op.kind == OP_HEAD) mix(op.box_conv >= 0);
    }
    return h;
}

// whether kernel `choice` can run layer `a` (what tune_conv would have offered): a cache line is only as
// trustworthy as the file it came from
bool Yolov8::choice_supported(const ConvArgs& a, int choice) const {
    if (choice < 0) return false;
    if (choice >= kSbBase) return conv_sb_supported(a, choice - kSbBase);
    const int c = choice % 1000, split = choice / 1000;
    const bool slabbed = a.in_slab_c || a.out_slab_c;
    if (split && c >= 800 && c < 900)
        return !slabbed && !a.in8 && c - 800 < conv_t32_num_tiles() && conv_t32_splitk_supported(a, c - 800, split, ctx_.num_cus) &&
               conv_t32_splitk_tiles(a, c - 800) <= kSplitKMaxTiles && conv_t32_splitk_ws_floats(a, c - 800, split) <= kSplitKWsFloats;
    if (split) {
        if (split > 64 || c < 100 || c >= 200 || slabbed || !conv_dma_supported(a) || c - 100 >= conv_dma_num_tiles()) return false;
        const ConvTile ct = conv_dma_tile(c - 100);
        return a.Cout_pad % ct.bn == 0 && conv_dma_splitk_tiles(a, c - 100) <= kSplitKMaxTiles &&
               conv_dma_splitk_ws_floats(a, c - 100, split) <= kSplitKWsFloats;
    }
    if (a.in8) return !split && c >= 900 && c - 900 < conv_t32f8_num_tiles() && conv_t32f8_supported(a, c - 900);
    if (c >= 980) return c - 980 < conv_w1d_num_tiles() && conv_w1d_supported(a, c - 980);
    if (c >= 950) return c - 950 < conv_g32_num_tiles() && conv_g32_supported(a, c - 950);
    if (c >= 900) return false;
    if (c >= 800) return c - 800 < conv_t32_num_tiles() && conv_t32_supported(a, c - 800);
    if (c >= 700) return c - 700 < conv_pw_num_variants() && conv_pw_supported(a, c - 700);
    if (slabbed) return false;  // only conv_pw addresses planar channel groups
    if (c >= 600) return !a.pre && c - 600 < conv_ws_s2_num_variants() && conv_ws_s2_supported(a, c - 600);
    if (c == 500) return conv_stem_supported(a);
    if (c >= 400) return c - 400 < conv_direct_num_tiles() && conv_direct_supported(a, c - 400);
    if (c >= 340) return false;   // fused bottlenecks (340.., kFusedAway): load_tuning() checks them against the op pair
    if (c >= 300) return !a.pre && c - 300 < conv_ws_num_variants() && conv_ws_supported(a, c - 300);
    if (c >= 200) return !a.pre && c - 200 < conv_halo_num_tiles() && conv_halo_supported(a, c - 200);
    if (c >= 100) return c - 100 < conv_dma_num_tiles() && conv_dma_supported(a) && a.Cout_pad % conv_dma_tile(c - 100).bn == 0;
    return c < conv_num_tiles() && a.Cout_pad % conv_tile(c).bn == 0;
}

// header: "rmr-tune <version> <ops> <w> <h> <plan signature> <CUs> <device name without blanks>"
// (the version moves whenever the set of candidate kernels does: 11 = conv_g32 added, 12 = conv_w1d, 13 = split-K conv_t32, 14 = conv_t32 tiles 13-14,
// 15 = conv_wsp (conv_ws variants 12-16), conv_w1d out of the product build, 16 = fused bottlenecks (conv_wsf, 340.. + 399),
// 17 = the small-batch family conv_sb (100000..))
static constexpr int kTuneFileVersion = 17;
int Yolov8::tune_file_version() { return kTuneFileVersion; }
static std::string device_tag(int device) {
    hipDeviceProp_t p;
    if (hipGetDeviceProperties(&p, device) != hipSuccess) return "unknown";
    std::string n = p.gcnArchName;
    for (char& ch : n)
        if (ch == ' ' || ch == '\t') ch = '_';
    return n.empty() ? "unknown" : n;
}

void Yolov8::load_tuning() {
    // RMR_PLAN=<file>: a pinned plan -- the kernel per (layer, batch) comes from that file and nothing is ever
    // timed, so two boxes (or two runs) launch the same kernels and produce bit-identical outputs
    std::ifstream f(tune_path_);
    if (!f) return;
    std::string tag, dev;
    int version = 0, n_ops = 0, w = 0, h = 0, cus = 0;
    unsigned long long sig = 0;
    f >> tag >> version >> n_ops >> w >> h >> sig >> cus >> dev;
    if (tag != "rmr-tune" || version != kTuneFileVersion || n_ops != (int)ops_.size() || w != in_w_ || h != in_h_ || sig != plan_signature())
        return;
    // timings from another chip say nothing about this one (a pinned plan is taken as it is)
    if (!pinned_ && (cus != ctx_.num_cus || dev != device_tag(ctx_.device))) return;
    int op, n, choice;
    while (f >> op >> n >> choice) {
        if (op < 0 || op >= (int)ops_.size() || ops_[op].kind != OP_CONV || n < 1 || n > chunk_) continue;
        if (choice == kGroupedAway) {
            if (ops_[op].group >= 0 && groups_[ops_[op].group].front() != op) tuned_[{op, n}] = choice;
        } else if (choice >= kSbGroupBase) {
            const int g = ops_[op].group;
            if (g >= 0 && groups_[g].front() == op) {
                const std::vector<ConvArgs> args = group_args(g, n);
                if (conv_sb_group_supported(args.data(), (int)args.size(), choice - kSbGroupBase)) tuned_[{op, n}] = choice;
            }
        } else if (choice == kFusedAway) {
            if (op > 0 && ops_[op - 1].kind == OP_CONV && ops_[op - 1].fuse_with == op) tuned_[{op, n}] = choice;
        } else if (choice >= 340 && choice < kFusedAway) {
            if (ops_[op].fuse_with >= 0 && conv_wsf_supported(fused_args(op, n, 0), choice - 340)) tuned_[{op, n}] = choice;
        } else if (choice_supported(conv_args(op, n, 0), choice)) {
            tuned_[{op, n}] = choice;
        }
    }
    // a fused bottleneck is two entries that only make sense together: "done by the layer before" without a fused choice
    // on that layer would leave a tensor unwritten
    for (auto it = tuned_.begin(); it != tuned_.end();) {
        const int op2 = it->first.first, n2 = it->first.second;
        bool drop = false;
        if (it->second == kFusedAway) {
            const auto f = tuned_.find({op2 - 1, n2});
            drop = f == tuned_.end() || f->second < 340 || f->second >= kFusedAway;
        }
        it = drop ? tuned_.erase(it) : std::next(it);
    }
    // a grouped launch is an entry on the group's first layer and "done by the group's launch" on all the others: anything
    // less (a hand-edited or truncated file) falls back to tuning the whole group again
    for (size_t g = 0; g < groups_.size(); ++g) {
        std::map<int, int> per_n;   // images -> 0 none, 1 consistent group, -1 broken
        for (const auto& kv : tuned_)
            if (ops_[kv.first.first].group == (int)g && (kv.second >= kSbGroupBase || kv.second == kGroupedAway)) per_n[kv.first.second] = 0;
        for (auto& pn : per_n) {
            const int n2 = pn.first;
            bool ok = tuned_.count({groups_[g].front(), n2}) && tuned_[{groups_[g].front(), n2}] >= kSbGroupBase;
            for (size_t k = 1; k < groups_[g].size() && ok; ++k) ok = tuned_.count({groups_[g][k], n2}) && tuned_[{groups_[g][k], n2}] == kGroupedAway;
            if (ok)
                ensure_group_table((int)g, n2, tuned_[{groups_[g].front(), n2}] - kSbGroupBase);
            else
                for (int op2 : groups_[g]) tuned_.erase({op2, n2});
        }
    }
    for (auto& kv : tuned_)
        if (kv.second >= 340 && kv.second < kFusedAway) {
            const auto f = tuned_.find({ops_[kv.first.first].fuse_with, kv.first.second});
            if (f == tuned_.end() || f->second != kFusedAway) tuned_[{ops_[kv.first.first].fuse_with, kv.first.second}] = kFusedAway;
        }
}

void Yolov8::save_tuning() {
    if (pinned_) return;
    // one process per GPU may share a pack: write a private file, then rename it over the cache (atomic)
    const std::string tmp = tune_path_ + ".tmp" + std::to_string((long)getpid());
    {
        std::ofstream f(tmp, std::ios::trunc);
        if (!f) return;  // read-only location: tune again next time
        f << "rmr-tune " << kTuneFileVersion << ' ' << ops_.size() << ' ' << in_w_ << ' ' << in_h_ << ' ' << plan_signature() << ' ' << ctx_.num_cus << ' '
          << device_tag(ctx_.device) << "\n";
        for (const auto& kv : tuned_) f << kv.first.first << ' ' << kv.first.second << ' ' << kv.second << "\n";
        if (!f) {
            std::remove(tmp.c_str());
            return;
        }
    }
    if (std::rename(tmp.c_str(), tune_path_.c_str()) != 0) std::remove(tmp.c_str());
}

ConvArgs Yolov8::conv_args(int op_index, int n, size_t img0) {
    const Op& op = ops_[op_index];
    auto hptr = [&](const View& v) { return arena_.p + v.off * chunk_; };
    auto fptr = [&](const View& v) { return arena32_.p + v.off * chunk_; };
    const ConvW& cw = convs_[op.conv];
    ConvArgs a{};
    a.in = op.in_is_input ? input_.p + img0 * in_h_ * in_w_ * 8 : hptr(op.in);
    a.in_cs = op.in.cs;
    a.in_co = op.in.co;
    a.N = n;
    a.H = op.in.h;
    a.W = op.in.w;
    a.Cin = cw.cin;
    a.Ho = op.out.h;
    a.Wo = op.out.w;
    a.KH = a.KW = cw.k;
    a.stride = op.stride;
    a.pad = cw.k / 2;
    a.wt = cw.w.p;
    a.bias = cw.b.p;
    if (op.out_f32)
        a.out32 = fptr(op.out);
    else
        a.out = hptr(op.out);
    a.out_cs = op.out.cs;
    a.out_co = op.out.co;
    if (op.res.c) {
        a.res = hptr(op.res);
        a.res_cs = op.res.cs;
        a.res_co = op.res.co;
    }
    if (op.pre.c) {
        a.pre = fptr(op.pre);
        a.pre_cs = op.pre.cs;
    }
    if (op.in_slab_c) {
        a.in_slab_c = op.in_slab_c;
        a.in_slab_stride = (unsigned)(op.in_slab_step * chunk_ * sizeof(__half));
    }
    if (op.out_slab_c) {
        a.out_slab_c = op.out_slab_c;
        a.out_slab_stride = (unsigned)(op.out_slab_step * chunk_ * sizeof(__half));
    }
    a.Cout_pad = cw.cout_pad;
    a.K = cw.K;
    a.Kp = cw.Kp;
    a.M = n * a.Ho * a.Wo;
    a.act = op.act;
    const size_t in_bytes = (size_t)n * a.H * a.W * a.in_cs * sizeof(__half) +
                            (op.in_slab_c ? (size_t)(op.in.c / op.in_slab_c - 1) * op.in_slab_step * chunk_ * sizeof(__half) : 0);
    // the kernels address activations through 32-bit buffer offsets; the constructor sized chunk_ so that
    // every view fits, this is the guard behind it (computed in 64 bits BEFORE it is narrowed)
    if (in_bytes > kMaxViewBytes)
        fail(RMR_ERR_CAPACITY, "conv %d: an input view of %zu bytes exceeds the 32-bit addressing of the conv kernels", op.conv, in_bytes);
    a.in_bytes = (unsigned)in_bytes;
    a.wt_bytes = (unsigned)((size_t)cw.cout_pad * cw.Kp * sizeof(__half));
    if (cw.w32.p) {
        a.wt_t32 = cw.w32.p;
        a.wt_t32_bytes = (unsigned)(cw.w32.n * sizeof(__half));
    }
    if (cw.w1d.p) {
        a.wt_w1d = cw.w1d.p;
        a.wt_w1d_bytes = (unsigned)(cw.w1d.n * sizeof(__half));
    }
    if (op.fp8) {
        const size_t q_bytes = (size_t)n * a.H * a.W * op.q_pitch;
        if (q_bytes > kMaxViewBytes) fail(RMR_ERR_CAPACITY, "conv %d: the e4m3 input view exceeds 32-bit addressing", op.conv);
        a.in8 = arena8_.p + op.q_off * chunk_;
        a.in8_cs = op.q_pitch;
        a.in8_bytes = (unsigned)q_bytes;
        a.wt8 = cw.w8.p;
        a.wt8_bytes = (unsigned)cw.w8.n;
        a.wscale = cw.wscale.p;
        if (op.q_out) {
            a.out8 = arena8_.p + op.q_out_off * chunk_;
            a.out8_cs = op.q_out_pitch;
            a.out8_only = op.q_only ? 1 : 0;
        }
    }
    a.flops = 2.0 * a.M * (double)cw.cout * (op.in_is_input ? 3 : cw.cin) * cw.k * cw.k;
    return a;
}

// the fused bottleneck that starts at op_index: x in (= the shortcut), y out, both filters; FLOPs of both convolutions
ConvArgs Yolov8::fused_args(int op_index, int n, size_t img0) {
    const Op& op = ops_[op_index];
    if (op.fuse_with < 0) fail(RMR_ERR_LOGIC, "layer %d is not the first convolution of a fusable bottleneck", op_index);
    ConvArgs f = conv_args(op_index, n, img0);
    const ConvArgs b = conv_args(op.fuse_with, n, img0);
    f.wt2 = b.wt;
    f.bias2 = b.bias;
    f.out = b.out;
    f.out_cs = b.out_cs;
    f.out_co = b.out_co;
    f.res = nullptr;
    f.flops += b.flops;
    return f;
}

void Yolov8::run_op(hipStream_t s, int op_index, int n, size_t img0) {
    const Op& op = ops_[op_index];
    auto hptr = [&](const View& v) { return arena_.p + v.off * chunk_; };
    auto fptr = [&](const View& v) { return arena32_.p + v.off * chunk_; };
    switch (op.kind) {
        case OP_CONV: {
            const ConvArgs a = conv_args(op_index, n, img0);
            if (op.in_is_input && lb_src_) {
                launch_conv_stem_letterbox(ctx_, s, a, lb_src_ + img0, lb_fill_, lb_scale_);
                break;
            }
            if (!autotune_) {
                if (a.in8) {  // fp8 plan without tuning: the first e4m3 tile that fits (the planner checked that one does)
                    launch_conv_t32f8(ctx_, s, a, conv_t32f8_first_tile(a.Cout_pad, a.W));
                } else if (a.in_slab_c || a.out_slab_c) {
                    int v = 0;
                    while (!conv_pw_supported(a, v)) ++v;  // the planner checked that one exists
                    launch_conv_pw(ctx_, s, a, v);
                } else {
                    launch_conv_auto(ctx_, s, a);
                }
                break;
            }
            if (op.group >= 0) {
                const std::vector<int>& members = groups_[op.group];
                if (!tuned_.count({op_index, n}) && !pinned_ && members.front() == op_index) tune_group(s, op.group, n, img0);
                const auto gi = tuned_.find({op_index, n});
                if (gi != tuned_.end() && gi->second == kGroupedAway) break;   // done by the launch of the group's first layer
                if (gi != tuned_.end() && gi->second >= kSbGroupBase) {
                    const auto tb = group_tables_.find({op_index, n});
                    if (tb == group_tables_.end()) fail(RMR_ERR_LOGIC, "grouped launch of layer %d at %d images has no problem table", op_index, n);
                    const std::vector<ConvArgs> args = group_args(op.group, n);
                    launch_conv_sb_group(ctx_, s, args.data(), (int)args.size(), tb->second.p, gi->second - kSbGroupBase);
                    break;
                }
            }
            auto key = std::make_pair(op_index, n);
            auto it = tuned_.find(key);
            if (it == tuned_.end() && conv_stem_supported(a)) {
                // the first layer has one kernel (tune_conv says so without timing anything): a pinned plan need not name it, so the
                // separate-letterbox paths (RMR_FUSE_LB=0) run under the committed plans too
                it = tuned_.emplace(key, 500).first;
            }
            if (it == tuned_.end()) {
                if (pinned_)
                    fail(RMR_ERR_RUNTIME, "pinned plan '%s' has no kernel for layer %d at %d images (RMR_PLAN names a file written for this pack, input size and batch sizes)",
                         tune_path_.c_str(), op_index, n);
                float ms = 0.f;
                it = tuned_.emplace(key, tune_conv(s, a, &ms)).first;
                tuned_dirty_ = true;
                if (op.fuse_with >= 0) tuned_ms_[key] = ms;
                // the second convolution of a fusable bottleneck: both are tuned now and both have run in this pass (the
                // hidden tensor and the output are valid), so the fused launch can be timed against their sum -- it rewrites
                // the same output bits.  Chip-filling batches only.
                const int first = op_index > 0 && ops_[op_index - 1].kind == OP_CONV && ops_[op_index - 1].fuse_with == op_index ? op_index - 1 : -1;
                const auto fk = std::make_pair(first, n);
                // RMR_FUSE_WS=1 only: in isolation the fused launch beats the two by 4-9 % (790 against 867 us at 256 images), inside
                // the network it does not (the second launch finds part of the hidden tensor in the Infinity Cache: 1.42 ms for
                // the four launches of model.2 against 1.56 ms for the two fused ones), so the run-off here is not trusted by
                // default; tools/make_plan.py decides it in the network and writes the result into the committed plan
                static const bool fuse_tune = std::getenv("RMR_FUSE_WS") && std::atoi(std::getenv("RMR_FUSE_WS")) != 0;
                if (fuse_tune && first >= 0 && n >= 16 && tuned_ms_.count(fk) && tuned_.count(fk) && tuned_[fk] < 340) {
                    launch_choice(s, a, it->second);   // this pass's own output first
                    const ConvArgs f = fused_args(first, n, img0);
                    const float pair_ms = tuned_ms_[fk] + ms;
                    float best_f = 1e30f;
                    int best_v = -1;
                    hipEvent_t e0, e1;
                    RMR_HIP(hipEventCreate(&e0));
                    RMR_HIP(hipEventCreate(&e1));
                    const int prof_was_on = ctx_.prof.on;
                    ctx_.prof.on = 0;
                    for (int v = 0; v < conv_wsf_num_variants(); ++v) {
                        if (!conv_wsf_supported(f, v)) continue;
                        float v_ms = 1e30f;
                        for (int rep = 0; rep < 3; ++rep) {
                            RMR_HIP(hipEventRecord(e0, s));
                            for (int k = 0; k < 3; ++k) launch_conv_wsf(ctx_, s, f, v);
                            RMR_HIP(hipEventRecord(e1, s));
                            RMR_HIP(hipEventSynchronize(e1));
                            float t = 0;
                            RMR_HIP(hipEventElapsedTime(&t, e0, e1));
                            if (rep > 0) v_ms = std::min(v_ms, t / 3);
                        }
                        if (v_ms < best_f) best_f = v_ms, best_v = v;
                    }
                    ctx_.prof.on = prof_was_on;
                    (void)hipEventDestroy(e0);
                    (void)hipEventDestroy(e1);
                    static const bool verbose = std::getenv("RMR_TUNE_VERBOSE") != nullptr;
                    if (verbose)
                        fprintf(stderr, "fuse layers %d + %d at %d images: two launches %.1f us, conv_wsf variant %d %.1f us -> %s\n", first, op_index, n,
                                pair_ms * 1e3f, best_v, best_f * 1e3f, best_v >= 0 && best_f < pair_ms ? "fused" : "two launches");
                    if (best_v >= 0 && best_f < pair_ms) {
                        tuned_[fk] = 340 + best_v;
                        it->second = kFusedAway;
                    }
                    break;
                }
            }
            if (it->second == kFusedAway) break;   // done by the launch of the layer before
            if (it->second >= 340 && it->second < kFusedAway) {
                launch_conv_wsf(ctx_, s, fused_args(op_index, n, img0), it->second - 340);
                break;
            }
            launch_choice(s, a, it->second);
            break;
        }
        case OP_QUANT:
            launch_quant_f8(ctx_, s, hptr(op.in), op.in.cs, op.in.co, op.in.c, arena8_.p + op.q_off * chunk_, op.q_pitch,
                            (long)n * op.in.h * op.in.w);
            break;
        case OP_SPPF:
            launch_sppf_pools(ctx_, s, hptr(op.in), n, op.in.h, op.in.w, op.in.cs, op.in.co, op.in.c);
            break;
        case OP_UP:
            launch_upsample2x(ctx_, s, hptr(op.in), op.in.cs, op.in.co, hptr(op.out), op.out.cs, op.out.co, n,
                              op.in.h, op.in.w, op.in.c);
            break;
        case OP_HEAD: {
            // consecutive scales leave in one launch.  ONE rule decides both who launches and what the launch covers: walk
            // the stretch of consecutive OP_HEADs from its start and cut it into runs of up to three scales with the
            // leader's class pitch; the leader of a run decodes the run, its other members have nothing left to do.
            int b = op_index;
            while (b > 0 && ops_[b - 1].kind == OP_HEAD) --b;
            int lead = b, len = 0;
            for (int i = b; i <= op_index; ++i) {
                if (len == 3 || ops_[i].cls.cs != ops_[lead].cls.cs) lead = i, len = 0;
                ++len;
            }
            if (lead != op_index && op.box_conv < 0) break;
            if (op.box_conv >= 0) {
                // fused form: the first OP_HEAD of the stretch launches for all its scales (same class-branch width by construction)
                if (op_index != b) break;
                HeadFusedScale sc[3];
                int k = 0;
                for (int i = op_index; i < (int)ops_.size() && k < 3 && ops_[i].kind == OP_HEAD && ops_[i].box_conv >= 0; ++i, ++k) {
                    const Op& o = ops_[i];
                    const ConvW &wb = convs_[o.box_conv], &wc = convs_[o.cls_conv];
                    sc[k] = HeadFusedScale{hptr(o.hb), hptr(o.hc), wb.w.p, wc.w.p, wb.b.p, wc.b.p, o.in.h, o.in.w, o.head_stride, o.a_off,
                                           o.hb.cs, o.hb.co, o.hc.cs, o.hc.co, wb.Kp, wc.Kp, wc.cin};
                }
                launch_head_fused(ctx_, s, k, sc, nc_, output_.p + img0 * (size_t)(4 + nc_) * anchors_, n, anchors_);
                break;
            }
            const float *box[3], *cls[3];
            int H[3], W[3], st[3], off[3], k = 0;
            for (int i = op_index; i < (int)ops_.size() && k < 3 && ops_[i].kind == OP_HEAD && ops_[i].cls.cs == op.cls.cs; ++i, ++k) {
                box[k] = fptr(ops_[i].box), cls[k] = fptr(ops_[i].cls);
                H[k] = ops_[i].in.h, W[k] = ops_[i].in.w, st[k] = ops_[i].head_stride, off[k] = ops_[i].a_off;
            }
            launch_head_decode3(ctx_, s, k, box, cls, op.cls.cs, nc_, output_.p + img0 * (size_t)(4 + nc_) * anchors_, n, H, W, st, off, anchors_);
            break;
        }
    }
}

bool Yolov8::read_feature(hipStream_t s, const std::string& name, int img, float* out, int dims[3]) {
    const auto it = named_.find(name);
    if (it == named_.end()) return false;
    const View& v = it->second.v;
    dims[0] = v.h, dims[1] = v.w, dims[2] = v.c;
    if (!out) return true;
    if (img < 0 || img >= chunk_) fail(RMR_ERR_INVALID_ARGUMENT, "read_feature: image %d is outside the last chunk", img);
    if (arena_reuse_)
        fail(RMR_ERR_LOGIC, "read_feature: stage outputs are overwritten by later layers when the arena is compacted; "
                            "create the detector with RMR_ARENA_REUSE=0 in the environment");
    // stage outputs are interleaved NHWC views (pixel pitch cs, first channel co)
    const size_t px = (size_t)v.h * v.w;
    std::vector<__half> host(px * v.cs);
    RMR_HIP(hipMemcpyAsync(host.data(), arena_.p + v.off * chunk_ + (size_t)img * px * v.cs, host.size() * sizeof(__half),
                           hipMemcpyDeviceToHost, s));
    RMR_HIP(hipStreamSynchronize(s));
    for (size_t p = 0; p < px; ++p)
        for (int c = 0; c < v.c; ++c) out[p * v.c + c] = __half2float(host[p * v.cs + v.co + c]);
    return true;
}

const __half* Yolov8::stage_rows(const std::string& name, int img, int dims[3], int64_t& ld) {
    const auto it = named_.find(name);
    if (it == named_.end()) return nullptr;
    const View& v = it->second.v;
    dims[0] = v.h, dims[1] = v.w, dims[2] = v.c;
    if (img < 0 || img >= chunk_) fail(RMR_ERR_INVALID_ARGUMENT, "stage %s: image %d is outside the last chunk", name.c_str(), img);
    if (arena_reuse_)
        fail(RMR_ERR_LOGIC, "stage outputs are overwritten by later layers when the arena is compacted; "
                            "create the detector with RMR_ARENA_REUSE=0 in the environment");
    ld = v.cs;
    return arena_.p + v.off * chunk_ + (size_t)img * v.h * v.w * v.cs + v.co;
}

Yolov8::~Yolov8() {
    for (auto& kv : graphs_) {
        if (kv.second.exec) (void)hipGraphExecDestroy(kv.second.exec);
        if (kv.second.graph) (void)hipGraphDestroy(kv.second.graph);
    }
}

bool Yolov8::all_tuned(int n) const {
    for (int i = 0; i < (int)ops_.size(); ++i)
        if (ops_[i].kind == OP_CONV && autotune_ && !(ops_[i].in_is_input && lb_src_) && !tuned_.count({i, n})) return false;
    return true;
}

void Yolov8::forward(hipStream_t s, int batch, const LetterboxDesc* src, int fill, float scale) {
    if (!src) fail(RMR_ERR_INVALID_ARGUMENT, "forward: no letterbox descriptors");
    if (batch <= 0) return;
    bool fused = fuse_lb_ && !ops_.empty() && ops_[0].kind == OP_CONV && ops_[0].in_is_input;
    if (fused) {
        const ConvArgs a = conv_args(0, 1, 0);
        fused = conv_stem_supported(a) && !a.out32;
    }
    if (!fused) {
        launch_letterbox(ctx_, s, src, batch, in_w_, in_h_, fill, scale, LB_F16_NHWC8, input_.p);
        forward(s, batch);
        return;
    }
    struct Reset {
        const LetterboxDesc*& p;
        ~Reset() { p = nullptr; }
    } reset{lb_src_};
    lb_src_ = src;
    lb_fill_ = fill;
    lb_scale_ = scale;
    forward(s, batch);
}

void Yolov8::forward(hipStream_t s, int batch) {
    if (batch < 0 || batch > max_batch_) fail(RMR_ERR_CAPACITY, "forward: batch %d exceeds max_batch_size %d", batch, max_batch_);
    // graph replay: one chunk, every layer tuned (tuning synchronises), no per-kernel events
    if (batch > 0 && batch <= graph_max_batch_ && batch <= chunk_ && !ctx_.prof.on && all_tuned(batch)) {
        auto it = graphs_.find(batch);
        if (it != graphs_.end() && it->second.src != lb_src_) {  // captured with another source array
            (void)hipGraphExecDestroy(it->second.exec);
            (void)hipGraphDestroy(it->second.graph);
            graphs_.erase(it);
            it = graphs_.end();
        }
        if (it == graphs_.end()) {
            Graph g;
            g.src = lb_src_;
            RMR_HIP(hipStreamBeginCapture(s, hipStreamCaptureModeThreadLocal));
            try {
                for (int i = 0; i < (int)ops_.size(); ++i) run_op(s, i, batch, 0);
            } catch (...) {
                hipGraph_t dead = nullptr;
                (void)hipStreamEndCapture(s, &dead);
                if (dead) (void)hipGraphDestroy(dead);
                throw;
            }
            RMR_HIP(hipStreamEndCapture(s, &g.graph));
            RMR_HIP(hipGraphInstantiate(&g.exec, g.graph, nullptr, nullptr, 0));
            it = graphs_.emplace(batch, g).first;
        }
        RMR_HIP(hipGraphLaunch(it->second.exec, s));
        return;
    }
    for (int c0 = 0; c0 < batch; c0 += chunk_) {
        const int n = std::min(chunk_, batch - c0);
        for (int i = 0; i < (int)ops_.size(); ++i) run_op(s, i, n, (size_t)c0);
    }
    if (tuned_dirty_) {
        save_tuning();
        tuned_dirty_ = false;
    }
}

}  // namespace rmr
