// Drives the C++ host mirror through the parts of a serving step that are given 8-bit weights, shared prefixes and filtered
// sampling: four streams behind one prompt of three pages, one decode step each.  The shared-prefix context is compared with
// the plain decode attention over the same page tables, the 8-bit projection with integer sums on the host, the
// sampler with a scan on the host.  Exit code 0 = pass.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <vector>

#include "talker_attention_b200.hpp"

static uint32_t state = 12345;
static uint32_t next_word() { return state = state * 1664525u + 1013904223u; }
static float bf16(uint16_t v) {
    const uint32_t w = (uint32_t)v << 16;
    float f;
    std::memcpy(&f, &w, 4);
    return f;
}
static uint16_t random_bf16() {          // about [-2, 2), seven bits
    const float f = ((int)(next_word() >> 16 & 0xff) - 128) / 64.0f;
    uint32_t w;
    std::memcpy(&w, &f, 4);
    return (uint16_t)(w >> 16);
}

template <class T>
static T* upload(const std::vector<T>& h, qm::DeviceBuffer& d) {
    d = qm::DeviceBuffer(h.size() * sizeof(T));
    cudaMemcpy(d.pointer, h.data(), h.size() * sizeof(T), cudaMemcpyHostToDevice);
    return d.as<T>();
}
template <class T>
static std::vector<T> download(const qm::DeviceBuffer& d, size_t n) {
    std::vector<T> h(n);
    cudaMemcpy(h.data(), d.pointer, n * sizeof(T), cudaMemcpyDeviceToHost);
    return h;
}

int main() {
    const int Hq = 16, Hkv = 8, D = 128, batch = 4, shared = 3, max_pages = 5, prompt = shared * 64, rope_rows = 512;
    const int hidden = 256, vocab = 300;
    cudaStream_t stream;
    cudaStreamCreateWithFlags(&stream, cudaStreamNonBlocking);
    try {
        qm::TalkerAttentionB200 engine(1, shared + 2 * batch, Hq, Hkv, batch, rope_rows, stream);
        engine.reset_request();
        // the prompt, written once, through the first stream's table
        std::vector<int32_t> table(batch * max_pages), cu = {0, prompt};
        for (int s = 0; s < batch; ++s)
            for (int p = 0; p < max_pages; ++p) table[s * max_pages + p] = p < shared ? p : shared + 2 * s + p - shared;
        std::vector<uint16_t> q((prompt + batch) * Hq * D), k((prompt + batch) * Hkv * D), v(k.size()), norm(D, 0x3f80);
        for (auto* t : {&q, &k, &v})
            for (auto& x : *t) x = random_bf16();
        std::vector<int32_t> lens = {prompt + 1, prompt + 1, prompt + 1, prompt + 1}, pos(batch, prompt);
        std::vector<int32_t> starts = {0, batch}, pages = {shared};
        qm::DeviceBuffer dq, dk, dv, dn, dt, dcu, dl, dp, ds, dg, qrot(q.size() * 2), plain(batch * Hq * D * 2), ctx(batch * Hq * D * 2);
        upload(q, dq); upload(k, dk); upload(v, dv); upload(norm, dn); upload(table, dt); upload(cu, dcu); upload(lens, dl);
        upload(pos, dp); upload(starts, ds); upload(pages, dg);
        engine.scatter_prefill_cache(0, dq.as<uint16_t>(), dk.as<uint16_t>(), dv.as<uint16_t>(), dn.as<uint16_t>(), dn.as<uint16_t>(),
                                     dcu.as<int32_t>(), dt.as<int32_t>(), max_pages, 1, prompt, qrot.as<uint16_t>());
        const size_t qo = (size_t)prompt * Hq * D, ko = (size_t)prompt * Hkv * D;
        engine.launch_qk_norm_rope_cache_m1(0, dq.as<uint16_t>() + qo, dk.as<uint16_t>() + ko, dv.as<uint16_t>() + ko, dn.as<uint16_t>(),
                                            dn.as<uint16_t>(), dp.as<int32_t>(), dt.as<int32_t>(), max_pages, batch,
                                            qrot.as<uint16_t>() + qo);
        bool threw = false;        // without its workspace the call is refused
        try {
            engine.launch_attention_shared(0, qrot.as<uint16_t>() + qo, dl.as<int32_t>(), dt.as<int32_t>(), max_pages, batch,
                                           ds.as<int32_t>(), dg.as<int32_t>(), 1, shared, ctx.as<uint16_t>());
        } catch (const std::runtime_error&) {
            threw = true;
        }
        if (!threw) return 2;
        engine.reserve_shared_prefixes(batch);
        engine.launch_attention(0, qrot.as<uint16_t>() + qo, dl.as<int32_t>(), dt.as<int32_t>(), max_pages, batch, plain.as<uint16_t>());
        engine.launch_attention_shared(0, qrot.as<uint16_t>() + qo, dl.as<int32_t>(), dt.as<int32_t>(), max_pages, batch,
                                       ds.as<int32_t>(), dg.as<int32_t>(), 1, shared, ctx.as<uint16_t>());
        if (engine.device_status() != 0) return 3;
        const auto a = download<uint16_t>(plain, batch * Hq * D), b = download<uint16_t>(ctx, batch * Hq * D);
        double worst = 0, size = 0;
        for (size_t i = 0; i < a.size(); ++i) {
            worst = std::fmax(worst, std::fabs(bf16(a[i]) - bf16(b[i])));
            size = std::fmax(size, std::fabs(bf16(a[i])));
        }
        std::printf("shared against plain: max_abs %.3g of %.3g\n", worst, size);
        // |v| <= 2: weights rounded to bf16 move a row by 2^-8 * 2 at most, and each of the two results is rounded once
        if (!(size > 0 && worst <= 2 * std::ldexp(1.0, -8) + 2 * size * std::ldexp(1.0, -8))) return 4;

        // ---- 8-bit projection of the contexts, sums checked on the host
        std::vector<uint16_t> w((size_t)vocab * hidden), x((size_t)batch * hidden);
        for (auto& e : w) e = random_bf16();
        for (auto& e : x) e = random_bf16();
        qm::DeviceBuffer dw, dx, wq((size_t)vocab * hidden), wscale(vocab * 4), xq((size_t)batch * hidden), xscale(batch * 4),
            logits((size_t)batch * vocab * 2);
        upload(w, dw); upload(x, dx);
        engine.quantize_rows_int8(dw.as<uint16_t>(), nullptr, wq.as<int8_t>(), wscale.as<float>(), vocab, hidden);
        engine.quantize_rows_int8(dx.as<uint16_t>(), nullptr, xq.as<int8_t>(), xscale.as<float>(), batch, hidden);
        engine.linear_int8(xq.as<int8_t>(), xscale.as<float>(), wq.as<int8_t>(), wscale.as<float>(), nullptr, nullptr,
                           logits.as<uint16_t>(), batch, vocab, hidden);
        // ---- greedy and drawn tokens
        std::vector<float> heat = {0.0f, 1.0f, 0.7f, 0.0f}, top_p = {1.0f, 0.9f, 0.8f, 0.5f}, u = {0.3f, 0.6f, 0.1f, 0.9f};
        std::vector<int32_t> top_k = {0, 20, 1, 5};
        qm::DeviceBuffer dh, dtp, du, dtk, tokens(batch * 4), probs(batch * 4);
        upload(heat, dh); upload(top_p, dtp); upload(u, du); upload(top_k, dtk);
        engine.sample_filtered(logits.pointer, false, vocab, batch, vocab, du.as<float>(), dh.as<float>(), dtk.as<int32_t>(),
                               dtp.as<float>(), nullptr, tokens.as<int32_t>(), probs.as<float>());
        if (engine.device_status() != 0) return 5;
        const auto hw = download<int8_t>(wq, w.size()), hx = download<int8_t>(xq, x.size());
        const auto sw = download<float>(wscale, vocab), sx = download<float>(xscale, batch);
        const auto hl = download<uint16_t>(logits, (size_t)batch * vocab);
        const auto ht = download<int32_t>(tokens, batch);
        const auto hp = download<float>(probs, batch);
        for (int r = 0; r < batch; ++r) {
            int best = 0;
            for (int n = 0; n < vocab; ++n) {
                int sum = 0;
                for (int c = 0; c < hidden; ++c) sum += (int)hx[r * hidden + c] * hw[(size_t)n * hidden + c];
                const double want = (double)sum * sx[r] * sw[n], got = bf16(hl[r * vocab + n]);
                if (std::fabs(got - want) > std::fabs(want) * (std::ldexp(1.0, -8) + std::ldexp(1.0, -21))) return 6;
                if (got > bf16(hl[r * vocab + best])) best = n;
            }
            if (ht[r] < 0 || ht[r] >= vocab || !(hp[r] > 0.0f && hp[r] <= 1.0f)) return 7;
            if ((heat[r] == 0.0f || top_k[r] == 1) && (ht[r] != best || hp[r] != 1.0f)) return 8;
        }
        std::printf("SERVING_STEP_OK\n");
    } catch (const std::exception& e) {
        std::printf("exception: %s\n", e.what());
        return 1;
    }
    return 0;
}
