"""The operators of a serving step in a row: norm and quantisation, 8-bit QKV, append, attention over a shared prefix, 8-bit
output and feed-forward projections with their residuals, head, filtered sampling.  Every step is held to its own
definition on the inputs that the step before produced (the bounds stand beside those checks), for several layers and
tokens on one workspace; then the whole step is captured and replayed.  And the same calls through the C++ mirror."""
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parent.parent
PKG = ROOT / "qingming-qwen3-tts_b200"
BINARY = ROOT / "tests" / "cpp" / "serving_step_test.bin"


def build_binary(qm):
    qm.build_library()
    cmd = ["nvcc", "-std=c++17", "-O2", "-I", str(ROOT / "include"), "-I", str(PKG / "host"),
           str(ROOT / "tests" / "cpp" / "serving_step_test.cpp"), "-o", str(BINARY), "-L", str(PKG / "lib"), "-lqm_attention_b200",
           "-Xlinker", f"-rpath={PKG / 'lib'}"]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    assert proc.returncode == 0, proc.stdout + proc.stderr


def test_the_mirror_compiles(qm):
    build_binary(qm)


@pytest.mark.gpu
def test_the_mirror_runs(qm):
    if not BINARY.exists():
        build_binary(qm)
    proc = subprocess.run([str(BINARY)], capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0, proc.stdout + proc.stderr
    assert "SERVING_STEP_OK" in proc.stdout


@pytest.mark.gpu
def test_layers_and_tokens_in_a_row(qm):
    import torch
    from tests.test_int8_gpu import check_linear, numbers
    from tests.test_sample_filtered_gpu import want as want_token
    from tests.test_shared_prefix_gpu import Case

    layers, kv, hidden, inner, vocab = 2, 2, 256, 512, 1000
    c = Case(qm, [(5, 3), (3, 1)], [30, 62, 5, 100, -70], kv_heads=kv, layers=layers, seed=20, loose_back=1, spare=6)
    eng, batch = c.eng, c.q.shape[0]
    pools = [eng.pool_view(i) for i in range(layers)]
    for i, (k, v) in enumerate(pools):
        k.copy_(numbers(100 + i, *k.shape))
        v.copy_(numbers(200 + i, *v.shape))
    # room for the tokens to come
    used = set(int(p) for p in c.table.flatten().tolist())
    free = [p for p in range(eng.num_pages) if p not in used]

    def packed(seed, rows, cols):
        return eng.quantize_rows_int8(numbers(seed, rows, cols, scale=cols ** -0.5))

    weights = [{"norm": numbers(10 * i + 1, hidden, scale=0.1) + 1, "post": numbers(10 * i + 2, hidden, scale=0.1) + 1,
                "qk": torch.ones(128, dtype=torch.bfloat16, device="cuda"),
                "q": packed(1000 + i, 2 * kv * 128, hidden), "k": packed(1010 + i, kv * 128, hidden), "v": packed(1020 + i, kv * 128, hidden),
                "o": packed(1030 + i, hidden, 2 * kv * 128), "gate": packed(1040 + i, inner, hidden), "up": packed(1050 + i, inner, hidden),
                "down": packed(1060 + i, hidden, inner)} for i in range(layers)]
    final, head = numbers(5, hidden, scale=0.1) + 1, packed(1070, vocab, hidden)
    embed = numbers(6, vocab, hidden)
    lens = c.seq.clone()
    position, cache = torch.zeros_like(lens), torch.zeros_like(lens)
    tokens = torch.zeros(batch, dtype=torch.int32, device="cuda")
    uniforms = torch.zeros(batch, device="cuda")
    heat = torch.tensor(([0.9, 0.0, 1.3] * batch)[:batch], device="cuda")
    top_k = torch.tensor(([0, 7, 50] * batch)[:batch], dtype=torch.int32, device="cuda")
    top_p = torch.full((batch,), 0.9, device="cuda")
    logits = torch.zeros((batch, vocab), dtype=torch.bfloat16, device="cuda")
    q_rot = torch.zeros((batch, 2 * kv, 128), dtype=torch.bfloat16, device="cuda")
    eng.rope_cos.fill_(1)          # positions do not matter here: no rotation, so that the cache holds the normed keys
    eng.rope_sin.fill_(0)

    def step(check):
        x = last = eng.embedding_gather(embed, tokens)
        for i, w in enumerate(weights):
            xq, xs = eng.quantize_rows_int8(x, w["norm"])
            q, k, v = eng.qkv_linear_int8(xq, xs, *w["q"], *w["k"], *w["v"])
            if check:
                for got, name in ((q, "q"), (k, "k"), (v, "v")):
                    check_linear(got, xq, xs, *w[name])
            eng.launch_qk_norm_rope_cache_m1_sliced(i, q.view(batch, 2 * kv, 128), k.view(batch, kv, 128), v.view(batch, kv, 128), w["qk"],
                                                    w["qk"], position, cache, c.table, q_rot)
            context = eng.launch_attention_shared(i, q_rot, lens, c.table, c.starts, c.pages, c.most)
            if check:
                c.k, c.v = pools[i]
                c.check(context, lens.tolist(), q_rot)
            cq, cs = eng.quantize_rows_int8(context.view(batch, -1))
            attended = eng.linear_int8(cq, cs, *w["o"], residual=x)
            pq, ps = eng.quantize_rows_int8(attended, w["post"])
            act = eng.gate_up_swiglu_int8(pq, ps, *w["gate"], *w["up"])
            aq, as_ = eng.quantize_rows_int8(act)
            x = eng.linear_int8(aq, as_, *w["down"], residual=attended)
            if check:
                check_linear(attended, cq, cs, *w["o"], residual=last)
                check_linear(x, aq, as_, *w["down"], residual=attended)
            last = x
        hq, hs = eng.quantize_rows_int8(x, final)
        eng.linear_int8(hq, hs, *head, out=logits)
        eng.sample_filtered(logits, uniforms, heat, top_k, top_p, tokens=tokens)

    def advance(n):
        """The next token of every stream that is not idle (a page boundary is crossed on the way)."""
        lens.add_((lens > 0).int())
        cache.copy_(lens - 1)                       # -1 for an idle stream: nothing is written
        for s, length in enumerate(lens.tolist()):
            page = (length - 1) // 64
            if length and int(c.table[s, page]) >= 10 ** 6:
                c.table[s, page] = free.pop()
        uniforms.copy_(torch.tensor(np.random.default_rng(n).random(batch, dtype=np.float32)))

    for n in range(4):
        advance(n)
        step(check=True)
        z = logits.double().cpu().numpy()
        for s in range(batch):
            token, _ = want_token(z[s], float(uniforms[s]), float(heat[s]), int(top_k[s]), float(np.float32(0.9)))
            assert int(tokens[s]) == token
    assert eng.status() == 0
    # captured: the same step, replayed on the next token, equals the step called kernel by kernel
    advance(4)
    before = tokens.clone()
    snapshot = [(k.clone(), v.clone()) for k, v in pools]
    step(check=False)
    want_tokens, want_logits = tokens.clone(), logits.clone()
    for (k, v), (k0, v0) in zip(pools, snapshot):
        k.copy_(k0)
        v.copy_(v0)
    tokens.copy_(before)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(check=False)
    for _ in range(3):
        tokens.copy_(before)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tokens, want_tokens) and torch.equal(logits, want_logits)
    assert eng.status() == 0
    eng.close()
