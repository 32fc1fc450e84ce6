"""Argument checks of the filtered sampler: every refusal comes back before any CUDA call."""
import pytest

P = 0x10000


def sample(qm, logits=P, fp32=1, stride=100, batch=2, vocab=100, uniforms=P, temperature=0, top_k=0, top_p=0, min_p=0, tokens=P, probs=0):
    return qm.load_library().qm_sample_filtered(logits, fp32, stride, batch, vocab, uniforms, temperature, top_k, top_p, min_p, tokens,
                                                probs, None)


@pytest.mark.parametrize("change,text", [
    ({"logits": None}, b"null"), ({"uniforms": None}, b"null"), ({"tokens": None}, b"null"), ({"batch": -1}, b"vocab"),
    ({"vocab": 0}, b"vocab"), ({"vocab": 262145, "stride": 262145}, b"vocab"), ({"stride": -1}, b"row_stride"),
    ({"logits": P + 2}, b"aligned"), ({"logits": P + 1, "fp32": 0}, b"aligned"), ({"uniforms": P + 1}, b"aligned"),
    ({"top_k": P + 2}, b"aligned"), ({"probs": P + 2}, b"aligned"), ({"tokens": P + 3}, b"aligned"),
])
def test_refusals(qm, change, text):
    assert sample(qm, **change) == qm.QM_EINVAL
    assert text in qm.load_library().qm_last_error_string()


def test_no_rows_is_no_work(qm):
    assert sample(qm, logits=None, uniforms=None, tokens=None, batch=0) == qm.QM_OK
