"""Host-side behaviour of the sequence-model operators: no CPU fallback, entry
points that check their arguments without launching."""

from __future__ import annotations

import pytest
import torch

import myelin_amd as myelin
from myelin_amd import _lib


def test_cpu_tensors_are_rejected():
    x = torch.zeros(3, 4)
    with pytest.raises(ValueError, match="ROCm device"):
        myelin.counter_dropout(x, 0.5, 0)
    with pytest.raises(ValueError, match="ROCm device"):
        myelin.token_log_probs(x, torch.zeros(3, dtype=torch.int64))


def test_log_probs_entry_points_validate():
    f = "myelin_token_log_probs"
    # logits, dtype, ld, targets, ignore, lp, entropy, lse, top_lp, top_tok, R, V, top, ws, bytes, stream
    ok = [16, 0, 10, None, -100, None, 16, 16, None, None, 4, 10, 0, None, 0, None]

    def bad(**kw):
        at = dict(logits=0, dtype=1, ld=2, targets=3, lp=5, entropy=6, top_lp=8, R=10, V=11, top=12, ws=13)
        args = list(ok)
        for k, v in kw.items():
            args[at[k]] = v
        return args

    for kw, message in ((dict(dtype=1), "unsupported dtype"), (dict(R=-1), "non-negative"), (dict(V=0), "V positive"),
                        (dict(V=2**31, ld=2**31), "below 2"), (dict(ld=9), "row stride"),
                        (dict(logits=None), "null pointer"), (dict(entropy=None), "null pointer"),
                        (dict(targets=16), "null pointer"), (dict(top=11), "top must be"),
                        (dict(top=3), "null pointer"), (dict(V=100000, ld=100000), "workspace of")):
        with pytest.raises(ValueError, match=message):
            _lib.call(f, *bad(**kw))
    assert _lib.load().myelin_token_log_probs(*bad(R=0)) == 0
    g = "myelin_token_log_probs_bwd"
    with pytest.raises(ValueError, match="null pointer"):
        _lib.call(g, 16, 0, 10, None, -100, None, 16, None, None, 16, 4, 10, None)
    with pytest.raises(ValueError, match="row stride"):
        _lib.call(g, 16, 0, 9, None, -100, 16, 16, None, None, 16, 4, 10, None)


def test_log_probs_workspace_is_for_split_rows_only():
    need = _lib.load().myelin_token_log_probs_workspace_bytes
    assert need(12800, 10, 0) == 0 and need(8192, 32768, 0) == 0
    assert need(1, 4096, 5) == 0  # one tile
    assert need(1, 100000, 0) == 25 * 16 and need(1, 100000, 20) == 25 * (16 + 160)


def test_dropout_entry_point_validates():
    f = "myelin_counter_dropout"
    with pytest.raises(ValueError, match="unsupported dtype"):
        _lib.call(f, 16, 5, None, 16, 1, 8, 0, 1.0, 0, 0, None, None)
    with pytest.raises(ValueError, match="negative size"):
        _lib.call(f, 16, 0, None, 16, 1, -8, 0, 1.0, 0, 0, None, None)
    with pytest.raises(ValueError, match="threshold must be"):
        _lib.call(f, 16, 0, None, 16, 1, 8, 2**32 + 1, 1.0, 0, 0, None, None)
    with pytest.raises(ValueError, match="null pointer"):
        _lib.call(f, 16, 0, None, None, 1, 8, 0, 1.0, 0, 0, None, None)
    assert _lib.load().myelin_counter_dropout(None, 0, None, None, 0, 8, 0, 1.0, 0, 0, None, None) == 0


def test_attention_rejects_cpu_tensors():
    q, d = torch.zeros(3, 2, 2, 4), torch.ones(2)
    with pytest.raises(ValueError, match="ROCm device"):
        myelin.decay_attention(q, q, q, d)
    with pytest.raises(ValueError, match="ROCm device"):
        myelin.decay_attention_step(q[0], q[0], q[0], d, torch.zeros(2, 2, 4, 4))


def test_attention_entry_points_validate():
    sizes = dict(T=4, B=2, H=4, Hk=2, Dk=8, Dv=8)

    def fwd(q=16, dtype=0, scale=1.0, **kw):
        z = {**sizes, **kw}
        _lib.call("myelin_decay_attention_fwd", q, 16, 16, dtype, 16, 16, None, None, 16, 16, *z.values(), scale, None,
                  0, None)

    for kw, message in ((dict(dtype=3), "unsupported dtype"), (dict(T=0), "positive"), (dict(B=-1), "positive"),
                        (dict(H=3), "multiple of Hk"), (dict(Dk=129), "Dk and Dv"), (dict(Dv=0), "Dk and Dv"),
                        (dict(scale=0.0), "not be zero"), (dict(scale=float("nan")), "not be zero"),
                        (dict(scale=float("inf")), "finite"), (dict(T=2**31), "too many"),
                        (dict(q=None), "null pointer")):
        with pytest.raises(ValueError, match=message):
            fwd(**kw)
    fwd(q=None, B=0)  # nothing to do
    bwd = ("myelin_decay_attention_bwd", 16, 16, 16, 16, 0, 16, 16, None, None, None, 16, 16, 16, None)
    with pytest.raises(ValueError, match="workspace of"):
        _lib.call(*bwd, *sizes.values(), 1.0, None, 0, None)
    step = ("myelin_decay_attention_step", 16, 16, 16, 0, 16, 16)
    with pytest.raises(ValueError, match="null pointer"):
        _lib.call(*step, None, 16, 16, 2, 4, 2, 8, 8, 1.0, None)
    with pytest.raises(ValueError, match="Dk and Dv"):
        _lib.call(*step, 16, 16, 16, 2, 4, 2, 8, 200, 1.0, None)


def test_more_rows_than_a_launch_has_are_refused():
    args = ("myelin_decay_attention_fwd", 16, 16, 16, 0, 16, 16, None, None, 16, 16)
    with pytest.raises(ValueError, match="too many rows"):
        _lib.call(*args, 1, 2**20 + 1, 2, 1, 8, 8, 1.0, None, 0, None)
    step = ("myelin_decay_attention_step", 16, 16, 16, 0, 16, 16, 16, 16, 16)
    with pytest.raises(ValueError, match="too many rows"):
        _lib.call(*step, 2**21 + 1, 1, 1, 8, 8, 1.0, None)
    # 2^34 elements are 2^24 workgroups of 4 a thread
    with pytest.raises(ValueError, match="too many elements"):
        _lib.call("myelin_counter_dropout", 16, 0, None, 16, 1, 2**34, 0, 1.0, 0, 0, None, None)


def test_attention_is_cut_for_the_workgroups_that_fit():
    """Segments' states in the workspace: one less than the workgroups that the 256
    CUs hold of a (b, h).  Two share the LDS of a CU in bf16 with keys past 64 and
    values up to 64, three with both up to 64 and in fp32, two of 8 waves."""

    def segments(dtype, Dk, Dv, heads):
        kt, vt = (64 if Dk <= 64 else 128), (128 if dtype and Dk > 64 and Dv > 64 else 64)
        n = _lib.load().myelin_decay_attention_workspace_elems(dtype, 3 * 2**18, 1, heads, heads, Dk, Dv, 0)
        assert n % (heads * kt * vt) == 0
        return n // (heads * kt * vt) + 1

    assert segments(2, 128, 64, 1) == 512 and segments(2, 64, 64, 1) == 768 and segments(2, 128, 128, 1) == 512
    assert segments(0, 64, 64, 1) == 768 and segments(0, 128, 64, 1) == 768
    assert segments(2, 128, 64, 4) == 128


def test_a_cast_module_keeps_its_decays():
    want = torch.tensor([0.75, 1 - 1 / 1024, 1.0])
    for cast in (lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.double(),
                 lambda m: m.to(torch.bfloat16).float()):
        model = cast(torch.nn.Sequential(myelin.DecayAttention([4.0, 1024.0, float("inf")]), torch.nn.Linear(2, 2)))
        assert torch.equal(model[0].decay, want) and "0.decay" in model.state_dict()
    assert model.to("meta")[0].decay.device.type == "meta"
    assert model.to(torch.bfloat16)[0].decay.dtype == torch.float32
