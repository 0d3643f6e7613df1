"""What the paged operators' torch functions do beside the kernels."""
import os
import subprocess
import sys

import pytest

import modelc_b200 as mb

gpu = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@gpu
@pytest.mark.parametrize("wants", ["q", "k", "v"])
def test_gradients_are_refused_aloud(wants):
    """A result of inputs that want gradients says so when they are asked for;
    values and calls that want none are as ever."""
    import torch
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = {n: torch.randn(5, 2, 64, generator=g, device="cuda").half() for n in "qkv"}
    cos, sin = mb.rope_table(8, 64)
    pool = mb.kv4_pool(1, 2, 64)
    mb.kv4_append(pool, x["k"], x["v"], t(0, 1, 2, 3, 4))

    def calls():
        rope = mb.rope(x["q"], x["k"], t(0, 1, 2, 3, 4), cos, sin)
        return {"rope": rope[0], "rope of k": rope[1], "rope of q": mb.rope(x["q"], None, t(*[0] * 5), cos, sin)[0],
                "prompt_attention": mb.prompt_attention(x["q"], x["k"], x["v"], t(0, 5)),
                "kv4_attention": mb.kv4_attention(x["q"], pool, t(0).view(1, 1), t(5), t(0, 5))}

    plain = calls()
    assert not any(y.requires_grad for y in plain.values())
    x[wants].requires_grad_()
    mb.kv4_append(pool, x["k"], x["v"], t(0, 1, 2, 3, 4))
    reached = {"q": list(plain), "k": ["rope", "rope of k", "prompt_attention"], "v": ["prompt_attention"]}[wants]
    for name, y in calls().items():
        assert torch.equal(y.detach(), plain[name]) and y.requires_grad == (name in reached)
        if name in reached:
            with pytest.raises(NotImplementedError, match=name.split()[0]):
                y.float().sum().backward()
    with torch.no_grad():
        assert not any(y.requires_grad for y in calls().values())
    assert x[wants].grad is None


@pytest.mark.parametrize("theta,scaling", [
    (1e4, dict(kind="llama3", low_turns=4.0, high_turns=4.0)), (1e4, dict(kind="llama3", low_turns=5.0)),
    (1.0, dict(kind="yarn", factor=4.0)), (0.5, dict(kind="yarn", factor=4.0)),
    (1e4, dict(kind="yarn", factor=4.0, slow=0.0)), (1e4, dict(kind="yarn", factor=4.0, fast=-1.0)),
    (1e4, dict(kind="yarn", factor=4.0, slow=8.0, fast=2.0)), (1e4, dict(kind="linear", factor=float("nan"))),
    (float("nan"), dict(kind="none")), (float("inf"), dict(kind="none"))], ids=str)
def test_scalings_without_a_meaning_are_refused(theta, scaling):
    with pytest.raises(ValueError, match="must be|wanted"):
        mb.rope_frequencies(64, theta, mb.RopeScaling(**scaling))


def test_scalings_at_the_edge_of_their_meaning():
    assert mb.rope_frequencies(64, 1.0)[0] == [1.0] * 32
    f, _ = mb.rope_frequencies(64, 1e4, mb.RopeScaling("llama3", 8.0, low_turns=3.999, high_turns=4.0))
    assert all(a > b for a, b in zip(f, f[1:]))
    mb.rope_frequencies(64, 1e4, mb.RopeScaling("yarn", 4.0, slow=2.0, fast=2.0))


@pytest.mark.parametrize("use", ["mb.paged.PAGE == 64", "mb.rope_frequencies(8)[1] == 1.0",
                                 "mb.paged.rope is mb.rope", "not hasattr(mb, 'paged_attention')"])
def test_names_before_the_first_use(use):
    """Everything is there in a fresh interpreter, whichever is asked for first."""
    r = subprocess.run([sys.executable, "-c", f"import modelc_b200 as mb; assert {use}"], cwd=ROOT,
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-1000:]


@gpu
def test_lengths_of_one_axis_are_wanted():
    """More axes were read as if the first ran through them, none gave an IndexError."""
    import torch
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    x = torch.zeros(4, 2, 64, device="cuda", dtype=torch.float16)
    pool = mb.kv4_pool(3, 2, 64)
    for bad in (lambda: mb.paged_slots(i(2, 2), i(2, 2), i(2, 4), i(1), i(1), 4),
                lambda: mb.paged_slots(i(), i(), i(1, 4), i(1), i(1), 4),
                lambda: mb.paged_slots(i(2), i(2), i(2, 4), i(1, 3), i(1), 4),
                lambda: mb.kv4_attention(x, pool, i(2, 3), i(2, 2), i(3)),
                lambda: mb.kv4_attention(x, pool, i(1, 3), i(), i(2)),
                lambda: mb.prompt_attention(x, x, x, i(2, 2)), lambda: mb.prompt_attention(x, x, x, i()),
                lambda: mb.kv4_append(pool, x[0, 0, 0], x, i(4))):
        with pytest.raises(ValueError):
            bad()
