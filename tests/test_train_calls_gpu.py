"""How the layer and head ops are called: streams, layouts and forms of the
arguments beside those of tests/test_train_gpu.py."""
import pytest

import train_ref as R
from test_train_gpu import _rand

pytestmark = pytest.mark.gpu


def _ops(inl, torch, dev):
    """Every op as (call with stream=, bytes of its largest output)."""
    m, hidden, inner, vocab = 1024, 256, 512, 1024
    x, dy = _rand(torch, dev, (m, hidden), 1), _rand(torch, dev, (m, hidden), 2, 0.1)
    w = _rand(torch, dev, (hidden, hidden), 3, 1 / 16)
    gu, down = _rand(torch, dev, (2 * inner, hidden), 4, 1 / 16), _rand(torch, dev, (hidden, inner), 5, 1 / 16)
    wv = _rand(torch, dev, (vocab, hidden), 6, 1 / 16)
    t = torch.arange(m, device=dev, dtype=torch.int32)
    _, pre, h = inl.gated_ffn(x, gu, down, save=True)
    _, lse = inl.softmax_xent(x, wv, t)
    dl = torch.ones(m, device=dev)
    heads = x.view(m, 4, 64)
    return {
        "dense": (lambda s: inl.dense(x, w, act="silu", stream=s), 2 * m * hidden),
        "dense_bwd": (lambda s: inl.dense_bwd(dy, x, w, bias_grad=True, stream=s), 2 * m * hidden),
        "gated_ffn": (lambda s: inl.gated_ffn(x, gu, down, save=True, stream=s), 4 * m * inner),
        "gated_ffn_bwd": (lambda s: inl.gated_ffn_bwd(dy, x, gu, down, pre, h, stream=s), 2 * m * hidden),
        "softmax_xent": (lambda s: inl.softmax_xent(x, wv, t, stream=s), 4 * m),
        "softmax_xent_bwd": (lambda s: inl.softmax_xent_bwd(dl, lse, x, wv, t, stream=s), 2 * m * hidden),
        "norm_rope_qk_bwd": (lambda s: inl.norm_rope_qk_bwd(dy.view(m, 4, 64), heads, 2, stream=s), 2 * m * hidden),
    }


@pytest.mark.parametrize("op", ["dense", "dense_bwd", "gated_ffn", "gated_ffn_bwd", "softmax_xent", "softmax_xent_bwd",
                                "norm_rope_qk_bwd"])
def test_memory_of_a_call_on_another_stream(op, cuda, inl):
    """Blocks that were freed while work on the current stream still reads them are
    not taken by a call on another stream, which does not wait for that work."""
    import torch
    call, size = _ops(inl, torch, cuda)[op]
    flat = lambda out: [t for t in (out if isinstance(out, tuple) else (out,)) if t is not None]
    want = flat(call(None))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    a, b = (torch.randn(4096, 4096, device=cuda) for _ in range(2))
    blocks = [torch.full((n,), 7, dtype=torch.uint8, device=cuda) for n in (size, size, 1024, 4096, 1 << 20, 1 << 22, 1 << 24)]
    spans = [(t.data_ptr(), t.data_ptr() + t.numel()) for t in blocks]
    torch.cuda.synchronize()
    for _ in range(20):   # some milliseconds of work in front of the reads
        a = (a @ b).clamp_(-1, 1)
    seen = [t.clone() for t in blocks]
    del blocks
    got = flat(call(side))
    torch.cuda.synchronize()
    for t in got:
        assert not any(lo < t.data_ptr() + t.numel() * t.element_size() and t.data_ptr() < hi for lo, hi in spans)
    assert all((t == 7).all() for t in seen)
    assert all(torch.equal(u, v) for u, v in zip(got, want))
