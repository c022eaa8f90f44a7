"""A training step of an encoder layer, run as a program would: the residual norm with dropout, the
projections, the q/k prologue, packed attention, the gated feed-forward block, pooling, the contrastive
loss, and every gradient back to the layer's input; in bf16 and captured into a graph, against the
same step in float64.

Every tensor between two ops is bf16 (the residual stream, its gradient and weight gradients are f32). The bound is
by norms: a rounding to bf16 moves a tensor by at most u = 2^-8 of its norm, and the ops behind pass a
relative change on by a factor near one (products with matrices of independent entries, norms, a softmax
of scores of deviation one, which moves by the change of its scores): with a factor of 2 for what they
amplify, a result behind k roundings in series, each of two branches at most, is within 2 k u of its
norm. Forward and back the longest way has 24 (three per op that rounds its operands and its output)."""
import math

import pytest

import step_ref as S
import train_ref as R

pytestmark = pytest.mark.gpu

HIDDEN, HQ, HKV, HD, INNER, THETA, EPS, SCALE = 256, 4, 2, 64, 512, 1e4, 1e-6, 4.0
LENGTHS = [37, 1, 128, 65, 90]
DROP = 0.1


def _weights(torch, dev):
    g = torch.Generator(device=dev).manual_seed(5)
    r = lambda *s, std: (torch.randn(*s, generator=g, device=dev) * std).to(torch.bfloat16)
    norm = lambda n: (1 + 0.1 * torch.randn(n, generator=g, device=dev)).to(torch.bfloat16)
    return dict(n1=norm(HIDDEN), qkv=r((HQ + 2 * HKV) * HD, HIDDEN, std=HIDDEN ** -0.5), qn=norm(HD), kn=norm(HD),
                o=r(HIDDEN, HQ * HD, std=(HQ * HD) ** -0.5), n2=norm(HIDDEN), gu=r(2 * INNER, HIDDEN, std=HIDDEN ** -0.5),
                down=r(HIDDEN, INNER, std=INNER ** -0.5), n3=norm(HIDDEN), docs=r(24, HIDDEN, std=HIDDEN ** -0.5))


def _step(inl, torch, x, w, plan, cu_list, cu, pos, cos, sin, targets, rng):
    """The step with this package's ops; returns the loss and every gradient."""
    n = x.shape[0]
    bf = torch.bfloat16
    # forward
    a, h1 = inl.add_rms_norm(x, w["n1"], eps=EPS, dropout=DROP, rng=rng, tag=1, out_dtype=bf, sum_dtype=torch.float32)
    qkv = inl.dense(a, w["qkv"]).view(n, HQ + 2 * HKV, HD)
    qk = inl.norm_rope_qk(qkv[:, :HQ + HKV], HQ, pos, cos, sin, q_weight=w["qn"], k_weight=w["kn"], eps=EPS)
    v = qkv[:, HQ + HKV:]
    out = torch.empty(n, HQ, HD, dtype=bf, device=x.device)
    plan.run(qk[:, :HQ], qk[:, HQ:], v, out)
    att = inl.dense(out.view(n, HQ * HD), w["o"])
    b, h2 = inl.add_rms_norm(att, w["n2"], residual=h1, eps=EPS, dropout=DROP, rng=rng, tag=2, out_dtype=bf)
    f, pre, hh = inl.gated_ffn(b, w["gu"], w["down"], act="silu", save=True)
    _, h3 = inl.add_rms_norm(f, residual=h2, eps=EPS, dropout=DROP, rng=rng, tag=3, out_dtype=bf)
    pooled = inl.pool_last(h3, cu, weight=w["n3"].float(), eps=EPS)
    p16 = pooled.to(bf)
    loss, lse = inl.softmax_xent(p16, w["docs"], targets, scale=SCALE)
    # and back
    dl = torch.full_like(loss, 1.0 / len(LENGTHS))
    dp, ddocs, _ = inl.softmax_xent_bwd(dl, lse, p16, w["docs"], targets, scale=SCALE, dx_dtype=torch.float32,
                                        dw_dtype=torch.float32)
    dh3, dn3 = inl.pool_last_bwd(dp, h3, cu, w["n3"].float(), eps=EPS)
    # past the last addition: dropout's gradient alone (its norm has no reader here)
    df, dh2, _ = inl.add_rms_norm_bwd(torch.zeros_like(f), h3, dh=dh3, eps=EPS, dropout=DROP, rng=rng, tag=3, dx_dtype=bf)
    db, dgu, ddown = inl.gated_ffn_bwd(df, b, w["gu"], w["down"], pre, hh, act="silu", dw_dtype=torch.float32)
    datt, dh1, dn2 = inl.add_rms_norm_bwd(db, h2, w["n2"], dh=dh2, eps=EPS, dropout=DROP, rng=rng, tag=2, dx_dtype=bf)
    dout, do_w, _ = inl.dense_bwd(datt, out.view(n, HQ * HD), w["o"], dw_dtype=torch.float32)
    dqkv = torch.empty(n, HQ + 2 * HKV, HD, dtype=bf, device=x.device)
    inl.varlen_attention_bwd(dout.view(n, HQ, HD), qk[:, :HQ], qk[:, HQ:], v, out, cu_list, causal=True,
                             grads=(dqkv[:, :HQ], dqkv[:, HQ:HQ + HKV], dqkv[:, HQ + HKV:]))
    # (in place: the prologue's gradient reads each head before it writes it)
    _, dqn, dkn = inl.norm_rope_qk_bwd(dqkv[:, :HQ + HKV], qkv[:, :HQ + HKV], HQ, pos, cos, sin, q_weight=w["qn"],
                                       k_weight=w["kn"], eps=EPS, out=dqkv[:, :HQ + HKV])
    da, dqkv_w, _ = inl.dense_bwd(dqkv.view(n, -1), a, w["qkv"], dw_dtype=torch.float32)
    dx, _, dn1 = inl.add_rms_norm_bwd(da, h1, w["n1"], dh=dh1, eps=EPS, dropout=DROP, rng=rng, tag=1, dx_dtype=torch.float32)
    return dict(loss=loss, x=dx, n1=dn1, qkv=dqkv_w, qn=dqn, kn=dkn, o=do_w, n2=dn2, gu=dgu, down=ddown, n3=dn3, docs=ddocs)


def _reference(torch, x, w, pos, cos, sin, targets, seed, step):
    """The same step in float64, its gradients by torch's autograd."""
    n = x.shape[0]
    x = x.double().requires_grad_()
    w = {k: t.double().requires_grad_() for k, t in w.items()}
    drop = [S.factor(n, HIDDEN, DROP, seed, step, tag, x.device) for tag in (1, 2, 3)]
    rms = lambda t, wt: t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * wt
    c, s = cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None]
    turn = lambda t: torch.cat([t[..., :HD // 2] * c - t[..., HD // 2:] * s, t[..., HD // 2:] * c + t[..., :HD // 2] * s], -1)
    h1 = x * drop[0]
    qkv = (rms(h1, w["n1"]) @ w["qkv"].T).view(n, HQ + 2 * HKV, HD)
    q, k, v = turn(rms(qkv[:, :HQ], w["qn"])), turn(rms(qkv[:, HQ:HQ + HKV], w["kn"])), qkv[:, HQ + HKV:]
    outs, at = [], 0
    for t in LENGTHS:
        kk, vv = (y[at:at + t].transpose(0, 1).repeat_interleave(HQ // HKV, 0) for y in (k, v))
        z = q[at:at + t].transpose(0, 1) @ kk.transpose(1, 2) * HD ** -0.5
        z = z.masked_fill(torch.ones(t, t, dtype=torch.bool, device=x.device).triu(1), -math.inf)
        outs.append((torch.softmax(z, -1) @ vv).transpose(0, 1))
        at += t
    h2 = h1 + (torch.cat(outs).reshape(n, HQ * HD) @ w["o"].T) * drop[1]
    gate, up = (rms(h2, w["n2"]) @ w["gu"].T).split(INNER, 1)
    h3 = h2 + ((gate * torch.sigmoid(gate) * up) @ w["down"].T) * drop[2]
    last = torch.tensor([sum(LENGTHS[:i + 1]) - 1 for i in range(len(LENGTHS))], device=x.device)
    z = rms(h3[last], w["n3"])
    y = z / torch.sqrt((z * z).sum(1, keepdim=True) + 1e-12)
    loss = torch.nn.functional.cross_entropy(SCALE * y @ w["docs"].T, targets.long(), reduction="none")
    loss.mean().backward()
    return dict(loss=loss.detach(), x=x.grad, **{k: t.grad for k, t in w.items()})


def test_step(cuda, inl):
    import torch
    n = sum(LENGTHS)
    cu_list = [sum(LENGTHS[:i]) for i in range(len(LENGTHS) + 1)]
    # (the forward's schedule, uploaded once: what a captured step needs)
    plan = inl.AttnPlan(inl.make_attn_desc(cu_list, HQ, HKV, HD, causal=True, q_row_stride=(HQ + HKV) * HD,
                                           k_row_stride=(HQ + HKV) * HD, v_row_stride=(HQ + 2 * HKV) * HD))
    cu = torch.tensor(cu_list, dtype=torch.int32, device=cuda)
    pos = torch.from_numpy(inl.positions(cu_list)).to(cuda)
    cos, sin = (torch.from_numpy(t).to(cuda) for t in inl.rope_table(HD, THETA, max(LENGTHS)))
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn(n, HIDDEN, generator=g, device=cuda)
    w = _weights(torch, cuda)
    targets = torch.tensor([3, 0, 23, 7, 7], dtype=torch.int32, device=cuda)
    rng = torch.tensor([11, 4], device=cuda)
    got = _step(inl, torch, x, w, plan, cu_list, cu, pos, cos, sin, targets, rng)
    torch.cuda.synchronize()
    ref = _reference(torch, x, w, pos, cos, sin, targets, 11, 4)
    assert got.keys() == ref.keys()
    for name, want in ref.items():
        off = (got[name].double() - want).norm().item() / want.norm().item()
        print(f"{name}: {off:.2e}", flush=True)
        assert off <= 2 * 24 * 2.0 ** -8, name
        # and each by its direction, which a wrong sign, scale or mask would turn
        cosine = (got[name].double().flatten() @ want.flatten()).item() / (got[name].double().norm() * want.norm()).item()
        assert cosine > 0.995, (name, cosine)
    # captured, replayed with another step of the dropout and other inputs
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = _step(inl, torch, x, w, plan, cu_list, cu, pos, cos, sin, targets, rng)
    for i in range(3):
        rng[1] += 1
        x.mul_(0.9)
        want = _step(inl, torch, x, w, plan, cu_list, cu, pos, cos, sin, targets, rng)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name in want:
            assert torch.equal(kept[name], want[name]), (i, name)
