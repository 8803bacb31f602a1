"""The text side's operators where the framework uses them: on the tape (lookup, packed attention, clipping in one training
step of a text layer), in the ControlNet's class conditioning by table, and in train_step's clipping.

Bounds: activations and their gradients are bf16, so a tensor's gradient carries a relative error of a few 2^-9 per contraction:
rel-L2 2e-2 per tensor, as for the other ops of the tape."""
import math

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from _common import SCHED, TINY, TINY_CE, build_pair, rel_l2

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _mods():
    from ccnet_amd import ops, training
    return ops, training


def _layer(V, C, H, Hkv, d, seed, dev):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, k=1.0: nn.Parameter((torch.randn(*s, generator=g) * k).to(BF16).float().to(dev))  # noqa: E731
    return dict(tok=r(V, C, k=0.05), g1=nn.Parameter(torch.ones(C, device=dev) + 0.1 * torch.randn(C, generator=g).to(dev)), b1=r(C, k=0.1),
                wqkv=r((H + 2 * Hkv) * d, C, k=C ** -0.5), wo=r(C, H * d, k=(H * d) ** -0.5), bo=r(C, k=0.1))


def _reference(p, ids, lens, H, Hkv, d, scale, dy):
    """The layer in fp32 by autograd: x = scale tok[id]; x + o(attention(qkv(norm(x)))) per sequence."""
    x = p["tok"][ids] * scale
    C = x.shape[1]
    qkv = F.layer_norm(x, (C,), p["g1"], p["b1"]) @ p["wqkv"].t()
    outs, first = [], 0
    for n in lens:
        q, k, v = qkv[first:first + n].split([H * d, Hkv * d, Hkv * d], 1)
        q, k, v = (t.reshape(n, -1, d).transpose(0, 1) for t in (q, k, v))
        k, v = (t.repeat_interleave(H // Hkv, 0) for t in (k, v))
        s = (q @ k.transpose(1, 2).contiguous()) * d ** -0.5
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), -math.inf)
        outs.append((torch.softmax(s, -1) @ v).transpose(0, 1).reshape(n, H * d))
        first += n
    y = x + torch.cat(outs) @ p["wo"].t() + p["bo"]
    (y * dy).sum().backward()
    return y


@pytest.mark.parametrize("H,Hkv,d", [(2, 2, 64), (4, 1, 64), (2, 1, 128)])
def test_a_text_layer_trains_through_lookup_attention_and_clipping(cuda, H, Hkv, d):
    ops, tr = _mods()
    V, C, lens = 300, 128, (77, 5, 1, 130, 40)
    rows, scale = sum(lens), math.sqrt(C)
    p = _layer(V, C, H, Hkv, d, H + d, cuda)
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(0, V, (rows,), generator=g)
    ids[torch.rand(rows, generator=g) < 0.4] = V - 1  # the padding token of a batch of prompts
    ids = ids.to(cuda)
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=cuda)
    dy = (torch.randn(rows, C, generator=g) * 0.1).to(BF16).to(cuda)
    with torch.enable_grad():
        y_ref = _reference(p, ids, lens, H, Hkv, d, scale, dy.float())
    T = tr.Tape()
    x = T.embedding(ids, p["tok"].detach(), scale=scale, param=p["tok"])
    n1 = T.layernorm(x, p["g1"].detach(), p["b1"].detach(), params=(p["g1"], p["b1"]))
    wqkv, wo = p["wqkv"].detach().to(BF16), p["wo"].detach().to(BF16)
    qkv = T.linear(n1, wqkv, None, wqkv.shape[0], params=([(p["wqkv"], 0, wqkv.shape[0])], None))
    o = T.attention_packed(qkv, 0, qkv, H * d, (H + Hkv) * d, cu, H, Hkv, d, d ** -0.5)
    y = T.linear(o, wo, p["bo"].detach(), C, res1=x, params=([(p["wo"], 0, C)], [(p["bo"], 0, C)]))
    assert rel_l2(y.a.t, y_ref.detach()) <= 2e-2
    y.accumulate(dy)
    T.backward()
    assert set(T.grads) == set(p.values())
    for name, q in p.items():
        assert rel_l2(T.grads[q], q.grad) <= 2e-2, (name, rel_l2(T.grads[q], q.grad))
    grads = [T.grads[q] for q in p.values()]
    before = [t.double() for t in grads]
    norm = math.sqrt(sum(float(t.square().sum()) for t in before))
    got = ops.clip_grad_norm(grads, norm / 3)
    assert abs(float(got) - norm) <= 2.0 ** -23 * norm
    for t, b in zip(grads, before):
        assert ((t.double() - b * (norm / 3 / (norm + 1e-6))).abs() <= 2.0 ** -22 * b.abs()).all()


def test_packed_attention_of_equal_lengths_is_the_text_towers(cuda):
    """Prompts of one length, one key head a head, d 64: what ccnet_attention_d64_causal_bf16 computes, to the rounding of both."""
    ops, _ = _mods()
    B, S, H = 3, 77, 4
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(B * S, 3 * H * 64, generator=g).to(BF16).to(cuda)
    q, k, v = qkv.split(H * 64, 1)
    cu = torch.arange(B + 1, dtype=torch.int32, device=cuda) * S
    a = ops.attention_d64_causal(q, k, v, B, H, S, 64 ** -0.5).double()
    b = ops.attention_packed(q, k, v, cu, H, H, 64, 64 ** -0.5).double()
    # P is rounded to bf16 (2^-8 of each, relative to a maximum that either may set differently) and then the result: twice
    bound = 2 * 2.0 ** -8 * (ops.attention_d64_causal(q, k, v.abs(), B, H, S, 64 ** -0.5).double() + a.abs()) * (1 + 2.0 ** -6)
    assert ((a - b).abs() <= bound).all()


def test_tape_adds_where_lookups_or_projections_are_shared(cuda):
    """One table read twice, one projection attended to twice: the gradients are sums, also where a buffer holds one already."""
    _, tr = _mods()
    V, C, H, d, n = 50, 128, 1, 64, 90
    g = torch.Generator().manual_seed(3)
    tok = nn.Parameter(torch.randn(V, C, generator=g).to(cuda))
    ids = [torch.randint(0, V, (n,), generator=g).to(cuda) for _ in range(2)]
    dys = [torch.randn(n, C, generator=g).to(BF16).to(cuda) for _ in range(2)]
    T = tr.Tape()
    for i, dy in zip(ids, dys):
        T.embedding(i, tok.detach(), scale=2.0, param=tok).accumulate(dy)
    frozen = nn.Parameter(tok.detach().clone(), requires_grad=False)
    assert not T.embedding(ids[0], frozen.detach(), param=frozen).rg
    T.backward()
    want = torch.zeros(V, C, dtype=torch.float64, device=cuda)
    for i, dy in zip(ids, dys):
        want.index_add_(0, i, dy.double(), alpha=2.0)
    assert ((T.grads[tok].double() - want).abs() <= 1e-5 * (1 + want.abs())).all()

    qkv0 = torch.randn(n, 3 * d, generator=g).to(BF16).to(cuda)
    cu = torch.tensor([0, 40, 90], dtype=torch.int32, device=cuda)
    do = [torch.randn(n, d, generator=g).to(BF16).to(cuda) for _ in range(2)]

    def run(uses):
        T = tr.Tape()
        x = tr._v2d(qkv0, True)
        for k in uses:
            T.attention_packed(x, 0, x, d, 2 * d, cu, H, H, d, 0.125).accumulate(do[k])
        T.backward()
        return x.g.double()

    a, b, both = run([0]), run([1]), run([0, 1])
    assert ((both - (a + b)).abs() <= 2.0 ** -8 * (both.abs() + 2.0 ** -20)).all()  # one rounding of the sum
    T = tr.Tape()  # keys and values that take no gradient, queries apart from them
    q, kv = tr._v2d(qkv0[:, :d].contiguous(), True), tr._v2d(qkv0[:, d:].contiguous(), False)
    T.attention_packed(q, 0, kv, 0, d, cu, H, H, d, 0.125).accumulate(do[0])
    T.backward()
    assert kv.g is None and torch.equal(q.g.double(), a[:, :d])


def test_class_table_training_against_oracle_autograd(cuda):
    """Class conditioning by nn.Embedding (num_class_embeds): the table's rows get the gradient of the labels that name them (a
    label twice in the batch: the sum), as autograd over the fp32 oracle gives it; all other parameters as before."""
    import oracle.schedulers as osch
    from ccnet_amd import schedulers as psch
    from ccnet_amd import training
    B, K = 3, 6
    cn, ocn = build_pair("controlnet", dict(TINY, num_class_embeds=K, **TINY_CE), 31, cuda)
    un, oun = build_pair("unet", dict(TINY, num_class_embeds=K), 32, cuda)
    g = torch.Generator().manual_seed(4)
    e, noise = (torch.randn(B, 4, 16, 16, generator=g) for _ in range(2))
    cond = torch.rand(B, 1, 128, 128, generator=g) * 2 - 1
    ctx = 0.5 * torch.randn(B, 77, 64, generator=g)
    t = torch.tensor([10, 500, 900])
    labels = torch.tensor([4, 1, 4])
    sch, osc = psch.DDPMScheduler(**SCHED), osch.DDPMScheduler(**SCHED)
    loss, grads = training.controlnet_loss_and_grads(cn, un, sch, e.to(cuda), noise.to(cuda), t.to(cuda), cond.to(cuda), ctx.to(cuda),
                                                     labels.to(cuda))
    for q in oun.parameters():
        q.requires_grad_(False)
    down, mid = ocn(osc.add_noise(original_samples=e, noise=noise, timesteps=t), t, cond, 1.0, ctx, labels)
    pred = oun(osc.add_noise(original_samples=e, noise=noise, timesteps=t), t, ctx, labels, down, mid)
    oloss = F.mse_loss(pred.float(), osc.get_velocity(e, noise, t).float())
    oloss.backward()
    assert abs(loss.item() - oloss.item()) <= 0.01 * abs(oloss.item())
    got, want = grads[cn.class_embedding.weight].cpu(), ocn.class_embedding.weight.grad
    assert got.shape == (K, want.shape[1])
    for row in range(K):
        assert (got[row] == 0).all() == (row not in (1, 4))
    a, b = got.reshape(-1), want.reshape(-1)
    print(f"class table: cosine {float(a @ b / a.norm() / b.norm()):.5f}, rel-L2 {rel_l2(a, b):.4f}")
    assert float(a @ b) >= 0.999 * float(a.norm() * b.norm()) and rel_l2(a, b) <= 0.05
    named = dict(cn.named_parameters())
    for name, q in ocn.named_parameters():
        assert (grads.get(named[name]) is None) == (q.grad is None), name
    with pytest.raises(IndexError):
        training.controlnet_loss_and_grads(cn, un, sch, e.to(cuda), noise.to(cuda), t.to(cuda), cond.to(cuda), ctx.to(cuda),
                                           torch.tensor([0, 1, K], device=cuda))


@pytest.mark.parametrize("mode,limit", [("norm", 0.05), ("norm", 1e6), ("value", 1e-3), (None, None)])
def test_train_step_clips_as_torch_does(cuda, mode, limit):
    """The gradients that train_step leaves, against torch's clipping of the ones it started from."""
    from ccnet_amd import schedulers as psch
    from ccnet_amd import training
    cn, _ = build_pair("controlnet", dict(TINY, **TINY_CE), 41, cuda, acq=True)
    un, _ = build_pair("unet", TINY, 42, cuda, acq=True)
    g = torch.Generator().manual_seed(5)
    e, noise, cond = torch.randn(2, 4, 16, 16, generator=g), torch.randn(2, 4, 16, 16, generator=g), torch.rand(2, 1, 128, 128, generator=g)
    ctx, t, acq = 0.5 * torch.randn(2, 77, 64, generator=g), torch.tensor([100, 700]), torch.tensor([[80.0, 300.0]])
    args = [v.to(cuda) for v in (e, noise, t, cond, ctx, acq)]
    sch = psch.DDPMScheduler(**SCHED)
    _, grads = training.controlnet_loss_and_grads(cn, un, sch, *args)
    twin = {p: nn.Parameter(p.detach().clone()) for p in grads}
    for p, q in twin.items():
        q.grad = grads[p].clone()
    if mode == "norm":
        want = float(torch.nn.utils.clip_grad_norm_(twin.values(), limit))
    else:
        want = float(torch.linalg.vector_norm(torch.stack([q.grad.norm() for q in twin.values()])))
        if mode == "value":
            torch.nn.utils.clip_grad_value_(twin.values(), limit)
    opt = torch.optim.SGD(cn.parameters(), lr=0.0)
    _, norm = training.train_step(cn, un, sch, opt, *args, clip_grad_norm_by=limit, clip_grad_norm_or_value=mode or "norm")
    assert (norm is None) == (mode is None)
    if norm is not None:
        assert abs(float(norm) - want) <= 1e-5 * want  # (torch sums in fp32)
    for p, q in twin.items():
        assert ((p.grad - q.grad).abs() <= 2e-5 * q.grad.abs()).all()


@pytest.mark.parametrize("q_off,k_off,v_off", [(0, 128, 128), (0, 0, 128), (64, 0, 128), (0, 0, 0)])
def test_tape_adds_where_queries_keys_and_values_share_columns(cuda, q_off, k_off, v_off):
    """Columns that serve twice (one projection for keys and values, for queries and keys, or slices that overlap) get the sum of what
    each use gives alone."""
    ops, tr = _mods()
    H, Hkv, d, n = 2, 2, 64, 90
    g = torch.Generator().manual_seed(6)
    x0 = torch.randn(n, 256, generator=g).to(BF16).to(cuda)
    do = torch.randn(n, H * d, generator=g).to(BF16).to(cuda)
    cu = torch.tensor([0, 40, 90], dtype=torch.int32, device=cuda)
    T = tr.Tape()
    x = tr._v2d(x0, True)
    T.attention_packed(x, q_off, x, k_off, v_off, cu, H, Hkv, d, 0.125).accumulate(do)
    T.backward()
    views = [x0[:, c:c + 128] for c in (q_off, k_off, v_off)]
    o, stats = ops.attention_packed(*views, cu, H, Hkv, d, 0.125, with_lse=True)
    want, mag = torch.zeros(n, 256, dtype=torch.float64, device=cuda), torch.zeros(n, 256, dtype=torch.float64, device=cuda)
    for c, gr in zip((q_off, k_off, v_off), ops.attention_packed_bwd(*views, o, do, stats, cu, H, Hkv, d, 0.125)):
        want[:, c:c + 128] += gr.double()
        mag[:, c:c + 128] += gr.double().abs()
    assert ((x.g.double() - want).abs() <= 2 * 2.0 ** -8 * (1 + 2.0 ** -8) * mag).all()  # two sums in bf16, each rounded
