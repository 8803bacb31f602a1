"""Token lookup and its gradient, packed causal attention forward and backward, gradient norm and clipping: every kernel
through its public entry point against the definition in 64 bits.  Tolerances count roundings: half a step of a value x is
at most 2^-24 |x| in fp32 and 2^-8 |x| in bf16."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
H16, H32 = 2.0 ** -8, 2.0 ** -24  # half a step, relative


def _ops():
    from ccnet_amd import ops
    return ops


def _randn(*shape, seed=0, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def _within(got, ref, tol, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((err - tol).max()):.3g} over its bound"


# ------------------------------------------------------------------ lookup
@pytest.mark.parametrize("T", [0, 1, 3, 77, 1000])
@pytest.mark.parametrize("C", [1, 7, 64, 320, 333, 1024, 1032])
@pytest.mark.parametrize("tdt,odt", [(F32, BF16), (F32, F32), (BF16, BF16), (BF16, F32)])
def test_lookup_is_one_rounding_of_the_scaled_row(cuda, T, C, tdt, odt):
    ops = _ops()
    table = _randn(50, C, seed=C, dtype=tdt)
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(0, 50, (T,), generator=g).cuda()
    for scale in (1.0, 22.627417):
        got = ops.embedding(ids, table, scale=scale, dtype=odt)
        assert got.dtype == odt and torch.equal(got, (table[ids].float() * scale).to(odt))
    assert torch.equal(ops.embedding(ids.int(), table, dtype=odt), ops.embedding(ids, table, dtype=odt))


def test_lookup_strides_shapes_and_ids_outside(cuda):
    ops = _ops()
    wide = _randn(40, 100, seed=1)
    ids = torch.tensor([[0, 39, -1], [40, 7, 1 << 40]], device="cuda")
    ref = wide[:, 4:68][ids.clamp(0, 39).reshape(-1)]
    ref[[2, 3, 5]] = 0
    for off in (4, 3):  # 16-byte aligned columns, and columns aligned to the element only
        ref = wide[:, off:off + 64][ids.clamp(0, 39).reshape(-1)]
        ref[[2, 3, 5]] = 0
        assert torch.equal(ops.embedding(ids, wide[:, off:off + 64], dtype=F32), ref)
        assert torch.equal(ops.embedding(ids.t(), wide[:, off:off + 64], dtype=F32), ref[[0, 3, 1, 4, 2, 5]])
    buf = torch.full((6, 80), 5.0, device="cuda")
    ops.embedding(ids, wide[:, :64], out=buf[:, 8:72])
    assert torch.equal(buf[:, 8:72], torch.where(torch.tensor([1, 1, 0, 0, 1, 0], device="cuda")[:, None] > 0, wide[ids.clamp(0, 39).reshape(-1), :64], 0.0))
    assert (buf[:, :8] == 5).all() and (buf[:, 72:] == 5).all()
    ids32 = torch.tensor([0, -1, 50, -(1 << 31), 39], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.embedding(ids32, wide, dtype=F32)[[1, 2, 3]], torch.zeros(3, 100, device="cuda"))


# ------------------------------------------------------------------ its gradient
def _grad_ref(ids, dy, vocab, scale, padding=None):
    ok = (ids >= 0) & (ids < vocab)
    if padding is not None:
        ok &= ids != padding
    ref = torch.zeros(vocab, dy.shape[1], dtype=F64, device="cuda")
    mag, count = torch.zeros_like(ref), torch.zeros(vocab, dtype=F64, device="cuda")
    ref.index_add_(0, ids[ok].long(), dy[ok].double())
    mag.index_add_(0, ids[ok].long(), dy[ok].double().abs())
    count.index_add_(0, ids[ok].long(), torch.ones(int(ok.sum()), dtype=F64, device="cuda"))
    # a sum of n terms in any tree: at most n - 1 roundings of partial sums, none above the sum of magnitudes (the tree of
    # long runs is shallower than 512); then one rounding of the product with the scale
    return ref * scale, (count.clamp(max=512)[:, None] * H32 * mag + 2 * H32 * ref.abs()) * scale


def _ids_of(kind, T, vocab, seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, vocab, (T,), generator=g)
    if kind == "one":
        ids[:] = vocab // 2
    elif kind == "mostly":
        ids[torch.rand(T, generator=g) < 0.8] = vocab - 1
    elif kind == "two":
        ids = torch.where(torch.arange(T) % 3 == 0, 0, vocab - 1)
    return ids.cuda()


@pytest.mark.parametrize("T,vocab,C", [(0, 5, 8), (1, 1, 1), (1, 300000, 8), (63, 2, 64), (64, 17, 333), (65, 1000, 1024), (97, 3, 520),
                                       (511, 17, 40), (512, 1, 512), (513, 2, 1032), (2464, 49408, 64), (8192, 1000, 24),
                                       (8193, 1000, 24), (8192, 262143, 8), (5000, 262144, 8), (20000, 70000, 16), (50001, 255, 72),
                                       (12289, 256, 9), (300, 20_000_000, 1), (9000, 20_000_000, 1)])
@pytest.mark.parametrize("kind", ["uniform", "one", "mostly", "two"])
def test_table_gradient(cuda, T, vocab, C, kind):
    ops = _ops()
    ids = _ids_of(kind, T, vocab, T + vocab)
    for dt in (F32, BF16):
        dy = _randn(T, C, seed=C, dtype=dt)
        ref, tol = _grad_ref(ids, dy, vocab, 22.0)
        got = ops.embedding_grad(ids, dy, vocab, scale=22.0)
        assert got.dtype == F32 and got.shape == (vocab, C)
        _within(got, ref, tol, f"T {T} vocab {vocab} C {C} {kind} {dt}")
        assert torch.equal(got, ops.embedding_grad(ids.int(), dy, vocab, scale=22.0)), "the sum's order depends on something else"


@pytest.mark.parametrize("kind", ["uniform", "mostly"])
def test_table_gradient_of_millions_of_positions(cuda, kind):
    """More than a million positions: a workgroup of the sort takes several blocks one after the other."""
    ops = _ops()
    T, vocab, C = 2_100_003, 70000, 8
    ids = _ids_of(kind, T, vocab, 5)
    dy = _randn(T, C, seed=6, dtype=BF16)
    at, x = ids.cpu(), dy.cpu().double()  # (on the CPU: one row's sum of 1.7 million terms takes atomics on the GPU minutes)
    ref, mag, count = torch.zeros(vocab, C, dtype=F64), torch.zeros(vocab, C, dtype=F64), torch.bincount(at, minlength=vocab).double()
    ref.index_add_(0, at, x)
    mag.index_add_(0, at, x.abs())
    # the sums of 512 rows (depth below 512), of which a long run's four waves each add every fourth in turn
    tol = (count.clamp(max=512) + count / 2048)[:, None] * H32 * mag + 2 * H32 * ref.abs()
    _within(ops.embedding_grad(ids, dy, vocab), ref.cuda(), tol.cuda(), kind)


def test_lookup_of_more_rows_than_a_launch_takes(cuda):
    ops = _ops()
    table = _randn(100, 3, seed=1, dtype=BF16)
    ids = torch.randint(0, 100, ((1 << 25) + 5,), device="cuda")
    got = ops.embedding(ids, table)
    assert torch.equal(got, table[ids])


def test_table_gradient_padding_and_ids_outside(cuda):
    ops = _ops()
    for T in (300, 9000):
        ids = _ids_of("mostly", T, 20, 3)
        ids[::7] = -1
        ids[1::7] = 20
        ids[2::7] = 1 << 33
        dy = _randn(T, 96, seed=4, dtype=BF16)
        ref, tol = _grad_ref(ids, dy, 20, 1.0, padding=19)
        got = ops.embedding_grad(ids, dy, 20, padding_idx=19)
        _within(got, ref, tol, "padding")
        assert (got[19] == 0).all()
        dy[ids == 19] = float("nan")  # what takes no part does not count, whatever it holds
        dy[ids < 0] = float("inf")
        assert torch.equal(got, ops.embedding_grad(ids, dy, 20, padding_idx=19))


def test_table_gradient_accumulates_and_leaves_other_rows(cuda):
    ops = _ops()
    ids = torch.tensor([3, 3, 9, 3], device="cuda")
    dy = _randn(4, 50, seed=1)
    base = _randn(12, 64, seed=2)
    out = base.clone()
    r = ops.embedding_grad(ids, dy, 12, scale=0.5, out=out[:, 7:57], accumulate=True)
    assert r.data_ptr() == out[:, 7:57].data_ptr()
    ref, tol = _grad_ref(ids, dy, 12, 0.5)
    want = base.double()
    want[:, 7:57] += ref
    _within(out[:, 7:57], want[:, 7:57], tol + H32 * want[:, 7:57].abs() * 2, "accumulate")
    keep = torch.ones(12, dtype=torch.bool)
    keep[[3, 9]] = False
    assert torch.equal(out[keep], base[keep]) and torch.equal(out[:, :7], base[:, :7]) and torch.equal(out[:, 57:], base[:, 57:])
    same = out.clone()
    ops.embedding_grad(ids[:0], dy[:0], 12, out=out[:, 7:57], accumulate=True)
    assert torch.equal(out, same)


def test_table_gradient_in_strided_memory(cuda):
    ops = _ops()
    ids = _ids_of("uniform", 500, 33, 1)
    wide = _randn(500, 200, seed=2, dtype=BF16)
    for off, C in ((8, 64), (3, 64), (8, 65)):
        dy = wide[:, off:off + C]
        ref, tol = _grad_ref(ids, dy, 33, 1.0)
        buf = torch.full((33, 160), 2.0, device="cuda")
        ops.embedding_grad(ids, dy, 33, out=buf[:, off:off + C])
        _within(buf[:, off:off + C], ref, tol, "strided")
        assert (buf[:, :off] == 2).all() and (buf[:, off + C:] == 2).all()


def test_table_gradient_in_a_graph_serves_other_ids(cuda):
    ops = _ops()
    for T, vocab in ((700, 90), (20000, 3000)):
        ids, dy = _ids_of("mostly", T, vocab, 1), _randn(T, 40, seed=1)
        out = torch.full((vocab, 40), 5.0, device="cuda")
        ops.embedding_grad(ids, dy, vocab, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.embedding_grad(ids, dy, vocab, out=out)
            rows = ops.embedding(ids, out, dtype=F32)
        for k, kind in enumerate(("uniform", "one", "two", "mostly")):
            ids.copy_(_ids_of(kind, T, vocab, k))
            dy.copy_(_randn(T, 40, seed=k + 5))
            graph.replay()
            torch.cuda.synchronize()
            got, looked = out.clone(), rows.clone()
            assert torch.equal(got, ops.embedding_grad(ids, dy, vocab)) and torch.equal(looked, got[ids]), kind


def test_table_gradient_against_differences(cuda):
    ops = _ops()
    ids = _ids_of("mostly", 200, 11, 5)
    dy = _randn(200, 24, seed=6)
    grad = ops.embedding_grad(ids, dy, 11, scale=3.0).double()
    w, u = _randn(11, 24, seed=7, dtype=F64), _randn(11, 24, seed=8, dtype=F64)
    loss = lambda t: float((3.0 * t[ids] * dy.double()).sum())  # noqa: E731
    slope = (loss(w + u) - loss(w - u)) / 2  # linear: the difference is the derivative
    _, tol = _grad_ref(ids, dy, 11, 3.0)
    assert abs(float((grad * u).sum()) - slope) <= float((tol * u.abs()).sum()) + 1e-9 * abs(slope)


# ------------------------------------------------------------------ packed causal attention
def _packed_inputs(lens, H, Hkv, d, pad=0, seed=0, gap=0):
    rows = sum(lens) + pad
    qkv = _randn(rows, (H + 2 * Hkv) * d + gap, seed=seed, dtype=BF16)
    q, k, v = qkv[:, :H * d], qkv[:, H * d:(H + Hkv) * d], qkv[:, (H + Hkv) * d:(H + 2 * Hkv) * d]
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)) if lens else [0], dtype=torch.int32).cuda()
    return q, k, v, _randn(rows, H * d, seed=seed + 1, dtype=BF16), cu


def _attention_ref(q, k, v, do, lens, H, Hkv, d, scale):
    """Outputs, log2-sum-exp and gradients by the formulas in 64 bits, each with its bound.  Roundings: P (2^-8 relative), the
    output; in the backward P, dS, the forward's P inside delta, and the result.  2^-10 covers the fp32 scores and
    exponentials (128 products of at most 2^-24 of the sum of magnitudes, which is below 2^9 here)."""
    rows, G = q.shape[0], H // Hkv
    z = lambda h: torch.zeros(rows, h * d, dtype=F64, device="cuda")  # noqa: E731
    o, to, dq, tq, dk, tk, dv, tv = z(H), z(H), z(H), z(H), z(Hkv), z(Hkv), z(Hkv), z(Hkv)
    lse = torch.full((H, rows), -math.inf, dtype=F64, device="cuda")
    first = 0
    for n in lens:
        r = slice(first, first + n)
        first += n
        future = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
        for h in range(H):
            a, b = slice(h * d, h * d + d), slice(h // G * d, h // G * d + d)
            Q, K, V, D = (x[r, c].double() for x, c in ((q, a), (k, b), (v, b), (do, a)))
            s = (scale * Q @ K.T).masked_fill(future, -math.inf)
            lse[h, r] = torch.logsumexp(s, 1) / math.log(2)
            p = torch.softmax(s, 1)
            O = p @ V
            o[r, a] = O
            near = (H16 + 2.0 ** -10) * (p @ V.abs())
            to[r, a] = near + H16 * (O.abs() + near)
            dp = D @ V.T
            delta = (D * O).sum(1, keepdim=True)
            ds = p * (dp - delta)
            # delta: the output as the kernel has it, before its rounding (and 2^-17 of that for the part kept beside it)
            eds = (H16 + 2.0 ** -10) * ds.abs() + p * (D.abs() * (near + 2.0 ** -16 * O.abs())).sum(1, keepdim=True) \
                + 2.0 ** -10 * p * (dp.abs() + delta.abs())
            dq[r, a] = scale * ds @ K
            tq[r, a] = scale * eds @ K.abs()
            dk[r, b] += scale * ds.T @ Q
            tk[r, b] += scale * eds.T @ Q.abs()
            dv[r, b] += p.T @ D
            tv[r, b] += (H16 + 2.0 ** -9) * p.T @ D.abs()
    out = {"o": (o, to), "lse": (lse, None)}
    for name, x, t in (("dq", dq, tq), ("dk", dk, tk), ("dv", dv, tv)):
        out[name] = (x, t + H16 * (x.abs() + t))
    return out


def _check_attention(got, ref, what):
    for name in ("o", "dq", "dk", "dv"):
        x, t = ref[name]
        _within(got[name], x, t, f"{what} {name}")
        # the worst case above adds magnitudes; of independent roundings (rms 2^-8 / sqrt 3 each, at most four in a row) the root
        # of the summed squares stays below 2^-7 of the result
        if x.norm() > 0 and x.shape[0] > 8:
            rel = float((got[name].double() - x).norm() / x.norm())
            assert rel <= 2.0 ** -7, f"{what} {name}: relative error {rel:.3g}"
    fin = ref["lse"][0] > -math.inf
    assert torch.equal(fin, got["lse"] > -math.inf)
    _within(got["lse"][fin], ref["lse"][0][fin], 2.0 ** -10 + 2.0 ** -20 * ref["lse"][0][fin].abs(), f"{what} lse")


NAMES = ("o", "lse", "dq", "dk", "dv")


def _run_attention(q, k, v, do, cu, H, Hkv, d, scale):
    ops = _ops()
    o, stats = ops.attention_packed(q, k, v, cu, H, Hkv, d, scale, with_lse=True)
    dq, dk, dv = ops.attention_packed_bwd(q, k, v, o, do, stats, cu, H, Hkv, d, scale)
    return {"o": o, "lse": stats.lse, "stats": stats, "dq": dq, "dk": dk, "dv": dv}


LENS = [(1,), (2,), (31,), (32,), (33,), (77,), (63, 64, 65), (127, 128, 129), (0, 5, 0, 0, 77, 0), (256,), (257, 300), (511, 3, 640),
        tuple(range(1, 78)), (1,) * 130, (96, 95, 65), (97, 64, 33, 96, 80), (0, 90, 200, 66, 1, 77, 96, 96)]
MANY = tuple((i * 37 + i // 5) % 71 for i in range(290)) + (0, 0, 301, 0, 130) + (3,) * 10  # (more sequences than are searched in order)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", LENS + [MANY], ids=lambda x: f"{len(x)}x{max(x)}")
def test_packed_attention(cuda, lens, d):
    for H, Hkv in ((1, 1), (6, 2)):
        q, k, v, do, cu = _packed_inputs(lens, H, Hkv, d, seed=sum(lens) + d + H)
        scale = d ** -0.5
        got = _run_attention(q, k, v, do, cu, H, Hkv, d, scale)
        _check_attention(got, _attention_ref(q, k, v, do, lens, H, Hkv, d, scale), f"{H}/{Hkv}")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(8, 8), (16, 8), (32, 8), (5, 5), (4, 1), (24, 8), (16, 16)])
def test_packed_attention_head_layouts(cuda, H, Hkv, d):
    lens = (40, 150, 1, 77)
    q, k, v, do, cu = _packed_inputs(lens, H, Hkv, d, pad=9, seed=H + d, gap=24)
    got = _run_attention(q, k, v, do, cu, H, Hkv, d, 0.2)
    _check_attention(got, _attention_ref(q, k, v, do, lens, H, Hkv, d, 0.2), f"{H}/{Hkv}")
    for name in ("o", "dq", "dk", "dv"):
        assert (got[name][sum(lens):] == 0).all()


@pytest.mark.parametrize("lens", [tuple(i * 7 % 9 for i in range(2600)) + (130, 0, 0), tuple(97 + i % 60 for i in range(1030)) + (0, 1, 300)],
                         ids=["short", "longer"])
def test_packed_attention_of_more_than_a_group_of_sequences(cuda, lens):
    q, k, v, do, cu = _packed_inputs(lens, 1, 1, 64, seed=9, pad=5)
    got = _run_attention(q, k, v, do, cu, 1, 1, 64, 0.125)
    _check_attention(got, _attention_ref(q, k, v, do, lens, 1, 1, 64, 0.125), f"{len(lens)} sequences")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(64, 64), (63, 21)])
def test_packed_attention_a_few_long_among_many_short(cuda, H, Hkv, d):
    """So many heads and sequences that a workgroup takes several heads of the sequences that are longer than most."""
    lens = tuple((i * 29) % 43 for i in range(100)) + (200,) + tuple((i * 29) % 41 for i in range(40)) + (65, 64) + (9,) * (8192 // Hkv // 2)
    lens = lens[:150] if Hkv == 64 else lens
    q, k, v, do, cu = _packed_inputs(lens, H, Hkv, d, seed=8, pad=30)
    got = _run_attention(q, k, v, do, cu, H, Hkv, d, 0.125)
    picks = [1, 5, 42, 100, 120, 141, 142, len(lens) - 1]
    first = [0] + list(torch.tensor(lens).cumsum(0))
    for i in picks:
        r = slice(int(first[i]), int(first[i + 1]))
        part = {n: (got[n][:, r] if n == "lse" else got[n][r]) for n in NAMES}
        _check_attention(part, _attention_ref(q[r], k[r], v[r], do[r], lens[i:i + 1], H, Hkv, d, 0.125), f"sequence {i} of {lens[i]}")
    n = sum(lens)
    assert all((got[x][n:] == 0).all() for x in ("o", "dq", "dk", "dv"))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(4, 1), (6, 1), (8, 2), (6, 3)])
def test_packed_attention_long_walks_of_few_key_heads(cuda, H, Hkv, d):
    """Mean length of 512 and more: the walk over a group's query heads is cut into parts that are summed afterwards."""
    lens = (700, 1200, 0, 513)
    q, k, v, do, cu = _packed_inputs(lens, H, Hkv, d, pad=77, seed=H + d)
    got = _run_attention(q, k, v, do, cu, H, Hkv, d, d ** -0.5)
    _check_attention(got, _attention_ref(q, k, v, do, lens, H, Hkv, d, d ** -0.5), f"{H}/{Hkv}")
    dq, dk, dv = (torch.full_like(got[x], 7.0) for x in ("dq", "dk", "dv"))
    _ops().attention_packed_bwd(q, k, v, got["o"], do, got["stats"], cu, H, Hkv, d, d ** -0.5, dq=dq, dk=dk, dv=dv)
    n = sum(lens)
    for x, name in ((dq, "dq"), (dk, "dk"), (dv, "dv")):
        assert (got[name][n:] == 0).all() and (x[n:] == 7).all() and torch.equal(x[:n], got[name][:n])


@pytest.mark.parametrize("d", [64, 128])
def test_packed_attention_without_sequences_or_rows(cuda, d):
    q, k, v, do, cu = _packed_inputs((), 2, 1, d, pad=70)
    for offsets in (cu, torch.zeros(4, dtype=torch.int32, device="cuda")):
        got = _run_attention(q, k, v, do, offsets, 2, 1, d, 0.1)
        for name in ("o", "dq", "dk", "dv"):
            assert (got[name] == 0).all()
    got = _run_attention(q[:0], k[:0], v[:0], do[:0], cu, 2, 1, d, 0.1)
    assert got["o"].shape == (0, 2 * d)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [(70, 33), MANY], ids=lambda x: f"{len(x)}x{max(x)}")
def test_rows_behind_the_last_sequence(cuda, lens, d):
    ops = _ops()
    H, Hkv = 4, 2
    q, k, v, do, cu = _packed_inputs(lens, H, Hkv, d, pad=141, seed=3)
    n = sum(lens)
    clean = _run_attention(q[:n], k[:n], v[:n], do[:n], cu, H, Hkv, d, 0.1)
    for t in (q, k, v, do):
        t[n:] = float("nan")
    got = _run_attention(q, k, v, do, cu, H, Hkv, d, 0.1)
    for name in ("o", "dq", "dk", "dv"):
        assert torch.equal(got[name][:n], clean[name]) and (got[name][n:] == 0).all(), name
    o = torch.full((n + 141, H * d), 7.0, dtype=BF16, device="cuda")
    both = torch.full((n + 141, (H + 2 * Hkv) * d), 7.0, dtype=BF16, device="cuda")
    ops.attention_packed(q, k, v, cu, H, Hkv, d, 0.1, out=o)
    dq, dk, dv = both[:, :H * d], both[:, H * d:(H + Hkv) * d], both[:, (H + Hkv) * d:]
    ops.attention_packed_bwd(q, k, v, got["o"], do, got["stats"], cu, H, Hkv, d, 0.1, dq=dq, dk=dk, dv=dv)
    for t, name in ((o, "o"), (dq, "dq"), (dk, "dk"), (dv, "dv")):
        assert torch.equal(t[:n], clean[name]) and (t[n:] == 7).all(), name


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [50, 300])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_values_that_are_not_finite_reach_only_who_sees_them(cuda, d, n, value):
    lens, H, Hkv = (20, n, 45), 2, 1
    q, k, v, do, cu = _packed_inputs(lens, H, Hkv, d, seed=n)
    clean = _ops().attention_packed(q, k, v, cu, H, Hkv, d, 0.1)
    for at in (0, 5, 31, 32, n - 1):
        for which in ("k", "v"):
            k2, v2 = k.clone(), v.clone()
            (k2 if which == "k" else v2)[20 + at, 3:6] = value
            got = _ops().attention_packed(q, k2, v2, cu, H, Hkv, d, 0.1)
            before = torch.ones(sum(lens), dtype=torch.bool)
            before[20 + at:20 + n] = False
            assert torch.equal(got[before], clean[before]), (which, at)
            if which == "v":  # every query that sees it has it, in its channels only
                after, cols = got[20 + at:20 + n].reshape(n - at, H, d), [3, 4, 5]
                rest = [c for c in range(d) if c not in cols]
                assert torch.equal(after[:, :, rest], clean[20 + at:20 + n].reshape(n - at, H, d)[:, :, rest])
                if math.isnan(value):
                    assert after[:, :, cols].isnan().all()
                else:  # (a probability that rounds to zero makes a NaN of it)
                    assert ((after[:, :, cols] == value) | after[:, :, cols].isnan()).all()
    k2, v2 = k.clone(), v.clone()
    k2[20:20 + n], v2[20:20 + n] = value, value
    got = _run_attention(q, k2, v2, do, cu, H, Hkv, d, 0.1)
    ref = _run_attention(q, k, v, do, cu, H, Hkv, d, 0.1)
    for name in ("o", "dq", "dk", "dv"):  # no other sequence notices, in any gradient
        assert torch.equal(got[name][:20], ref[name][:20]) and torch.equal(got[name][20 + n:], ref[name][20 + n:]), name


@pytest.mark.parametrize("d", [64, 128])
def test_packed_attention_scores_of_any_size(cuda, d):
    """Scores far below and above zero, rising along the keys (the running maximum grows all the way) and falling."""
    n, H = 200, 1
    for sign, big in ((1, 8.0), (-1, 8.0), (1, 3e4), (-1, 3e4)):
        q = torch.zeros(n, d, dtype=BF16, device="cuda")
        k = torch.zeros(n, d, dtype=BF16, device="cuda")
        q[:, 0] = sign
        k[:, 0] = (torch.arange(n, device="cuda") * big).to(BF16)
        v, do = _randn(n, d, seed=1, dtype=BF16), _randn(n, d, seed=2, dtype=BF16)
        cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        got = _run_attention(q, k, v, do, cu, H, H, d, 1.0)
        ref = _attention_ref(q, k, v, do, (n,), H, H, d, 1.0)
        # a score of 2^22 is known to 2^-24 of it: exponents off by 0.25 at most where big = 3e4, where one key takes all
        _within(got["o"], ref["o"][0], ref["o"][1] + (0 if big < 1e3 else 1e-6), f"{sign} {big}")
        assert all(torch.isfinite(got[x]).all() for x in ("dq", "dk", "dv"))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [(1, 1, 5, 1, 70), (1, 300, 1, 700)], ids=lambda x: f"{len(x)}x{max(x)}")
def test_a_query_that_sees_one_key_has_no_gradient(cuda, lens, d):
    """softmax of one score is 1 whatever the score is: dq of every sequence's first row and dk of a sequence of one row are zero, to
    the bit, and its dv is the sum of its group's do."""
    H, Hkv = 6, 3
    q, k, v, do, cu = _packed_inputs(lens, H, Hkv, d, seed=12)
    got = _run_attention(q, k, v, do, cu, H, Hkv, d, 0.7)
    first = [0] + list(torch.tensor(lens).cumsum(0))
    for n, at in zip(lens, map(int, first)):
        assert (got["dq"][at] == 0).all()
        if n == 1:
            assert (got["dk"][at] == 0).all()
            assert torch.equal(got["dv"][at], do[at].float().reshape(Hkv, 2, d).sum(1).reshape(-1).to(BF16))


@pytest.mark.parametrize("d", [64, 128])
def test_packed_attention_gradients_against_differences(cuda, d):
    lens, H, Hkv, scale = (45, 70), 2, 1, 0.15
    q, k, v, do, cu = _packed_inputs(lens, H, Hkv, d, seed=11)
    got = _run_attention(q, k, v, do, cu, H, Hkv, d, scale)
    ref = _attention_ref(q, k, v, do, lens, H, Hkv, d, scale)

    def loss(q, k, v):
        return float((_attention_ref(q, k, v, do, lens, H, Hkv, d, scale)["o"][0] * do.double()).sum())

    args = {"dq": q.double(), "dk": k.double(), "dv": v.double()}
    for i, name in enumerate(args):
        u, eps = _randn(*args[name].shape, seed=20 + i, dtype=F64), 1e-4
        up = [a + eps * u if n == name else a for n, a in args.items()]
        dn = [a - eps * u if n == name else a for n, a in args.items()]
        slope = (loss(*up) - loss(*dn)) / (2 * eps)
        have = float((got[name].double() * u).sum())
        assert abs(have - slope) <= float((ref[name][1] * u.abs()).sum()) + 1e-5 * abs(slope)
        # and much nearer than that bound, which adds magnitudes: the errors' signs are independent
        near = float((ref[name][1] * u).square().sum().sqrt()) * 4
        assert abs(have - slope) <= near + 1e-5 * abs(slope), (name, have, slope, near)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens", [(300, 7, 129, 64), (40, 64, 3, 77, 33) * 60, (77, 96, 70) * 30, (900, 2000, 64)],
                         ids=["mixed", "prompts", "padded", "long"])
def test_packed_attention_repeats_bit_for_bit(cuda, lens, d):
    q, k, v, do, cu = _packed_inputs(lens, 8, 2, d, seed=5)
    a = _run_attention(q, k, v, do, cu, 8, 2, d, 0.1)
    for _ in range(5):
        b = _run_attention(q, k, v, do, cu, 8, 2, d, 0.1)
        assert all(torch.equal(a[x], b[x]) for x in NAMES)


def test_packed_attention_rows_past_two_gigabytes(cuda):
    """Row offsets of more than 2^31 bytes, and a sequence that begins behind them."""
    rows, ld, d = 70000, 16384, 64
    big = torch.zeros(rows, ld, dtype=BF16, device="cuda")
    lens = (69000, 600, 400)
    small = _randn(1000, 3 * d, seed=9, dtype=BF16)
    big[69000:, 16000:16000 + 3 * d] = small
    q, k, v = (big[:, 16000 + i * d:16000 + (i + 1) * d] for i in range(3))
    assert 69000 * ld * 2 > 1 << 31
    cu = torch.tensor([0, 69000, 69600, 70000], dtype=torch.int32, device="cuda")
    do = torch.zeros(rows, d, dtype=BF16, device="cuda")
    do[69000:] = _randn(1000, d, seed=10, dtype=BF16)
    got = _run_attention(q, k, v, do, cu, 1, 1, d, 0.125)
    alone = _run_attention(small[:, :d], small[:, d:2 * d], small[:, 2 * d:], do[69000:], cu[1:] - 69000, 1, 1, d, 0.125)
    for name in ("o", "dq", "dk", "dv"):
        assert torch.equal(got[name][69000:], alone[name]), name
    assert (got["o"][:69000] == 0).all() and torch.equal(got["lse"][:, 69000:], alone["lse"])
    del lens


def test_packed_attention_offsets_that_are_wrong_stay_inside(cuda):
    """Offsets are clamped to the rows and to rising order by the kernel: such calls give rows of no meaning, no access outside."""
    q, k, v, do, _ = _packed_inputs((100,), 2, 2, 64, seed=1)
    ref = _run_attention(q, k, v, do, torch.tensor([0, 100], dtype=torch.int32, device="cuda"), 2, 2, 64, 0.1)
    got = _run_attention(q, k, v, do, torch.tensor([0, 5000], dtype=torch.int32, device="cuda"), 2, 2, 64, 0.1)
    assert all(torch.equal(got[x], ref[x]) for x in NAMES)
    got = _run_attention(q, k, v, do, torch.tensor([0, 100, 40], dtype=torch.int32, device="cuda"), 2, 2, 64, 0.1)
    assert torch.isfinite(got["o"]).all()
    cu = torch.randint(-10, 120, (400,), generator=torch.Generator().manual_seed(2), dtype=torch.int32).cuda()
    got = _run_attention(q, k, v, do, cu, 2, 2, 64, 0.1)
    assert got["o"].shape == ref["o"].shape and torch.equal(_run_attention(q, k, v, do, torch.tensor([0] + [100] * 300, dtype=torch.int32, device="cuda"),
                                                                         2, 2, 64, 0.1)["o"], ref["o"])


def test_packed_attention_in_a_graph_serves_other_lengths(cuda):
    H, Hkv, d = 4, 2, 64
    q, k, v, do, cu = _packed_inputs((60, 40, 100), H, Hkv, d, seed=6)
    _run_attention(q, k, v, do, cu, H, Hkv, d, 0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _run_attention(q, k, v, do, cu, H, Hkv, d, 0.1)
    for lens in ((60, 40, 100), (1, 198, 1), (0, 0, 200), (10, 20, 30), (60, 40, 100)):
        cu.copy_(torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32))
        q.copy_(_randn(*q.shape, seed=sum(lens), dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        ref = _run_attention(q, k, v, do, cu, H, Hkv, d, 0.1)
        assert all(torch.equal(got[x], ref[x]) for x in NAMES), lens


# ------------------------------------------------------------------ gradient norm and clipping
SIZES = [0, 1, 2, 3, 4, 5, 7, 8, 9, 255, 1000, 4096, 32768 * 4 + 3, 1, 0]


def _grads(dtype, seed=0, scale=1.0, odd=True):
    flat = _randn(sum(SIZES) + 64, seed=seed, dtype=dtype, scale=scale)
    out, at = [], 1 if odd else 0
    for n in SIZES:
        out.append(flat[at:at + n])
        at += n
        if not odd:
            at = -(-at // 8) * 8
    return flat, out


def _norm64(grads):
    return math.sqrt(math.fsum(float(g.double().square().sum()) for g in grads))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("odd", [True, False])
@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e3, 1e9])
def test_clip_by_norm(cuda, dtype, odd, max_norm):
    ops = _ops()
    flat, grads = _grads(dtype, odd=odd)
    before = flat.clone()
    copies = [g.clone() for g in grads]
    norm = _norm64(grads)
    assert abs(float(ops.grad_norm(grads)) - norm) <= 2 * H32 * norm
    outs = [torch.full_like(g, 9.0) for g in grads]
    got = ops.clip_grad_norm(grads, max_norm, out=outs)
    assert got.dtype == F32 and got.dim() == 0 and abs(float(got) - norm) <= 2 * H32 * norm
    assert torch.equal(flat, before)  # `out`: the gradients stay
    got = ops.clip_grad_norm(grads, max_norm)
    factor = min(1.0, max_norm / (norm + 1e-6))
    for g, o, c in zip(grads, outs, copies):
        assert torch.equal(g, o)
        # the factor's rounding and the product's (bf16: the product's to fp32 too)
        _within(g, c.double() * factor, c.double().abs() * factor * (H16 + 4 * H32 if dtype == BF16 else 4 * H32), "clipped")
    if factor == 1.0:
        assert torch.equal(flat, before)
    inside = torch.zeros_like(flat, dtype=torch.bool)
    for g in grads:
        inside[g.storage_offset():g.storage_offset() + g.numel()] = True
    assert torch.equal(flat[~inside], before[~inside])  # nothing between and behind the tensors


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_clip_by_value(cuda, dtype):
    ops = _ops()
    flat, grads = _grads(dtype)
    flat[40:44] = torch.tensor([float("nan"), float("inf"), float("-inf"), 0.25])
    want = [g.clamp(-0.25, 0.25) for g in grads]
    outs = [torch.empty_like(g) for g in grads]
    ops.clip_grad_value(grads, 0.25, out=outs)
    ops.clip_grad_value(grads, 0.25)
    for g, o, w in zip(grads, outs, want):
        assert torch.equal(g.nan_to_num(7), w.nan_to_num(7)) and torch.equal(o.nan_to_num(7), w.nan_to_num(7))
        assert torch.equal(g.isnan(), w.isnan())


def test_norm_of_many_tensors_and_of_any_size(cuda):
    ops = _ops()
    many = [_randn(1 + i % 37, seed=i) for i in range(401)]
    norm = _norm64(many)
    assert abs(float(ops.grad_norm(many)) - norm) <= 2 * H32 * norm
    assert abs(float(ops.clip_grad_norm(many, norm / 2)) - norm) <= 2 * H32 * norm
    assert abs(_norm64(many) - norm / 2) <= 1e-5 * norm
    for scale in (1e30, 1e-30, 1e-42):  # squares that leave the range of fp32
        g = [_randn(1000, seed=1, scale=scale), _randn(33, seed=2, scale=scale)]
        norm = _norm64(g)
        assert abs(float(ops.grad_norm(g)) - norm) <= 2 * H32 * norm + 2.0 ** -149
    assert float(ops.grad_norm([torch.zeros(0, device="cuda"), torch.zeros(3, device="cuda")])) == 0.0
    assert float(ops.grad_norm([torch.zeros(0, device="cuda")])) == 0.0
    g = torch.ones(5, device="cuda")
    assert abs(float(ops.grad_norm([g, g])) - math.sqrt(10)) <= 1e-6  # reading one tensor twice is no race


def test_dense_tensors_in_any_order_of_dimensions(cuda):
    ops = _ops()
    base = _randn(6, 5, 3, 4, seed=1)
    g = base.permute(0, 3, 1, 2)
    want = base.double() * (1.0 / (float(base.double().norm()) + 1e-6))
    ops.clip_grad_norm([g], 1.0)
    _within(base, want, want.abs() * 4 * H32, "permuted")
    out = torch.empty(6, 5, 3, 4, device="cuda").permute(0, 3, 1, 2)
    ops.clip_grad_norm([g], 0.5, out=[out])
    _within(out, g.double() * (0.5 / (float(g.double().norm()) + 1e-6)), g.double().abs() * 4 * H32, "permuted out")


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_a_norm_that_is_not_finite_scales_nothing(cuda, value):
    ops = _ops()
    flat, grads = _grads(F32)
    flat[1000] = value
    before = flat.clone()
    norm = ops.clip_grad_norm(grads, 1.0)
    assert not math.isfinite(float(norm)) and math.isnan(float(norm)) == math.isnan(value)
    assert torch.equal(flat.nan_to_num(7), before.nan_to_num(7))


def test_clip_in_a_graph(cuda):
    ops = _ops()
    flat, grads = _grads(F32, odd=False)
    outs = [torch.empty_like(g) for g in grads]
    ops.clip_grad_norm(grads, 1.0, out=outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grad_norm(grads, 1.0, out=outs)
    for seed in (3, 4, 5):
        flat.copy_(_randn(flat.numel(), seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        ref = ops.clip_grad_norm(grads, 1.0, out=outs)
        assert torch.equal(norm, ref) and all(torch.equal(a, b) for a, b in zip(got, outs))


# ------------------------------------------------------------------ streams and devices
def test_text_ops_on_another_stream(cuda):
    ops = _ops()
    ids = _ids_of("mostly", 9000, 500, 1)
    dy = _randn(9000, 64, seed=1, dtype=BF16)
    q, k, v, do, cu = _packed_inputs((300, 77), 4, 4, 64, seed=2)
    grads = [_randn(100000, seed=3), _randn(77, seed=4)]
    want = (ops.embedding_grad(ids, dy, 500), _run_attention(q, k, v, do, cu, 4, 4, 64, 0.1), ops.grad_norm(grads))
    torch.cuda.synchronize()
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):  # two streams at once, each with workspaces of its own
        for st in s:
            with torch.cuda.stream(st):
                got.append((ops.embedding_grad(ids, dy, 500), _run_attention(q, k, v, do, cu, 4, 4, 64, 0.1), ops.grad_norm(grads)))
    torch.cuda.synchronize()
    for g in got:
        assert torch.equal(g[0], want[0]) and all(torch.equal(g[1][x], want[1][x]) for x in NAMES) and torch.equal(g[2], want[2])


def test_a_single_row_of_any_stride(cuda):
    ops = _ops()
    wide = _randn(3, 300, seed=1, dtype=BF16)  # (600 bytes a row: no multiple of 16)
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    q, k, v = (wide[:1, c:c + 64] for c in (0, 64, 128))
    assert torch.equal(ops.attention_packed(q, k, v, cu, 1, 1, 64, 0.1), v)
    ids = torch.tensor([0], device="cuda")
    assert torch.equal(ops.embedding(ids, wide[:1, :64]), wide[:1, :64])
    out = torch.zeros(2, 67, device="cuda")
    ops.embedding_grad(ids, wide[:1, :64], 1, out=out[:1, :64])
    assert torch.equal(out[0, :64], wide[0, :64].float()) and (out[0, 64:] == 0).all() and (out[1] == 0).all()


# ------------------------------------------------------------------ batches of prompts of 64 to 96 rows, and what pins the precision
def _check_picks(got, q, k, v, do, lens, H, Hkv, d, scale, picks):
    first = [0] + torch.tensor(lens).cumsum(0).tolist()
    for i in picks:
        r = slice(first[i], first[i + 1])
        part = {n: (got[n][:, r] if n == "lse" else got[n][r]) for n in NAMES}
        _check_attention(part, _attention_ref(q[r], k[r], v[r], do[r], lens[i:i + 1], H, Hkv, d, scale), f"sequence {i} of {lens[i]}")
    assert all((got[x][first[-1]:] == 0).all() for x in ("o", "dq", "dk", "dv"))


PROMPTS = tuple(60 + i * 13 % 41 for i in range(140)) + (97, 0, 300, 200, 1)  # 60 to 100 rows, and a few longer ones


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(2, 1), (32, 32), (48, 16)])
def test_packed_attention_of_many_prompts_of_up_to_96_rows(cuda, H, Hkv, d):
    """More sequences than are searched in order, a mean of 64 to 96 rows, longer ones among them and rows behind the last; with many
    heads a workgroup takes several heads of the longer ones."""
    pad = 75
    rows, n_seq = sum(PROMPTS) + pad, len(PROMPTS)
    assert n_seq > 127 and 64 * n_seq < rows <= 96 * n_seq
    q, k, v, do, cu = _packed_inputs(PROMPTS, H, Hkv, d, seed=H + d, pad=pad)
    got = _run_attention(q, k, v, do, cu, H, Hkv, d, 0.1)
    picks = range(n_seq) if H == 2 else [0, 3, 37, 63, 64, 127, 128, 139, 140, 142, 143, 144]
    _check_picks(got, q, k, v, do, PROMPTS, H, Hkv, d, 0.1, picks)


@pytest.mark.parametrize("d", [64, 128])
def test_packed_attention_of_a_few_prompts_of_up_to_96_rows_with_many_heads(cuda, d):
    lens = tuple(70 + i * 7 % 27 for i in range(50)) + (130, 97, 0, 260)
    q, k, v, do, cu = _packed_inputs(lens, 64, 64, d, seed=d, pad=40)
    assert 64 * len(lens) < sum(lens) + 40 <= 96 * len(lens)
    got = _run_attention(q, k, v, do, cu, 64, 64, d, 0.1)
    _check_picks(got, q, k, v, do, lens, 64, 64, d, 0.1, [0, 1, 26, 49, 50, 51, 53])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,pad", [((96, 90, 70), 40), ((65, 96, 33, 81, 96), 120), ((60, 64, 1, 33), 300)])
def test_which_kernels_take_prompts_does_not_show(cuda, lens, pad, d):
    """The backward of prompts in one piece and the general one, which takes them where rows behind the last sequence lift the mean
    above 96: equal bits (no head group is cut at these lengths)."""
    H, Hkv, n = 6, 2, sum(lens)
    assert n <= 96 * len(lens) < n + pad < 512 * len(lens)
    q, k, v, do, cu = _packed_inputs(lens, H, Hkv, d, seed=n + d, pad=pad)
    a = _run_attention(q[:n], k[:n], v[:n], do[:n], cu, H, Hkv, d, 0.1)
    b = _run_attention(q, k, v, do, cu, H, Hkv, d, 0.1)
    for x in ("o", "dq", "dk", "dv"):
        assert torch.equal(a[x], b[x][:n]), x


# every backward kernel: general, its walks cut into parts, prompts of up to 64 and 96 rows, longer sequences among prompts
KERNELS = {"general": ((200, 130, 300, 64), 8, 4), "parts": ((700, 600), 8, 2), "64": ((64, 60, 33, 64) * 8, 8, 4), "96": ((96, 90, 77) * 8, 8, 4),
           "among": ((40,) * 40 + (300, 200), 8, 4), "among96": ((80,) * 40 + (300, 200), 8, 4)}


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("which", KERNELS)
def test_precision_of_the_row_sums_and_of_the_low_parts(cuda, which, d):
    """What the rounding of o takes away (o_low) and what the rounding of dS takes away from the first 16 of every 64 keys (queries)
    are carried, to 2^-8 of themselves.  Scores are zero here (q = 0 or k = 0), so that P has one value a row and its rounding
    in the forward takes nothing away; only those 16 rows of k (q) are not zero, so that only their dS enters dq (dk).  What is left
    beside the last rounding of a gradient: dS to 2^-17 and fp32 sums, together below 2^-14 of the result (its terms have independent
    signs), so the error is that of rounding the exact gradient, to (1 + (2^-14 / 1.6e-3)^2)^(1/2) < 1.001.  Without the low parts it
    would be 2^(1/2) of that; without o_low a query's dS would be off by 2^-9 of |o| |dO| altogether: above 1.05 in all of these.
    1.02 leaves room for elements that lie next to the border between two roundings."""
    lens, H, Hkv = KERNELS[which]
    q, k, v, do, cu = _packed_inputs(lens, H, Hkv, d, seed=d + len(lens))
    at = torch.cat([torch.arange(n) for n in lens]).cuda()
    few, zero = (at % 64 < 16)[:, None], torch.zeros_like
    for name, (q1, k1) in {"dq": (zero(q), k * few), "dk": (q * few, zero(k))}.items():
        got = _run_attention(q1, k1, v, do, cu, H, Hkv, d, 0.125)
        ref = _attention_ref(q1, k1, v, do, lens, H, Hkv, d, 0.125)
        x = ref[name][0]
        one = (x.to(BF16).double() - x).norm()
        ratio = float((got[name].double() - x).norm() / one)
        print(f"{which} d {d} {name}: {ratio:.4f} times one rounding")
        assert 0 < ratio <= 1.02, (name, ratio)
        # o_low: half a step of itself, at most half a step of o (2^-8 each), the division 2^-21; sums of at + 1 values in fp32
        _within(got["o"].double() + got["stats"].o_low.double(), ref["o"][0],
                (2.0 ** -16 + 2.0 ** -21) * ref["o"][0].abs() + 2.0 ** -23 * (at + 1)[:, None] * float(v.abs().max()), "o + o_low")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sign", [1, -1])
def test_packed_attention_gradients_of_scores_of_hundreds(cuda, sign, d):
    """Scores up to 1592 (2297 in base 2: fp32 knows them to 2^-13, inside the 2^-10 of the reference's bounds), rising or falling along the
    keys by 8 a key."""
    n = 200
    q, k = (torch.zeros(n, d, dtype=BF16, device="cuda") for _ in range(2))
    q[:, 0] = sign
    k[:, 0] = (torch.arange(n, device="cuda") * 8.0).to(BF16)
    v, do = _randn(n, d, seed=1, dtype=BF16), _randn(n, d, seed=2, dtype=BF16)
    for pad in (0, 20):
        cu = torch.tensor([0, n] if pad == 0 else [0, n] + [n] * 3, dtype=torch.int32, device="cuda")  # (general; among prompts)
        got = _run_attention(q, k, v, do, cu, 1, 1, d, 1.0)
        ref = _attention_ref(q, k, v, do, (n,), 1, 1, d, 1.0)
        for x in ("o", "dq", "dk", "dv"):
            # P and dS below 2^-126, out of the normal range of fp32 and bf16, may count as zero: each of the n < 2^8 terms of a sum is
            # then off by at most 2^-126 times |dO|, |V| or |dP - delta| (below 2^8) and |q| or |k| (below 2^11)
            _within(got[x], ref[x][0], ref[x][1] + 2.0 ** (8 + 8 + 11 - 126), f"{x} {pad}")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,pad", [((300, 77, 40, 0, 200, 129), 50), ((64, 1, 33, 90, 77, 50), 9), ((700, 1200, 513), 0), ((40, 64, 3, 77, 33) * 30, 20)],
                         ids=["mixed", "prompts", "parts", "many"])
def test_bits_of_a_sequence_follow_from_its_rows_and_the_totals(cuda, lens, pad, d):
    """The same sequences in another order, beside other values: equal totals (rows, sequences, heads), equal bits."""
    H, Hkv = 8, 2
    q, k, v, do, cu = _packed_inputs(lens, H, Hkv, d, pad=pad, seed=d)
    a = _run_attention(q, k, v, do, cu, H, Hkv, d, 0.1)
    first = cu.tolist()
    order = torch.randperm(len(lens), generator=torch.Generator().manual_seed(1)).tolist()
    keep = order[::2]  # these keep their values, the others get new ones
    q2, k2, v2, do2, cu2 = _packed_inputs([lens[i] for i in order], H, Hkv, d, pad=pad, seed=d + 1)
    at = cu2.tolist()
    where = [(slice(first[i], first[i + 1]), slice(at[j], at[j + 1])) for j, i in enumerate(order) if i in keep]
    for x, y in ((q, q2), (k, k2), (v, v2), (do, do2)):
        for r, s in where:
            y[s] = x[r]
    b = _run_attention(q2, k2, v2, do2, cu2, H, Hkv, d, 0.1)
    for r, s in where:
        assert torch.equal(a["lse"][:, r], b["lse"][:, s])
        for x in ("o", "dq", "dk", "dv"):
            assert torch.equal(a[x][r], b[x][s]), x
