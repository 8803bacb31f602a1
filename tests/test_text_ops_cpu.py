"""What the entry points for token lookup, packed attention and gradient clipping refuse, on the host: nothing here launches."""
import ctypes as C
import math

import pytest
import torch

BF16 = torch.bfloat16
EINVAL, EUNSUP, EWS = -1, -2, -4


def _err():
    from ccnet_amd.lib import CcnetError
    return CcnetError


def _lib():
    from ccnet_amd import lib
    return lib.load()


def test_cpu_tensors_are_refused():
    from ccnet_amd import ops
    ids, x = torch.zeros(4, dtype=torch.int64), torch.zeros(4, 64)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    b = x.to(BF16)
    for call in (lambda: ops.embedding(ids, x), lambda: ops.embedding_grad(ids, x, 9), lambda: ops.attention_packed(b, b, b, cu, 1, 1, 64, 1.0),
                 lambda: ops.attention_packed_bwd(b, b, b, b, b, ops.PackedStats(x[:1, :4], b), cu, 1, 1, 64, 1.0), lambda: ops.grad_norm([x]),
                 lambda: ops.clip_grad_norm([x], 1.0), lambda: ops.clip_grad_value([x], 1.0)):
        with pytest.raises(_err(), match="GPU only"):
            call()


def test_wrapper_refusals_before_any_launch():
    from ccnet_amd import ops
    x = torch.zeros(4, 64)
    ids = torch.zeros(4, dtype=torch.int64)
    for call in (lambda: ops.embedding(ids, x[0]), lambda: ops.embedding(ids, x.t()), lambda: ops.embedding(ids, x.half()),
                 lambda: ops.embedding_grad(ids, x, 9, accumulate=True), lambda: ops.embedding_grad(ids, x, 0),
                 lambda: ops.embedding_grad(ids, x, 9, padding_idx=9), lambda: ops.grad_norm([]), lambda: ops.grad_norm([x, x.to(BF16)]),
                 lambda: ops.grad_norm([x.half()]), lambda: ops.grad_norm([x[:, :3]]), lambda: ops.grad_norm([x[:1].expand(4, 64)]),
                 lambda: ops.clip_grad_norm([x], -1.0), lambda: ops.clip_grad_norm([x], float("nan")),
                 lambda: ops.clip_grad_value([x], -1.0), lambda: ops.clip_grad_norm([x], 1.0, out=[]),
                 lambda: ops.clip_grad_norm([x], 1.0, out=[x.t()]), lambda: ops.clip_grad_norm([x], 1.0, out=[x.to(BF16)])):
        with pytest.raises(_err()):
            call()


def test_clip_outputs_must_not_overlap_other_gradients():
    """The aliasing rules of the C entry points, on host addresses that are never dereferenced: the calls that break one return
    CCNET_EINVAL before a launch; the ones that keep them get as far as the next check, a workspace that is too small."""
    l = _lib()
    base = 1 << 20

    def go(grads, outs):
        n = len(grads)
        mk = lambda v: (C.c_void_p * n)(*[base + 4 * lo for lo, _ in v])  # noqa: E731
        num = (C.c_int64 * n)(*[hi - lo for lo, hi in grads])
        out = mk(outs)
        return l.ccnet_clip_grad_norm(mk(grads), out, num, n, 0, 1.0, C.c_void_p(base), 0, C.c_void_p(base), None)

    a, b, c, d = (0, 10), (10, 20), (20, 30), (40, 50)
    e = (0, 0)
    for grads, outs in (([a, b, c], [a, b, c]), ([a, b], [c, d]), ([a, b], [a, c]), ([c, a], [(50, 60), a]), ([a, e, b], [c, e, d]), ([a, a], [b, c])):
        assert go(grads, outs) == EWS, (grads, outs)
    for grads, outs in (([a, b], [b, a]), ([a, b], [(5, 15), c]), ([a], [(1, 11)]), ([a, b, c], [(50, 60), (12, 22), (70, 80)]), ([a, b], [c, c]),
                        ([a, b], [(60, 70), (65, 75)]), ([(0, 50), (60, 70)], [(50, 100), (30, 40)]), ([a, a], [a, a]), ([a, a], [a, b])):
        assert go(grads, outs) == EINVAL, (grads, outs)


def test_overlapping_clip_is_named():
    from ccnet_amd import ops
    with pytest.raises(_err(), match="overlap"):
        ops._check_clip(EINVAL, "clip_grad_norm")
    with pytest.raises(_err(), match="workspace"):
        ops._check_clip(EWS, "clip_grad_norm")


def test_dense_layouts():
    from ccnet_amd import ops
    x = torch.zeros(4, 6, 5)
    assert all(ops._dense(t) for t in (x, x.permute(2, 0, 1), x.transpose(0, 1), x[1], x[:1], torch.zeros(0), x[1, 1, 1]))
    assert not any(ops._dense(t) for t in (x[:, ::2], x[:, :3], x[..., 1], x[:1].expand(4, 6, 5)))


def test_c_abi_refusals():
    l = _lib()
    p, *P = [C.c_void_p((1 + k) << 20) for k in range(12)]  # never dereferenced: every call here returns before a launch
    E = l.ccnet_embedding
    ok = [p, 8, 4, 10, P[0], 0, 64, 64, 1.0, P[1], 1, 64, None]
    for i, v in ((1, 2), (2, -1), (3, 0), (4, None), (5, 2), (6, 63), (7, 0), (9, None), (10, 3), (11, 10), (0, None), (0, C.c_void_p(1028)),
                 (4, C.c_void_p(1026)), (9, C.c_void_p(1025))):
        a = list(ok)
        a[i] = v
        assert E(*a) == EINVAL, (i, v)
    a = list(ok)
    a[2] = 0
    assert E(*a) == 0  # no rows: nothing to do
    G = l.ccnet_embedding_grad
    need = l.ccnet_embedding_grad_workspace_bytes(1000, 64)
    assert need > 1000 * 16 and l.ccnet_embedding_grad_workspace_bytes(0, 64) == 0
    ok = [p, 8, 1000, 10, P[0], 1, 64, 64, 1.0, -1, P[1], 64, 0, P[2], need, None]
    for i, v, rc in ((1, 3, EINVAL), (2, -1, EINVAL), (3, 0, EINVAL), (3, 0x7fffffff, EINVAL), (4, None, EINVAL), (5, 2, EINVAL), (6, 8, EINVAL),
                     (7, 0, EINVAL), (10, None, EINVAL), (10, C.c_void_p(1026), EINVAL), (11, 63, EINVAL), (13, None, EINVAL),
                     (13, C.c_void_p(1028), EINVAL), (14, need - 1, EWS), (2, (1 << 30) + 1, EUNSUP)):
        a = list(ok)
        a[i] = v
        assert G(*a) == rc, (i, v)
    assert G(None, 8, 0, 10, None, 1, 64, 64, 1.0, -1, P[1], 64, 1, None, 0, None) == 0  # no positions: nothing to add
    F = l.ccnet_attention_packed_bf16
    ok = [p, 256, P[0], 128, P[1], 128, P[2], 256, P[3], 3, 100, 4, 2, 64, 0.125, 1, None, None, None]
    odd = C.c_void_p(1 << 20 | 8)
    for i, v, rc in ((0, None, EINVAL), (0, odd, EINVAL), (1, 255, EINVAL), (1, 248, EINVAL), (2, None, EINVAL), (3, 64, EINVAL), (4, odd, EINVAL),
                     (5, 132, EINVAL), (6, None, EINVAL), (7, 192, EINVAL), (8, None, EINVAL), (9, -1, EINVAL), (10, -1, EINVAL), (11, 0, EINVAL),
                     (11, 3, EINVAL), (12, 0, EINVAL), (13, 96, EUNSUP), (13, 32, EUNSUP), (14, 0.0, EINVAL), (14, -1.0, EINVAL),
                     (14, float("nan"), EINVAL), (14, float("inf"), EINVAL), (3, 1 << 25, EUNSUP), (17, odd, EINVAL), (10, (1 << 30) + 1, EUNSUP), (11, 1 << 21, EUNSUP), (9, 1 << 28, EUNSUP)):
        a = list(ok)
        a[i] = v
        assert F(*a) == rc, (i, v)
    a = list(ok)
    a[10] = 0
    assert F(*a) == 0
    B = l.ccnet_attention_packed_bwd_bf16
    size = l.ccnet_attention_packed_bwd_workspace_bytes
    need = size(3, 100, 4, 2, 64)
    assert need >= 100 * 4 * 4 and size(1, 4096, 16, 4, 64) >= 4096 * 16 * 4 + 2 * 2 * 4096 * 4 * 64 * 4  # (long walks of few key heads are cut)
    ok = [p, 256, P[0], 128, P[1], 128, P[2], 256, P[3], P[4], 256, P[5], P[6], 256, P[7], 128, P[8], 128, P[9], 3, 100, 4, 2, 64, 0.125, 1, P[10], need, None]
    for i in (0, 2, 4, 6, 9, 11, 12, 14, 16, 18, 26):
        a = list(ok)
        a[i] = None
        assert B(*a) == EINVAL, i
    for i in (1, 3, 5, 7, 10, 13, 15, 17):
        a = list(ok)
        a[i] = 100
        assert B(*a) == EINVAL, i
    for i, v, rc in ((8, odd, EINVAL), (26, odd, EINVAL), (21, 3, EINVAL), (23, 80, EUNSUP), (24, 0.0, EINVAL), (20, 0, 0), (20, (1 << 30) + 1, EUNSUP), (27, need - 1, EWS)):
        a = list(ok)
        a[i] = v
        assert B(*a) == rc, (i, v)
    ptrs, n = (C.c_void_p * 2)(1 << 20, 1 << 24), (C.c_int64 * 2)(1000, 70000)
    need = l.ccnet_grad_norm_workspace_bytes(ptrs, n, 2, 0)
    assert need == 8 * (1 + 1 + 5)
    for args, rc in (((ptrs, n, 2, 2, p, need, p, None), EINVAL), ((ptrs, n, -1, 0, p, need, p, None), EINVAL), ((None, n, 2, 0, p, need, p, None), EINVAL),
                     ((ptrs, n, 2, 0, None, need, p, None), EINVAL), ((ptrs, n, 2, 0, p, need - 1, p, None), EWS), ((ptrs, n, 2, 0, p, need, None, None), EINVAL)):
        assert l.ccnet_grad_norm(*args) == rc
    bad = (C.c_void_p * 2)(1 << 20 | 2, 1 << 24)
    none = (C.c_void_p * 2)(1 << 20, None)
    neg = (C.c_int64 * 2)(-1, 5)
    for q in (bad, none):
        assert l.ccnet_grad_norm(q, n, 2, 0, p, need, p, None) == EINVAL
        assert l.ccnet_clip_grad_norm(ptrs, q, n, 2, 0, 1.0, p, need, p, None) == EINVAL
        assert l.ccnet_clip_grad_value(ptrs, q, n, 2, 0, 1.0, None) == EINVAL
    assert l.ccnet_grad_norm(ptrs, neg, 2, 0, p, need, p, None) == EINVAL and l.ccnet_grad_norm_workspace_bytes(ptrs, neg, 2, 0) == 0
    for m in (-1.0, float("nan")):
        assert l.ccnet_clip_grad_norm(ptrs, ptrs, n, 2, 0, m, p, need, p, None) == EINVAL
        assert l.ccnet_clip_grad_value(ptrs, ptrs, n, 2, 0, m, None) == EINVAL
    assert l.ccnet_clip_grad_norm(ptrs, ptrs, n, 2, 0, 1.0, p, need - 1, p, None) == EWS


def test_results_must_not_share_memory_with_operands():
    """Addresses that are never dereferenced: a call that breaks the rule returns CCNET_EINVAL, one that keeps it gets as far as the
    next check or, in the last lines, to the size that no launch can have."""
    l = _lib()
    p = lambda b: C.c_void_p((1 << 30) + b)  # noqa: E731

    def look(table, ldt, out, ldo, ids=0, T=4):  # table fp32 [10][64], out bf16 [T][64]
        return l.ccnet_embedding(p(ids), 8, T, 10, p(table), 0, ldt, 64, 1.0, p(out), 1, ldo, None)

    for a in ((4096, 64, 4096, 64), (4096, 64, 4096 + 2556, 64), (4096, 64, 4096 - 510, 64), (4096, 64, 16, 64), (4096, 256, 4096 + 2, 512), (4096, 256, 4096 + 256, 260)):
        assert look(*a) == EINVAL, a
    G, need = l.ccnet_embedding_grad, l.ccnet_embedding_grad_workspace_bytes(100, 64)
    for dy, lddy, out, ldg, ids in ((1 << 20, 64, 1 << 20, 64, 0), (1 << 20, 64, (1 << 20) + 64 * 100 * 4 - 4, 64, 0), (1 << 20, 64, 400, 64, 0),
                                    (1 << 20, 128, (1 << 20) + 252, 128, 0), (1 << 20, 128, (1 << 20) + 260, 128, 0), (1 << 20, 128, (1 << 20) + 256, 132, 0)):
        assert G(p(ids), 8, 100, 10, p(dy), 0, lddy, 64, 1.0, -1, p(out), ldg, 0, p(1 << 25), need, None) == EINVAL, (dy, lddy, out, ldg)

    most = 1 << 28  # sequences: more workgroups than a launch has, the check behind this one

    def fwd(q, k, v, o, ldq=768, ldk=768, ldv=768, ldo=768, low=None):
        return l.ccnet_attention_packed_bf16(p(q), ldq, p(k), ldk, p(v), ldv, p(o), ldo, p(0), most, 100, 4, 4, 64, 1.0, 1, None, low and p(low), None)

    m = 1 << 20
    for a in ((m, m + 512, m + 1024, 4 * m), (m, m + 512, m + 1024, m), (m, 2 * m, 3 * m, m + 512), (m, m + 512, 2 * m, m + 1024), (m, m + 512, m + 1024, m + 1536 * 100)):
        assert fwd(*a) == EUNSUP, a
    for a in ((m, m + 512, m + 1024, m + 512), (m, m + 512, m + 1024, m + 1024), (m, m + 512, m + 1024, m + 16), (m, 2 * m, 3 * m, m + 1536), (m, m + 512, m + 1024, m + 1536 * 99)):
        assert fwd(*a) == EINVAL, a
    assert fwd(m, 2 * m, 3 * m, m, ldo=776) == EINVAL and fwd(m, 2 * m, 3 * m, m + 512, ldo=776) == EINVAL
    assert fwd(m, 2 * m, 3 * m, 4 * m, low=5 * m) == EUNSUP and fwd(m, 2 * m, 3 * m, 4 * m, low=4 * m) == EINVAL
    size = l.ccnet_attention_packed_bwd_workspace_bytes(most, 100, 4, 4, 64)

    def bwd(dq, dk, dv, ld=768):  # q, k, v slices of one matrix at 1 m, o at 2 m, o_low 3 m, do 4 m, lse 5 m
        return l.ccnet_attention_packed_bwd_bf16(p(m), 768, p(m + 512), 768, p(m + 1024), 768, p(2 * m), 256, p(3 * m), p(4 * m), 256, p(5 * m), p(dq), ld,
                                                 p(dk), ld, p(dv), ld, p(0), most, 100, 4, 4, 64, 1.0, 1, p(9 * m), size, None)

    for a in ((6 * m, 6 * m + 512, 6 * m + 1024), (6 * m, 7 * m, 8 * m)):
        assert bwd(*a) == EUNSUP, a
    for a in ((m, 6 * m, 7 * m), (6 * m, 6 * m, 7 * m), (6 * m, 7 * m, 7 * m + 256), (6 * m, m + 512, 7 * m), (6 * m, 7 * m, m + 1024), (2 * m, 6 * m, 7 * m),
              (3 * m + 51184, 6 * m, 7 * m), (6 * m, 4 * m, 7 * m), (6 * m, 7 * m, 5 * m + 1584), (6 * m + 16, 7 * m, 6 * m + 512)):
        assert bwd(*a) == EINVAL, a


def test_packed_attention_wrapper_refusals():
    from ccnet_amd import ops
    b = torch.zeros(4, 256, dtype=BF16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(_err(), match="divide"):
        ops._packed_operands(b, b, b, cu, 3, 2, 64)
    for bad in (cu.long(), cu[None], cu[:0], torch.zeros(4, dtype=torch.int32)[::2]):
        with pytest.raises(_err(), match="cu_seqlens"):
            ops._packed_operands(b, b, b, bad, 4, 4, 64)
    for q, k, v in ((b.float(), b, b), (b[:, :64], b, b), (b, b[:2], b), (b, b, b[:, ::2]), (b[0], b, b)):
        with pytest.raises(_err()):
            ops._packed_operands(q, k, v, cu, 4, 4, 64)
    with pytest.raises(_err(), match="all of dq"):
        ops.attention_packed_bwd(b, b, b, b, b, ops.PackedStats(b, b), cu, 4, 4, 64, 1.0, dq=b)


def _packed_fwd(lse=None, low=None, cu=0, n_seq=1 << 28):
    """The forward over 100 rows of q, k, v = column slices of one matrix at 1 MiB (4 heads of 64 each), o at 4 MiB; addresses that are
    never dereferenced, and so many sequences that the call ends at the size no launch can have."""
    m = 1 << 20
    p = lambda b: C.c_void_p((1 << 31) + b)  # noqa: E731
    return _lib().ccnet_attention_packed_bf16(p(m), 768, p(m + 512), 768, p(m + 1024), 768, p(4 * m), 256, p(cu), n_seq, 100, 4, 4, 64, 1.0, 1,
                                              None if lse is None else p(lse), None if low is None else p(low), None)


def test_row_statistics_must_not_share_memory_with_operands_or_results():
    m = 1 << 20  # (q, k, v: 153,600 bytes; o and o_low: 51,200; lse: 1,600)
    for lse in (8 * m, m + 153600, m - 1600, 4 * m + 51200, 4 * m - 1600, 5 * m + 51200):
        assert _packed_fwd(lse=lse, low=5 * m) == EUNSUP, lse
    for lse in (m, m + 153596, m - 1596, m + 512, m + 1024, 4 * m, 4 * m + 51196, 4 * m - 4, 5 * m, 5 * m + 51196):
        assert _packed_fwd(lse=lse, low=5 * m) == EINVAL, lse


def _packed_bwd(ws, dq=6, lse=None, n_seq=1 << 28, extra=0, cu=0, shift=0):
    """The backward over 100 rows, 4 heads of 64: q, k, v slices of one matrix at 1 MiB, o at 2, o_low 3, do 4, lse 5, dq 6, dk 7, dv 8."""
    m, l = 1 << 20, _lib()
    p = lambda b: C.c_void_p((1 << 31) + b)  # noqa: E731
    size = l.ccnet_attention_packed_bwd_workspace_bytes(n_seq, 100, 4, 4, 64)
    return l.ccnet_attention_packed_bwd_bf16(p(m), 768, p(m + 512), 768, p(m + 1024), 768, p(2 * m), 256, p(3 * m), p(4 * m), 256, p(5 * m + shift), p(dq * m),
                                             256, p(7 * m), 256, p(8 * m), 256, p(cu), n_seq, 100, 4, 4, 64, 1.0, 1, p(ws), size + extra, None)


def test_backward_workspace_must_not_share_memory_with_operands_or_results():
    m = 1 << 20  # (the workspace: 100 x 4 sums of 4 bytes, in whole 256)
    assert _lib().ccnet_attention_packed_bwd_workspace_bytes(1 << 28, 100, 4, 4, 64) == 1792
    for ws in (9 * m, 8 * m + 51200, m - 1792, 5 * m + 1600):
        assert _packed_bwd(ws) == EUNSUP, ws
    assert _packed_bwd(m - 1792, extra=1 << 20) == EUNSUP  # what is handed over beyond the need is not touched
    for ws in (m, m + 512, m + 1024, m + 153584, m - 1776, 2 * m, 3 * m + 16, 4 * m, 5 * m, 5 * m + 1584, 6 * m, 7 * m + 51184, 8 * m - 16, 8 * m):
        assert _packed_bwd(ws) == EINVAL, ws


def test_offsets_must_not_share_memory_with_results():
    m = 1 << 20  # (4 offsets: 16 bytes, which every workgroup reads while others write results)
    for cu in (4 * m, 4 * m + 51196, 4 * m - 12, 5 * m, 5 * m + 51196, 8 * m, 8 * m + 1596):
        assert _packed_fwd(lse=8 * m, low=5 * m, cu=cu, n_seq=3) == EINVAL, cu
    for cu in (6 * m, 6 * m - 4, 7 * m, 8 * m + 51196, 9 * m, 9 * m + 1788):
        assert _packed_bwd(9 * m, cu=cu, n_seq=3) == EINVAL, cu


def test_row_statistics_offsets_and_norms_are_aligned():
    m = 1 << 20
    assert _packed_fwd(lse=8 * m + 4) == EUNSUP
    for bad in (1, 2):
        assert _packed_fwd(lse=8 * m + bad) == EINVAL and _packed_fwd(cu=16 * m + bad) == EINVAL
        assert _packed_bwd(9 * m, shift=bad) == EINVAL and _packed_bwd(9 * m, cu=16 * m + bad) == EINVAL
        l, g, n = _lib(), (C.c_void_p * 1)(1 << 20), (C.c_int64 * 1)(1000)
        p = lambda b: C.c_void_p((1 << 31) + b)  # noqa: E731
        assert l.ccnet_grad_norm(g, n, 1, 0, p(0), 16, p(64 + bad), None) == EINVAL
        assert l.ccnet_clip_grad_norm(g, g, n, 1, 0, 1.0, p(0), 16, p(64 + bad), None) == EINVAL


def test_table_gradient_workspace_must_not_share_memory_with_operands_or_results():
    l, m = _lib(), 1 << 20
    p = lambda b: C.c_void_p((1 << 31) + b)  # noqa: E731
    need = l.ccnet_embedding_grad_workspace_bytes(100, 64)  # ids: 800 bytes at 1 MiB, dy: 25,600 at 2, the table: 2,560 at 3

    def go(ws):
        return l.ccnet_embedding_grad(p(m), 8, 100, 10, p(2 * m), 0, 64, 64, 1.0, -1, p(3 * m), 64, 0, p(ws), need, None)

    for ws in (m, m + 784, m - need + 16, 2 * m, 2 * m + 25584, 2 * m - need + 16, 3 * m, 3 * m + 2544, 3 * m - 16):
        assert go(ws) == EINVAL, ws


def test_norm_and_its_workspace_must_not_share_memory_with_the_tensors():
    l, m = _lib(), 1 << 20
    at = lambda b: (1 << 31) + b  # noqa: E731
    p = lambda b: C.c_void_p(at(b))  # noqa: E731
    g, o, n = (C.c_void_p * 3)(at(m), None, at(2 * m)), (C.c_void_p * 3)(at(3 * m), None, at(4 * m)), (C.c_int64 * 3)(1000, 0, 70000)
    need = l.ccnet_grad_norm_workspace_bytes(g, n, 3, 0)
    assert need == 8 * (1 + 1 + 5)
    far = 8 * m
    for ws, norm in ((m, far), (m + 3992, far), (m - 8, far), (2 * m + 279992, far), (far, m), (far, m + 3996), (far, 2 * m + 279996), (far, far),
                     (far, far + need - 4)):
        assert l.ccnet_grad_norm(g, n, 3, 0, p(ws), need, p(norm), None) == EINVAL, (ws, norm)
        assert l.ccnet_clip_grad_norm(g, o, n, 3, 0, 1.0, p(ws), need, p(norm), None) == EINVAL, (ws, norm)
    for ws, norm in ((3 * m, far), (3 * m - 8, far), (4 * m + 279992, far), (far, 3 * m), (far, 4 * m + 279996)):
        assert l.ccnet_clip_grad_norm(g, o, n, 3, 0, 1.0, p(ws), need, p(norm), None) == EINVAL, (ws, norm)


@pytest.mark.parametrize("mode,limit", [("norm", 0.5), ("value", 0.5), ("norm", None)])
@pytest.mark.parametrize("bad", [None, float("inf"), float("nan")])
def test_train_step_leaves_the_gradients_of_a_skipped_step_as_they_are(monkeypatch, mode, limit, bad):
    """A loss that is not finite skips the step even where every gradient is finite (an overflowing square has a finite derivative): no
    parameter moves and no gradient is clipped.  The clipping calls are replaced by what they document, on the CPU."""
    from ccnet_amd import ops, training

    def norm_of(grads):
        return torch.stack([g.double().square().sum() for g in grads]).sum().sqrt().float()

    def clip(grads, max_norm):
        n = norm_of(grads)
        f = min(1.0, max_norm / (float(n) + 1e-6)) if torch.isfinite(n) else 1.0
        for g in grads:
            g *= f
        return n

    def clip_value(grads, lim):
        for g in grads:
            g.clamp_(-lim, lim)

    for name, fn in (("grad_norm", norm_of), ("clip_grad_norm", clip), ("clip_grad_value", clip_value)):
        monkeypatch.setattr(ops, name, fn)
    net = torch.nn.Linear(3, 2)
    net._invalidate = lambda: None
    grads = {p: torch.arange(1, p.numel() + 1).float().reshape(p.shape) for p in net.parameters()}
    want = math.sqrt(sum(float(g.square().sum()) for g in grads.values()))
    before = {p: (p.detach().clone(), g.clone()) for p, g in grads.items()}
    loss = torch.tensor(2.0 if bad is None else bad)
    monkeypatch.setattr(training, "controlnet_loss_and_grads", lambda *a: (loss, grads))
    opt = torch.optim.SGD(net.parameters(), lr=0.1)
    got, norm = training.train_step(net, None, None, opt, *[None] * 5, clip_grad_norm_by=limit, clip_grad_norm_or_value=mode)
    assert got is loss and (norm is None) == (bad is not None or limit is None)
    if norm is not None:
        assert norm.shape == () and abs(float(norm) - want) <= 1e-6 * want
    for p, (value, grad) in before.items():
        if bad is not None:
            assert torch.equal(p, value) and torch.equal(p.grad, grad)
        else:
            scaled = grad if limit is None else grad * (limit / (want + 1e-6)) if mode == "norm" else grad.clamp(-limit, limit)
            assert torch.allclose(p.grad, scaled) and torch.allclose(p, value - 0.1 * scaled)


def test_the_stride_of_a_single_row_says_nothing():
    """One row of a matrix whose stride is no multiple of 16 bytes, or is below the row's width (a view of one row may say so), is as
    good as a row by itself."""
    from ccnet_amd import ops
    wide = torch.zeros(3, 100, dtype=BF16)
    assert wide[:1, :64].stride() == (100, 1)
    for t in (wide[:1, :64], wide[1:2, 32:96], wide[0, :64].expand(1, 64), torch.zeros(64, dtype=BF16).as_strided((1, 64), (1, 1)), wide[:0, :64]):
        assert ops._rows_ld(t, "q", t.shape[0], 64, (BF16,)) == 64
    assert ops._rows_ld(wide[:1, :61], "q", 1, 61, (BF16,)) == 64  # (whole 16-byte vectors)
    assert ops._rows_ld(wide[:2, :64], "q", 2, 64, (BF16,)) == 100
    assert ops._rows_ld(torch.zeros(1, 64, dtype=BF16).as_strided((1, 64), (1 << 40, 1)), "q", 1, 64, (BF16,)) == 64
