"""Group norm, projections with adapters per row and the gated recurrence without a GPU: what the plan calls refuse, the
buffers a plan gives their side tensors, and what the step generator writes for them."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

from fortis_amd import plan as P, shim_hip as SH, step
from test_host_logic import pool, stats  # noqa: F401  (fixture)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _f(*shape):
    return np.ones(shape, np.float32)


@pytest.fixture
def plan(L):
    p = P.Plan()
    yield p
    p.close()


def test_group_norm_refusals(plan, capfd):
    x, y, small = plan.tensor(2 * 5 * 12), plan.tensor(2 * 5 * 12), plan.tensor(2 * 5 * 12 - 1)
    ok = dict(src=x, dst=y, NB=2, S=5, C_=12, G=3)
    for change in (dict(G=5), dict(G=0), dict(G=-3), dict(NB=0), dict(S=0), dict(S=-5), dict(C_=0), dict(eps=-1e-5), dict(eps=float("nan")),
                   dict(dst=x), dict(src=small), dict(dst=small), dict(src=99), dict(dst=-1), dict(NB=1 << 40, S=1 << 40)):
        with pytest.raises(ValueError):
            plan.group_norm(**dict(ok, **change))
    assert "group_norm" in capfd.readouterr().err
    assert plan._L.fortis_plan_group_norm(plan.handle, x, y, None, None, 1e-5, 2, 5, 12, 3, 0, 4, 0.0) == -1     # no such activation
    with pytest.raises(KeyError):
        plan.group_norm(act="gelu", **ok)
    plan.group_norm(**ok)                                      # and the call they all vary is accepted


def test_sizes_the_kernels_do_not_address_are_refused(plan):
    x, y = plan.tensor(1 << 20), plan.tensor(1 << 20)
    with pytest.raises(ValueError):
        plan.group_norm(x, y, 1, 1, 1 << 20, 1)                # channels
    plan.group_norm(x, y, 1, 1, (1 << 20) - 1, 1)
    i, one = plan.tensor(4), plan.tensor(4)
    with pytest.raises(ValueError):
        plan.linear_adapters(x, one, i, _f(1, 1 << 19), None, _f(1, 1, 1 << 19), _f(1, 1, 1), 1)
    with pytest.raises(ValueError):
        plan.linear_adapters(one, x, i, _f(1 << 19, 1), None, _f(1, 1, 1), _f(1, 1 << 19, 1), 1)


def test_overlapping_windows_are_refused(plan):
    base = plan.tensor(400)
    a, b, c = plan.view(base, 0, 120), plan.view(base, 116, 120), plan.view(base, 240, 120)
    for src, dst in ((a, b), (b, a), (a, base), (base, c)):
        with pytest.raises(ValueError):
            plan.group_norm(src, dst, 2, 5, 12, 3)
    plan.group_norm(a, c, 2, 5, 12, 3)


def test_linear_adapters_refusals(plan, capfd):
    x, i, y, small = plan.tensor(6 * 9), plan.tensor(6), plan.tensor(6 * 7), plan.tensor(5)
    L, h = plan._L, plan.handle
    W, A, U = _f(7, 9), _f(3, 2, 9), _f(3, 7, 2)

    def call(src=x, dst=y, index=i, w=P._p(W), a=P._p(A), u=P._p(U), B=6, K=9, N=7, nadapt=3, rank=2, act=0):
        return L.fortis_plan_linear_adapters(h, src, dst, index, w, None, a, u, None, B, K, N, nadapt, rank, act, 0.0)

    for change in (dict(src=y), dict(dst=x), dict(index=x), dict(index=y), dict(index=small), dict(index=-1), dict(index=50), dict(w=None), dict(a=None),
                   dict(u=None), dict(B=0), dict(B=7), dict(K=0), dict(K=10), dict(N=0), dict(N=8), dict(nadapt=0), dict(nadapt=4097),
                   dict(rank=0), dict(rank=257), dict(act=-1), dict(act=4), dict(B=1 << 31), dict(K=1 << 22, B=1)):
        assert call(**change) == -1, change
    assert "linear_adapters" in capfd.readouterr().err
    assert call(act=3) == 0
    for bad in (dict(A=_f(3, 2, 8)), dict(U=_f(3, 6, 2)), dict(U=_f(2, 7, 2)), dict(scale=_f(4)), dict(bias=_f(6))):
        with pytest.raises(AssertionError):
            plan.linear_adapters(**dict(dict(src=x, dst=y, index=i, W=W, bias=None, A=A, U=U, B=6), **bad))


def test_silu_stays_with_the_operators_that_compute_it(plan):
    x, y = plan.tensor(36), plan.tensor(36)
    with pytest.raises(KeyError):
        plan.linear(x, y, _f(6, 6), None, 6, "silu")
    assert plan._L.fortis_plan_linear(plan.handle, x, y, P._p(_f(6, 6)), None, 6, 6, 6, 3, 0.0) == -1


def test_convolutions_refuse_activations_that_they_do_not_compute(plan):
    x, y, w = plan.tensor(4 * 8 * 8 * 8), plan.tensor(4 * 16 * 16 * 16), _f(4, 4, 3, 3, 3)
    L, h = plan._L, plan.handle
    for act, rc in ((0, 0), (1, 0), (2, 0), (3, -1), (4, -1), (-1, -1)):
        assert L.fortis_plan_conv2d(h, x, y, P._p(w), None, None, None, None, None, 1e-5, 4, 8, 8, 4, 3, 3, 1, 1, act, 0.1, 0, 0) == rc
        assert L.fortis_plan_convt2d(h, x, y, P._p(w), None, 4, 8, 8, 4, 2, 2, 2, 0, 0, act, 0.1, 0, 0) == rc
        assert L.fortis_plan_conv3d(h, x, y, -1, P._p(w), None, 4, 8, 8, 8, 4, 3, 1, act, 0.1) == rc


def test_recurrence_refusals(plan, capfd):
    q, n, c = 4, 3, 5
    x, y, h0, h1, le = plan.tensor(q * n * 2 * c), plan.tensor(q * n * c), plan.tensor(q * c), plan.tensor(q * c), plan.tensor(q)
    small = plan.tensor(3)
    w = plan.view(x, 40, 20)
    ok = dict(src=x, dst=y, nseq=q, length=n, ch=c, h_in=h0, h_out=h1, lengths=le)
    for change in (dict(nseq=0), dict(length=0), dict(ch=0), dict(nseq=5), dict(length=4), dict(ch=6), dict(dst=x), dict(h_in=y), dict(h_out=x),
                   dict(h_out=y), dict(lengths=h1), dict(lengths=h0), dict(h_in=small), dict(h_out=small), dict(lengths=small), dict(h_in=70),
                   dict(h_in=w), dict(h_out=w), dict(nseq=1 << 33, length=1 << 30)):
        with pytest.raises(ValueError):
            plan.recurrence(**dict(ok, **change))
    assert "recurrence" in capfd.readouterr().err
    plan.recurrence(**ok)
    plan.recurrence(**dict(ok, h_in=h0, h_out=h0))
    plan.recurrence(**dict(ok, h_in=-1, h_out=-1, lengths=-1))


def test_half_overlapping_states_are_refused(plan):
    x, y, s = plan.tensor(16), plan.tensor(8), plan.tensor(12)
    a, b = plan.view(s, 0, 8), plan.view(s, 4, 8)
    with pytest.raises(ValueError):
        plan.recurrence(x, y, 1, 1, 8, h_in=a, h_out=b)
    plan.recurrence(x, y, 1, 1, 8, h_in=a, h_out=a)


def test_finalized_plans_take_no_operator(pool):  # noqa: F811
    L, dev = pool
    p = L.fortis_plan_create()
    x, y, h = L.fortis_plan_tensor(p, 64), L.fortis_plan_tensor(p, 32), L.fortis_plan_tensor(p, 32)
    assert L.fortis_plan_recurrence(p, x, y, h, h, -1, 1, 1, 8, 1, 0) == 0
    assert L.fortis_plan_finalize(p, x, y) == 0
    assert L.fortis_plan_recurrence(p, x, y, h, h, -1, 1, 1, 8, 1, 0) == -1
    assert L.fortis_plan_group_norm(p, x, y, None, None, 1e-5, 1, 1, 8, 1, 0, 0, 0.0) == -1
    assert L.fortis_plan_kernel_name(p, 0) == b"recurrence"
    L.fortis_plan_destroy(p)


def test_states_and_lengths_keep_buffers_of_their_own(pool):  # noqa: F811
    """A carried state, the lengths and a state that goes out live as long as the plan: no temporary of the pass shares
    their buffers, also where a state is a window beside one that a kernel writes."""
    L, dev = pool
    p = L.fortis_plan_create()
    T = lambda n: L.fortis_plan_tensor(p, 4 * n)  # noqa: E731
    x, a, b, c, d = T(16), T(8), T(16), T(8), T(8)
    both = T(32)
    written, state = L.fortis_plan_view(p, both, 0, 64), L.fortis_plan_view(p, both, 64, 32)
    out, le = T(8), T(8)
    ok = lambda r: r == 0 or pytest.fail("refused")  # noqa: E731
    ok(L.fortis_plan_recurrence(p, x, a, -1, -1, -1, 1, 1, 8, 1, 0))
    ok(L.fortis_plan_mask_relu(p, a, c, 1, 8, 8))
    ok(L.fortis_plan_concat_copy(p, c, written, 1, 8, 0, 2))
    ok(L.fortis_plan_concat_copy(p, c, written, 1, 8, 1, 2))
    ok(L.fortis_plan_recurrence(p, written, d, state, out, le, 1, 1, 8, 1, 0))
    ok(L.fortis_plan_mask_relu(p, d, b, 1, 8, 8))
    assert L.fortis_plan_finalize(p, x, b) == 0
    ptr = {t: L.fortis_plan_tensor_ptr(p, t) for t in (x, a, b, c, d, both, out, le)}
    for t in (both, out, le):
        assert all(ptr[t] != q for k, q in ptr.items() if k != t), t
    L.fortis_plan_destroy(p)
    assert stats(L)[1] == 0


def test_side_tensors_that_a_kernel_writes_in_part_keep_buffers_of_their_own(pool):  # noqa: F811
    """The lengths and the state lie in tensors whose front an earlier operation writes: the rest is still the caller's."""
    L, dev = pool
    dev.capacity = 4000
    p = L.fortis_plan_create()
    T = lambda n: L.fortis_plan_tensor(p, 4 * n)  # noqa: E731
    x, c, d, e, y = T(16), T(16), T(8), T(36), T(46)
    le, st = T(40), T(48)
    lengths, state = L.fortis_plan_view(p, le, 64, 96), L.fortis_plan_view(p, st, 64, 128)
    ok = lambda r: r == 0 or pytest.fail("refused")  # noqa: E731
    ok(L.fortis_plan_mask_relu(p, x, c, 1, 16, 16))
    ok(L.fortis_plan_mask_relu(p, c, le, 1, 16, 16))
    ok(L.fortis_plan_mask_relu(p, c, st, 1, 16, 16))
    ok(L.fortis_plan_recurrence(p, c, d, state, -1, lengths, 1, 1, 8, 1, 0))
    ok(L.fortis_plan_mask_relu(p, d, e, 1, 8, 8))
    ok(L.fortis_plan_mask_relu(p, e, y, 1, 8, 8))
    assert L.fortis_plan_finalize(p, x, y) == 0
    ptr = {t: L.fortis_plan_tensor_ptr(p, t) for t in (x, c, d, e, y, le, st)}
    for t in (le, st):
        assert all(ptr[t] != q for k, q in ptr.items() if k != t), t
    L.fortis_plan_destroy(p)


def test_rows_left_as_they_were_share_no_buffer(pool):  # noqa: F811
    """The output of a recurrence with lengths, at the end of a plan and between two operations."""
    L, dev = pool
    dev.capacity = 4000
    p = L.fortis_plan_create()
    T = lambda n: L.fortis_plan_tensor(p, 4 * n)  # noqa: E731
    x, a, b, c, d, e, y, le = T(16), T(16), T(16), T(8), T(16), T(16), T(8), T(1)
    ok = lambda r: r == 0 or pytest.fail("refused")  # noqa: E731
    ok(L.fortis_plan_mask_relu(p, x, a, 1, 16, 16))
    ok(L.fortis_plan_mask_relu(p, a, b, 1, 16, 16))
    ok(L.fortis_plan_recurrence(p, b, c, -1, -1, le, 1, 1, 8, 1, 0))
    ok(L.fortis_plan_concat_copy(p, c, d, 1, 8, 0, 2))
    ok(L.fortis_plan_concat_copy(p, c, d, 1, 8, 1, 2))
    ok(L.fortis_plan_mask_relu(p, d, e, 1, 16, 16))
    ok(L.fortis_plan_recurrence(p, e, y, -1, -1, le, 1, 1, 8, 1, 0))
    assert L.fortis_plan_finalize(p, x, y) == 0
    ptr = {t: L.fortis_plan_tensor_ptr(p, t) for t in (x, a, b, c, d, e, y, le)}
    for t in (c, y):
        assert all(ptr[t] != q for k, q in ptr.items() if k != t), t
    L.fortis_plan_destroy(p)


def test_one_row_of_a_batched_step_moves_no_states(pool, capfd):  # noqa: F811
    L, dev = pool
    for h_in, h_out in ((True, True), (False, True)):
        p = P.Plan()
        x, y, st = p.tensor(4 * 6), p.tensor(4 * 3), p.tensor(4 * 3)
        p.recurrence(x, y, 4, 1, 3, h_in=st if h_in else -1, h_out=st if h_out else -1)
        p.finalize(x, y)
        step.reset()
        step.bind(p, 24, 12, verdict="batched", count=4)
        out, errors = np.full(3, -5, np.float32), L.fortis_error_count()
        step.mlp_forward(np.ones(6, np.float32), out)
        assert (out == -5).all() and L.fortis_error_count() == errors            # nothing was asked of a device
        assert "one row" in capfd.readouterr().err
        step.reset()
        p.close()


def test_model_tensor_without_a_step(L):
    L.fortis_step_reset()
    assert L.fortis_model_tensor(0) is None


def _block(p, rows, q, n, c):
    """Projection with adapters -> recurrence -> group norm + SiLU -> projection with adapters."""
    rng = np.random.default_rng(0)
    w = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    x, i, g, h, st, z, y = p.tensor(rows * 6), p.tensor(rows), p.tensor(rows * 2 * c), p.tensor(rows * c), p.tensor(q * c), p.tensor(rows * c), p.tensor(rows * 5)
    p.linear_adapters(x, g, i, w(2 * c, 6), w(2 * c), w(3, 2, 6), w(3, 2 * c, 2), rows, w(3))
    p.recurrence(g, h, q, n, c, h_in=st, h_out=st)
    p.group_norm(h, z, rows, 1, c, 2, w(c), w(c), act="silu")
    p.linear_adapters(z, y, i, w(5, c), None, w(3, 2, c), w(3, 5, 2), rows, act="leaky", alpha=0.1)
    return p.finalize(x, y)


def test_generator_writes_the_operators(tmp_path):
    ops = _block(SH.OpList(), 12, 4, 3, 8)
    data = ops.as_json()
    outline = ops.outline("tensor<12x6xf32>", "tensor<12x5xf32>")
    text, _ = SH.emit_step({}, outline, data)
    assert text.count("fortis_plan_linear_adapters(p, ") == 2 and "t[4], t[4], -1, 4L, 3L, 8, 1, 0" in text and "2, 0, 3, 0.0f" in text
    (tmp_path / "step_tables.c").write_text(text)
    subprocess.check_call(["gcc", "-Wall", "-Werror", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), str(tmp_path / "step_tables.c")])
    for op, key, value in ((0, "index", -1), (0, "act", "gelu"), (1, "h_in", -2), (1, "lengths", 40), (2, "act", "tanh"), (2, "gamma", "w99")):
        broken = dict(data, ops=[dict(o) for o in data["ops"]])
        broken["ops"][op][key] = value
        with pytest.raises(ValueError):
            SH.emit_step({}, outline, broken)


def test_op_lists_refuse_weights_of_other_shapes():
    """What a live plan asserts: the generated C hands the sizes of W and A to calls that read the other blobs with them."""
    o = SH.OpList()
    x, i, y = o.tensor(54), o.tensor(6), o.tensor(42)
    ok = dict(src=x, dst=y, index=i, W=_f(7, 9), bias=_f(7), A=_f(3, 2, 9), U=_f(3, 7, 2), B=6, scale=_f(3))
    for bad in (dict(A=_f(3, 2, 8)), dict(U=_f(3, 2, 7)), dict(U=_f(2, 7, 2)), dict(bias=_f(6)), dict(scale=_f(4))):
        with pytest.raises(ValueError):
            o.linear_adapters(**dict(ok, **bad))
    for bad in (dict(gamma=_f(11)), dict(beta=_f(12, 1))):
        with pytest.raises(ValueError):
            o.group_norm(x, y, 2, 2, 12, 3, **bad)
    assert not o.ops and not o.weights
    o.linear_adapters(**ok)
    o.group_norm(x, y, 2, 2, 12, 3, "g0", _f(12))


def test_recurrence_without_host_memory_is_refused():
    """In a process of its own whose memory is bounded: the call says so instead of ending the program."""
    code = """
import resource
from fortis_amd import plan as P
p = P.Plan()
x, y = p.tensor(2), p.tensor(1)
call, h = p._L.fortis_plan_recurrence, p.handle
size = 1024 * int(next(l for l in open("/proc/self/status") if l.startswith("VmSize")).split()[1])
resource.setrlimit(resource.RLIMIT_AS, (size + (64 << 20),) * 2)
n = 0
while n < 1000000 and call(h, x, y, -1, -1, -1, 1, 1, 1, 1, 0) == 0:
    n += 1
print("refused", n < 1000000)
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "refused True" in r.stdout and "recurrence: out of host memory" in r.stderr, r
