"""The operators on token ids, logits and pairs of answers (ml-ease_amd/operators.py, include/mlease_operators.h) against plain
64-bit computations. Tolerances count roundings: u = 2^-24 for a 32-bit operation, half a step of the result's type for the last one."""
import ctypes
import json
import math
import os
import re
import subprocess
import sys
import threading

import numpy as np
import pytest
import torch

import mlease_amd  # noqa: F401
from mlease_amd import operators
from mlease_amd.operators import HipOperators

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
gpu = pytest.mark.gpu


def half_step(value, dtype):
    """Half a step of dtype at |value| (64 bits): relative eps / 2, and half the smallest subnormal step near 0."""
    f = torch.finfo(dtype)
    return value.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def within(got, want, tol):
    got, want = got.double().cpu(), want.double().cpu()
    tol = tol.double().cpu() if torch.is_tensor(tol) else torch.full_like(want, tol)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), "%d of %d off, worst %g of its tolerance" % (bad.sum(), bad.numel(), ((got - want).abs() / tol.clamp(min=1e-300))[bad].max())


def rng(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


# ---------------------------------------------------------------------------------------------- without a GPU
def test_header_and_binding_name_the_same_entry_points():
    hdr = open(os.path.join(ROOT, "include", "mlease_operators.h")).read()
    declared = set(re.findall(r"^int (mlx_[a-z_0-9]+)\s*\(", hdr, re.M))
    assert declared == set(operators.OPERATOR_SYMBOLS)
    lib = operators.load_operators()
    for sym in declared:
        assert hasattr(lib, sym), sym


P = 1 << 20        # an address that is never followed: every call below is refused before the device is asked for


@pytest.mark.parametrize("change", [
    dict(type=3), dict(type=-1), dict(id_type=2), dict(n_rows=-1), dict(n_rows=2 ** 31), dict(n_ids=-1), dict(n_ids=2 ** 31), dict(width=0), dict(table=None), dict(out=None),
    dict(ids=None), dict(ld_out=15), dict(ld_table=-1), dict(table=P + 1), dict(out=2 * P + 1), dict(ids=4 * P + 4), dict(out=P), dict(out=4 * P), dict(ld_table=2 ** 62)])
def test_lookup_refuses(change):
    a = dict(type=1, table=P, n_rows=8, width=16, ld_table=16, id_type=1, ids=4 * P, n_ids=5, scale=1.0, out=2 * P, ld_out=16)
    a.update(change)
    L = operators.load_operators()
    assert L.mlx_embedding_lookup(0, None, *[a[k] for k in ("type", "table", "n_rows", "width", "ld_table", "id_type", "ids", "n_ids", "scale", "out", "ld_out")]) == -1
    assert b"mlx_embedding_lookup" in L.mlx_last_error(None)


@pytest.mark.parametrize("change", [
    dict(type=5), dict(id_type=-1), dict(grad_type=2), dict(n_rows=2 ** 31), dict(n_ids=-5), dict(width=0), dict(width=2 ** 31), dict(grad_out=None), dict(ids=None), dict(grad=None),
    dict(ld_grad=15), dict(ld_grad_out=-16), dict(workspace=None), dict(workspace=8 * P + 64), dict(workspace_bytes=8), dict(grad=P), dict(grad=4 * P), dict(grad=8 * P), dict(ids=4 * P + 2)])
def test_gradient_refuses(change):
    L = operators.load_operators()
    need = ctypes.c_size_t()
    assert L.mlx_embedding_gradient_workspace(8, 16, 600, ctypes.byref(need)) == 0 and need.value > 0
    a = dict(type=1, grad_out=P, ld_grad_out=16, id_type=1, ids=4 * P, n_ids=600, scale=1.0, accumulate=0, grad_type=1, grad=2 * P, n_rows=8, width=16, ld_grad=16,
             workspace=8 * P, workspace_bytes=need.value)
    a.update(change)
    assert L.mlx_embedding_gradient(0, None, *[a[k] for k in ("type", "grad_out", "ld_grad_out", "id_type", "ids", "n_ids", "scale", "accumulate", "grad_type", "grad", "n_rows",
                                                              "width", "ld_grad", "workspace", "workspace_bytes")]) == -1
    assert b"mlx_embedding_gradient" in L.mlx_last_error(None)


@pytest.mark.parametrize("n,width,needs", [(1, 1, False), (512, 64, False), (513, 64, True), (512, 2048, False), (512, 2049, True), (16, 65536, False), (16, 65537, True)])
def test_gradient_of_few_entries_needs_no_workspace(n, width, needs):
    """One launch up to 512 entries and 4096 workgroups of 64 lanes' columns of float32, told by the query for both widths of elements."""
    need = ctypes.c_size_t()
    assert operators.load_operators().mlx_embedding_gradient_workspace(100, width, n, ctypes.byref(need)) == 0 and (need.value > 0) == needs


@pytest.mark.parametrize("change", [dict(type=9), dict(id_type=3), dict(n_tokens=-1), dict(n_tokens=2 ** 31), dict(n_classes=0), dict(logits=None), dict(logits=P + 1), dict(ld=-1),
                                    dict(target=None), dict(target=2 * P + 4), dict(logp=None), dict(stats=None), dict(stats=3 * P + 2), dict(logp=P), dict(stats=2 * P), dict(logp=4 * P)])
def test_loglik_refuses(change):
    L = operators.load_operators()
    a = dict(type=1, logits=P, n_tokens=4, n_classes=10, ld=10, id_type=1, target=2 * P, logp=3 * P, stats=4 * P, workspace=8 * P, workspace_bytes=P)
    a.update(change)
    assert L.mlx_token_loglik(0, None, *[a[k] for k in ("type", "logits", "n_tokens", "n_classes", "ld", "id_type", "target", "logp", "stats", "workspace", "workspace_bytes")]) == -1
    assert b"mlx_token_loglik" in L.mlx_last_error(None)


@pytest.mark.parametrize("change", [dict(type=9), dict(id_type=3), dict(n_tokens=-1), dict(n_classes=2 ** 31), dict(logits=None), dict(target=None), dict(stats=None), dict(g=None),
                                    dict(out=None), dict(ld_out=9), dict(out=P + 2), dict(out=P, ld_out=12), dict(out=2 * P), dict(out=3 * P), dict(out=4 * P)])
def test_loglik_gradient_refuses(change):
    L = operators.load_operators()
    a = dict(type=1, logits=P, n_tokens=4, n_classes=10, ld=10, id_type=1, target=2 * P, stats=3 * P, g=4 * P, out=5 * P, ld_out=10)
    a.update(change)
    assert L.mlx_token_loglik_gradient(0, None, *[a[k] for k in ("type", "logits", "n_tokens", "n_classes", "ld", "id_type", "target", "stats", "g", "out", "ld_out")]) == -1
    assert b"mlx_token_loglik_gradient" in L.mlx_last_error(None)


@pytest.mark.parametrize("change", [dict(n=-1), dict(n=2 ** 31), dict(pairs=-1), dict(pairs=2 ** 30), dict(beta=math.inf), dict(beta=math.nan), dict(scale=math.nan), dict(smoothing=-0.1),
                                    dict(smoothing=1.5), dict(smoothing=math.nan), dict(logp=None), dict(seq=None), dict(loss=None), dict(pair_loss=None), dict(seq=3 * P + 4),
                                    dict(logp=P + 1), dict(grad=P), dict(grad=2 * P), dict(margin=3 * P), dict(loss=6 * P), dict(ratio=7 * P), dict(grad=9 * P), dict(grad=4 * P)])
def test_preference_refuses(change):
    L = operators.load_operators()
    a = dict(logp=P, ref=2 * P, n=100, seq=3 * P, pairs=3, beta=0.1, smoothing=0.0, scale=1.0, mean=0, mask=4 * P, weight=5 * P, offset=6 * P, loss=7 * P, pair_loss=8 * P, margin=9 * P,
             ratio=10 * P, grad=11 * P, workspace=16 * P, workspace_bytes=P)
    a.update(change)
    assert L.mlx_preference_loss(0, None, *[a[k] for k in ("logp", "ref", "n", "seq", "pairs", "beta", "smoothing", "scale", "mean", "mask", "weight", "offset", "loss", "pair_loss",
                                                           "margin", "ratio", "grad", "workspace", "workspace_bytes")]) == -1
    assert b"mlx_preference_loss" in L.mlx_last_error(None)


@pytest.mark.parametrize("call", ["mlx_embedding_gradient_workspace", "mlx_token_loglik_workspace", "mlx_preference_loss_workspace"])
def test_workspace_queries_refuse(call):
    f = getattr(operators.load_operators(), call)
    n = len(f.argtypes) - 1
    need = ctypes.c_size_t(7)
    assert f(*[4] * n, None) == -1
    assert f(*[-1] * n, ctypes.byref(need)) == -1
    assert f(*[2 ** 31] * n, ctypes.byref(need)) == -1
    assert need.value == 7


def _on_cpu():
    """The binding with tensors of this host: what it refuses, it refuses before a pointer reaches the library."""
    ops = HipOperators.__new__(HipOperators)
    ops.L, ops.device = operators.load_operators(), 0
    ops._setup(torch)
    ops._at = torch.device("cpu")
    ops._stream = lambda: None
    return ops


def test_binding_refuses():
    ops = _on_cpu()
    t, i = torch.zeros(4, 6), torch.zeros(5, dtype=torch.int64)
    f, seq = torch.zeros(5), torch.zeros(5, dtype=torch.int64)
    for call in (
        lambda: ops.embedding_lookup(t[0], i),                                   # not a matrix
        lambda: ops.embedding_lookup(t.double(), i),                             # type
        lambda: ops.embedding_lookup(t.t(), i),                                  # rows not contiguous
        lambda: ops.embedding_lookup(t, i.to(torch.int16)),
        lambda: ops.embedding_lookup(t, i[None]),
        lambda: ops.embedding_lookup(t, torch.zeros(10, dtype=torch.int64)[::2]),
        lambda: ops.embedding_lookup(t, i, out=torch.zeros(5, 5)),
        lambda: ops.embedding_lookup(t, i, out=torch.zeros(5, 6, dtype=torch.float16)),
        lambda: ops.embedding_lookup(t.to("meta"), i),                           # another device
        lambda: ops.embedding_lookup(t, i.to("meta")),
        lambda: ops.embedding_gradient(t, i, 3),                                 # 4 rows, 5 ids
        lambda: ops.embedding_gradient(t, i[:4], 3, accumulate=True),            # nothing to add to
        lambda: ops.embedding_gradient(t, i[:4], 3, out=torch.zeros(4, 6)),
        lambda: ops.embedding_gradient(t, i[:4], 3, dtype=torch.float64),
        lambda: ops.token_loglik(t, i),
        lambda: ops.token_loglik_gradient(t, i[:4], torch.zeros(4, 3), f[:4]),
        lambda: ops.token_loglik_gradient(t, i[:4], torch.zeros(4, 2), f),
        lambda: ops.token_loglik_gradient(t, i[:4], torch.zeros(4, 2, dtype=torch.float64), f[:4]),
        lambda: ops.preference_loss(f, None, seq[:4]),                           # an even number of bounds
        lambda: ops.preference_loss(f, f[:4], seq),
        lambda: ops.preference_loss(f.double(), None, seq),
        lambda: ops.preference_loss(f, None, seq.to(torch.int32)),
        lambda: ops.preference_loss(f, None, seq, mask=f),
        lambda: ops.preference_loss(f, None, seq, weight=f),
        lambda: ops.preference_loss(f, None, seq, offset=torch.zeros(2, dtype=torch.float64)),
    ):
        with pytest.raises(ValueError):
            call()
    for call in (
        lambda: ops.embedding_gradient(t, i[:4], 3, dtype=torch.float16),        # refused by the library
        lambda: ops.preference_loss(f, None, seq, smoothing=2.0),
        lambda: ops.preference_loss(f, None, seq, beta=math.inf),
    ):
        with pytest.raises(RuntimeError, match="mlease_hip error -1"):
            call()


def _float_arguments(ops):
    """For each floating tensor that a call takes: its name, the call with that tensor replaced, and a tensor that it takes."""
    i, seq = torch.zeros(5, dtype=torch.int64), torch.tensor([0, 2, 5])
    t, f, stats, pair = torch.zeros(4, 6), torch.zeros(5), torch.zeros(5, 2), torch.zeros(1)
    rows = torch.zeros(5, 6)
    return [
        ("table", lambda x: ops.embedding_lookup(x, i), t), ("out", lambda x: ops.embedding_lookup(t, i, out=x), rows),
        ("grad_out", lambda x: ops.embedding_gradient(x, i, 3), rows), ("out", lambda x: ops.embedding_gradient(rows, i, 4, out=x), t),
        ("out", lambda x: ops.embedding_gradient(rows, i, 4, out=x, accumulate=True), t), ("logits", lambda x: ops.token_loglik(x, i), rows),
        ("logits", lambda x: ops.token_loglik_gradient(x, i, stats, f), rows), ("stats", lambda x: ops.token_loglik_gradient(rows, i, x, f), stats),
        ("grad_logp", lambda x: ops.token_loglik_gradient(rows, i, stats, x), f), ("out", lambda x: ops.token_loglik_gradient(rows, i, stats, f, out=x), rows.clone()),
        ("logp", lambda x: ops.preference_loss(x, None, seq), f), ("ref_logp", lambda x: ops.preference_loss(f, x, seq), f.clone()),
        ("weight", lambda x: ops.preference_loss(f, None, seq, weight=x), pair), ("offset", lambda x: ops.preference_loss(f, None, seq, offset=x), pair.clone())]


def test_what_automatic_differentiation_follows_is_refused():
    """A gradient that would be missing without a word; where torch itself records nothing, or from a detached tensor, the call is made."""
    for what, call, tensor in _float_arguments(_on_nothing()):
        call(tensor)
        with pytest.raises(ValueError, match="%s requires a gradient" % what):
            call(tensor.clone().requires_grad_())
        with pytest.raises(ValueError, match="%s requires a gradient" % what):
            call(tensor.clone().requires_grad_() * 2)
        call(tensor.clone().requires_grad_().detach())
        with torch.no_grad():
            call(tensor.clone().requires_grad_())
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(ValueError, match="%s carries a forward-mode tangent" % what):
                call(torch.autograd.forward_ad.make_dual(tensor.clone(), torch.ones_like(tensor)))
            call(tensor)


def test_views_that_torch_negates_are_refused():
    """The memory of imag(conj(z)) holds the negatives of its values."""
    ops = _on_nothing()
    z = torch.complex(torch.ones(4, 1), torch.ones(4, 1)).conj()
    lazy, seq = torch.imag(z), torch.zeros(3, dtype=torch.int64)
    assert lazy.is_neg()
    for x in (lazy, lazy[:1]):
        i = torch.zeros(x.shape[0], dtype=torch.int64)
        with pytest.raises(ValueError, match="negates"):
            ops.embedding_lookup(x, i)
        with pytest.raises(ValueError, match="negates"):
            ops.embedding_lookup(torch.zeros(9, 1), i, out=x)
        ops.embedding_lookup(x.resolve_neg(), i)
    with pytest.raises(ValueError, match="negates"):
        ops.preference_loss(lazy[0], None, seq)
    ops.preference_loss(lazy[0].resolve_neg(), None, seq)


def _on_nothing(rc=0):
    """The binding with tensors of this host and a library that only says what it was called for: every launch gives rc."""
    ops = _on_cpu()
    real, ops.called = ops.L, []

    class Library:
        def __getattr__(self, name):
            if name.endswith("_workspace") or name == "mlx_last_error":
                return getattr(real, name)
            return lambda *a: ops.called.append(name) or rc
    ops.L = Library()
    return ops


@pytest.mark.parametrize("rc", [0, -1, -2])
def test_a_tensor_written_in_place_gets_a_new_version(rc):
    """torch's version counter of the caller's `out`, also where it is a view or the logits themselves; a call that was refused wrote nothing."""
    ops = _on_nothing(rc)
    i, f, stats = torch.zeros(5, dtype=torch.int64), torch.zeros(5), torch.zeros(5, 2)
    whole, logits = torch.zeros(5, 9), torch.zeros(5, 6)
    for out, call in ((whole, lambda: ops.embedding_lookup(torch.zeros(4, 6), i, out=whole[:, 1:7])),
                      (whole, lambda: ops.embedding_gradient(torch.zeros(5, 6), i, 5, out=whole[:, :6])),
                      (whole, lambda: ops.embedding_gradient(torch.zeros(5, 6), i, 5, out=whole[:, :6], accumulate=True)),
                      (logits, lambda: ops.token_loglik_gradient(logits, i, stats, f, out=logits)),
                      (logits, lambda: ops.token_loglik_gradient(logits, i, stats, f, out=logits.detach())),
                      (whole, lambda: ops.token_loglik_gradient(logits, i, stats, f, out=whole[:, :6]))):
        before = out._version, stats._version, f._version
        if rc:
            with pytest.raises(RuntimeError, match="mlease_hip error %d" % rc):
                call()
        else:
            call()
        assert (out._version > before[0]) == (rc != -1) and (stats._version, f._version) == before[1:]


def test_preference_results_are_tensors_of_their_own():
    """What comes back can be written in place, by a tensor that requires a gradient too, and kept, whatever happens to the others."""
    ops = _on_nothing()
    f = torch.zeros(1000)
    r = ops.preference_loss(f, None, torch.zeros(2001, dtype=torch.int64))
    assert r.loss.untyped_storage().nbytes() < 64 and r.loss.shape == () and r.grad.untyped_storage().nbytes() == 4000
    w = torch.ones((), requires_grad=True)
    kept = [(x * w).sum() for x in r]                      # (each keeps its factor for w's gradient)
    versions = [x._version for x in r]
    r.loss.div_(8)
    assert [x._version - v for x, v in zip(r, versions)] == [1, 0, 0, 0, 0]
    for k in kept[1:]:
        k.backward()
    for x in r:
        x.mul_(w)
        assert x.requires_grad
    assert ops.preference_loss(f, None, torch.zeros(1, dtype=torch.int64)).ratio.shape == (0,)


@pytest.mark.parametrize("pairs", [0, 1, 2, 3, 7, 8, 16, 63, 64, 100, 255, 256, 512, 1000, 100000, 2 ** 21, 2 ** 29])
def test_preference_workspace_is_bounded_by_the_pairs(pairs):
    L, need = operators.load_operators(), ctypes.c_size_t()
    for each in (0, 1, 4, 5, 64, 65, 8192, 8193, 100000, 2 ** 29):
        n = min(2 ** 31 - 2, 2 * pairs * each)
        assert L.mlx_preference_loss_workspace(n, pairs, ctypes.byref(need)) == 0 and need.value <= 16384 + 8 * pairs


@gpu
def test_an_overwritten_tensor_that_a_graph_kept_is_noticed(ops):
    """A soft cap keeps its result for its backward pass; the gradient written over it must not pass for it."""
    w = torch.randn(7, 50, device="cuda", requires_grad=True)
    target = torch.arange(7, device="cuda")
    logits = torch.tanh(w)
    plain = logits.detach()
    logp, stats = ops.token_loglik(plain, target)
    ops.token_loglik_gradient(plain, target, stats, torch.ones(7, device="cuda"), out=plain)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        logits.sum().backward()


@pytest.mark.skipif(torch.cuda.is_available(), reason="asks what happens without a device")
def test_no_device():
    with pytest.raises(RuntimeError, match="no HIP device"):
        HipOperators()
    ops = _on_cpu()
    with pytest.raises(RuntimeError, match="mlease_hip error -3"):
        ops.embedding_lookup(torch.zeros(4, 6), torch.zeros(5, dtype=torch.int64))


# The HIP runtime's part of a call, as far as the entry points use it: launches are counted and not made, the FAIL-th fails, and the thread's last error
# is what an earlier call of somebody else's left there.
FAKE_RUNTIME = r"""
#include <stdlib.h>
static int launches, last = 700;
int launches_made(void) { return launches; }
void start_again(void) { launches = 0; last = 700; }
int hipGetDevice(int *d) { *d = 0; return 0; }
int hipSetDevice(int d) { (void)d; return 0; }
int hipGetLastError(void) { int e = last; last = 0; return e; }
int hipPeekAtLastError(void) { return last; }
struct d3 { unsigned x, y, z; };
int __hipPushCallConfiguration(struct d3 g, struct d3 b, size_t n, void *s) { (void)g; (void)b; (void)n; (void)s; return 0; }
int __hipPopCallConfiguration(struct d3 *g, struct d3 *b, size_t *n, void **s)
{ struct d3 one = { 1, 1, 1 }; *g = *b = one; *n = 0; *s = 0; return 0; }
int hipLaunchKernel(const void *f, struct d3 g, struct d3 b, void **a, size_t n, void *s)
{
    (void)f; (void)g; (void)b; (void)a; (void)n; (void)s;
    return ++launches == atoi(getenv("FAIL")) ? last = 719 : 0;
}
"""
CALLS_ON_IT = """
import ctypes, json, sys
fake = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
import mlease_amd
from mlease_amd import operators
L = operators.load_operators()
P, need, out = 1 << 30, ctypes.c_size_t(), {}
def call(name, f, *a):
    fake.start_again()
    out[name] = [f(*a), fake.launches_made(), fake.hipPeekAtLastError(), L.mlx_last_error(None).decode()]
call("lookup", L.mlx_embedding_lookup, 0, None, 1, P, 8, 16, 16, 1, 2 * P, 5, 1.0, 3 * P, 16)
L.mlx_embedding_gradient_workspace(300000, 64, 60000, ctypes.byref(need))
call("gradient", L.mlx_embedding_gradient, 0, None, 1, P, 64, 1, 2 * P, 60000, 1.0, 1, 0, 3 * P, 300000, 64, 64, 8 * P, need.value)
L.mlx_token_loglik_workspace(3, 2000000, ctypes.byref(need))
call("loglik", L.mlx_token_loglik, 0, None, 1, P, 3, 2000000, 2000000, 1, 2 * P, 3 * P, 4 * P, 8 * P, need.value)
call("dlogits", L.mlx_token_loglik_gradient, 0, None, 1, P, 3, 100, 100, 1, 2 * P, 3 * P, 4 * P, P, 100)
L.mlx_preference_loss_workspace(100000, 2, ctypes.byref(need))
call("preference", L.mlx_preference_loss, 0, None, P, None, 100000, 2 * P, 2, 0.1, 0.0, 1.0, 0, None, None, None, 3 * P, 4 * P, 5 * P, 6 * P, 7 * P, 8 * P, need.value)
print(json.dumps(out))
"""


@pytest.fixture(scope="module")
def on_fake_runtime(tmp_path_factory):
    d = tmp_path_factory.mktemp("runtime")
    (d / "fake.c").write_text(FAKE_RUNTIME)
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-O1", "-w", "-o", str(d / "fake.so"), str(d / "fake.c")])

    def calls(fail):
        done = subprocess.run([sys.executable, "-c", CALLS_ON_IT, str(d / "fake.so")], cwd=ROOT, env=dict(os.environ, FAIL=str(fail)), capture_output=True, text=True, timeout=300)
        assert done.returncode == 0, done.stderr
        return json.loads(done.stdout)
    return calls


def test_an_error_that_was_there_before_is_not_a_calls(on_fake_runtime):
    """A thread's last error stays until it is read: one that somebody else left is neither reported by a call whose launches all succeeded (its caller
    would make it again, and accumulate twice) nor taken from its owner."""
    for name, (rc, launches, last, _) in on_fake_runtime(0).items():
        assert rc == 0 and last == 700, name
        assert launches == {"lookup": 1, "gradient": 8, "loglik": 2, "dlogits": 1, "preference": 3}[name]


@pytest.mark.parametrize("fail", [1, 2, 3, 5, 7, 8])
def test_nothing_is_launched_behind_a_launch_that_failed(on_fake_runtime, fail):
    """The sums take row numbers from what the sort has written: without the sort they must not run."""
    most = on_fake_runtime(0)
    for name, (rc, launches, last, text) in on_fake_runtime(fail).items():
        if fail > most[name][1]:
            assert rc == 0 and launches == most[name][1]
        else:
            assert rc == -2 and launches == fail and last == 0 and "launch failed" in text, name


# ---------------------------------------------------------------------------------------------- lookup
@pytest.fixture(scope="module")
def ops():
    return HipOperators(0)


def some_ids(g, n, rows, kind, absent=True):
    ids = torch.randint(-1 if absent else 0, rows, (n,), generator=g, device="cuda")
    if absent and n > 3:
        ids[1], ids[2] = rows, -(2 ** 31)
    return ids.to(kind)


def plain_lookup(table, ids, scale):
    here = (ids >= 0) & (ids < table.shape[0])
    rows = (table[ids.clamp(0, table.shape[0] - 1).long()].float() * torch.tensor(scale, dtype=torch.float32, device=table.device)).to(table.dtype)
    return torch.where(here[:, None], rows, torch.zeros_like(rows))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,width", [(1, 1, 1), (1, 50, 4096), (3, 7, 5), (65, 11, 8), (300, 17, 9), (129, 1000, 1001), (70, 33, 256), (1000, 9, 3), (5, 40, 20011), (2049, 300, 64)])
def test_lookup(ops, dtype, n, rows, width):
    g = rng(n + rows)
    table = torch.randn(rows, width, generator=g, device="cuda").to(dtype)
    for kind in (torch.int32, torch.int64):
        ids = some_ids(g, n, rows, kind)
        assert torch.equal(ops.embedding_lookup(table, ids, scale=3.7), plain_lookup(table, ids, 3.7))      # one product and one rounding: the same bits
    assert torch.equal(ops.embedding_lookup(table, ids), plain_lookup(table, ids, 1.0))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_lookup_strides_and_alignment(ops, dtype):
    g = rng(5)
    whole = torch.randn(40, 77, generator=g, device="cuda").to(dtype)
    ids = some_ids(g, 90, 40, torch.int64)
    for first in range(5):
        table = whole[:, first:first + 70]
        into = torch.full((90, 80), 9.0, device="cuda", dtype=dtype)
        out = ops.embedding_lookup(table, ids, scale=0.5, out=into[:, 3 + first:73 + first])
        assert out.data_ptr() == into[:, 3 + first:].data_ptr()
        want = torch.full_like(into, 9.0)
        want[:, 3 + first:73 + first] = plain_lookup(table, ids, 0.5)
        assert torch.equal(into, want)                                           # nothing beside the rows is written
    one = whole[:1].expand(40, 77)                                               # a table of one row, repeated
    assert torch.equal(ops.embedding_lookup(one, ids), plain_lookup(one, ids, 1.0))


@gpu
def test_lookup_special_values_and_nothing(ops):
    t = torch.tensor([[math.inf, -math.inf, math.nan, 0.0, -0.0, 3e38]], device="cuda")
    ids = torch.tensor([0, -1, 1, 0], device="cuda")
    out = ops.embedding_lookup(t, ids, scale=2.0)
    assert torch.equal(out.isnan(), torch.tensor([[False, False, True] + 3 * [False], 6 * [False], 6 * [False], [False, False, True] + 3 * [False]], device="cuda"))
    assert torch.equal(out.nan_to_num(7.0, posinf=5.0, neginf=-5.0)[0], torch.tensor([5.0, -5.0, 7.0, 0.0, 0.0, 5.0], device="cuda"))
    assert not out[1:3].any()
    assert ops.embedding_lookup(t, ids[:0]).shape == (0, 6)
    assert not ops.embedding_lookup(t[:0], ids).any()                            # an empty table: every id is absent
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.embedding_lookup(t, ids[:1], out=t)
    with pytest.raises(RuntimeError, match="ld of out"):
        ops.embedding_lookup(t, ids, out=torch.empty(6, device="cuda").expand(4, 6))


# ---------------------------------------------------------------------------------------------- gradient of the lookup
def check_gradient(got, grad_out, ids, rows, scale, before=None):
    """Against 64 bits. c terms of an id are summed in 32 bits: at most c + 1 additions (the sum being added to included) and the
    product with the scale, each off by u of at most the sum of the terms' sizes; then the result's rounding."""
    x, i = grad_out.double(), ids.long()
    here = (i >= 0) & (i < rows)
    at = torch.where(here, i, torch.full_like(i, rows))
    want = torch.zeros(rows + 1, x.shape[1], dtype=torch.float64, device=x.device).index_add_(0, at, x)[:rows] * scale
    size = torch.zeros_like(torch.empty(rows + 1, x.shape[1]), dtype=torch.float64, device=x.device).index_add_(0, at, x.abs())[:rows] * abs(scale)
    count = torch.zeros(rows + 1, dtype=torch.float64, device=x.device).index_add_(0, at, torch.ones_like(at, dtype=torch.float64))[:rows, None]
    if before is not None:
        want, size = want + before.double(), size + before.double().abs()
    within(got, want, (count + 3) * U * size + half_step(want, got.dtype) * (1 + 1e-6))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,width", [(1, 1, 1), (1, 300, 64), (31, 5, 7), (32, 70000, 3), (33, 2, 130), (64, 1, 65), (1000, 17, 9), (2048, 256, 8), (2049, 257, 33), (5000, 65537, 1),
                                          (700, 900, 1001), (20000, 3, 20), (100, 4, 9000), (17000, 40000, 64), (66000, 1000, 8),
                                          (4096, 511, 4), (4097, 512, 4), (9000, 513, 6), (9000, 262143, 2), (5000, 262144, 3), (300000, 5000, 4), (262145, 300000, 1),
                                          (5000, 900, 2051), (4500, 9000, 2048), (4500, 9001, 2055), (4097, 8194, 2300)])
def test_gradient(ops, dtype, n, rows, width):
    g = rng(n + width)
    go = torch.randn(n, width, generator=g, device="cuda").to(dtype)
    for kind in (torch.int32, torch.int64):
        ids = some_ids(g, n, rows, kind)
        got = ops.embedding_gradient(go, ids, rows, scale=1.25)
        assert got.dtype == dtype and torch.equal(got, ops.embedding_gradient(go, ids, rows, scale=1.25))       # the same inputs, the same bits
        check_gradient(got, go, ids, rows, 1.25)
    got = ops.embedding_gradient(go, ids, rows, dtype=torch.float32)
    check_gradient(got, go, ids, rows, 1.0)
    acc = torch.randn(rows, width, generator=g, device="cuda")
    for start in (acc, acc.to(dtype)):
        out = start.clone()
        ops.embedding_gradient(go, ids, rows, scale=-0.5, out=out, accumulate=True)
        check_gradient(out, go, ids, rows, -0.5, before=start)
        used = torch.zeros(rows + 1, dtype=torch.bool, device="cuda")
        used[torch.where((ids >= 0) & (ids < rows), ids, torch.full_like(ids, rows)).long()] = True
        assert torch.equal(out[~used[:rows]], start[~used[:rows]])                # rows without an id are not touched


def test_gradient_marks_its_rows_by_their_bytes():
    """The workspace told is enough for every pair of types: a mark a row from 4096 bytes of a float32 row on, where entries are half of the rows."""
    def needs(n, rows, width):
        need = ctypes.c_size_t()
        assert operators.load_operators().mlx_embedding_gradient_workspace(rows, width, n, ctypes.byref(need)) == 0
        return need.value
    assert needs(5000, 10000, 1024) - needs(5000, 10000, 1023) >= 4 * 10000
    assert needs(5000, 10002, 1024) == needs(5000, 10002, 1023) and needs(4096, 100, 1024) == needs(4096, 100, 1023)


@gpu
@pytest.mark.parametrize("dtype,grad_type", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float32)])
@pytest.mark.parametrize("n,rows,width", [(5000, 9000, 1023), (5000, 9000, 1024), (5000, 10002, 1024), (5000, 6000, 1031), (9000, 700, 2047), (5000, 9000, 2048), (5000, 9001, 2060)])
def test_gradient_around_the_rule_of_marked_rows(ops, dtype, grad_type, n, rows, width):
    g = rng(width + rows)
    go, ids = torch.randn(n, width, generator=g, device="cuda").to(dtype), some_ids(g, n, rows, torch.int64)
    got = torch.full((rows, width + 1), 9.0, device="cuda", dtype=grad_type)
    ops.embedding_gradient(go, ids, rows, out=got[:, :width])
    check_gradient(got[:, :width], go, ids, rows, 1.0)
    assert (got[:, width] == 9).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,width", [(40, 70), (4096, 24), (30000, 12), (30000, 260), (2100, 520)])
def test_gradient_of_one_id_and_of_none(ops, dtype, n, width):
    """Every entry the same id (one sum over all pieces), every entry absent, two ids that alternate, ids in descending order."""
    g = rng(n)
    go = torch.randn(n, width, generator=g, device="cuda").to(dtype)
    k = torch.arange(n, device="cuda")
    for ids in (torch.full((n,), 3, device="cuda"), torch.full((n,), -1, device="cuda"), 2 + 3 * (k % 2), (n - 1 - k), torch.where(k < n // 2, 0, 6)):
        check_gradient(ops.embedding_gradient(go, ids, 7, scale=2.0), go, ids, 7, 2.0)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,rows,width", [(2, 9000, 1), (63, 4097, 7), (64, 1000, 9), (65, 129, 64), (127, 300, 200), (129, 65, 520), (255, 40, 12), (256, 8192, 3), (257, 31, 8),
                                          (400, 700, 130), (511, 33, 512), (512, 12289, 2), (512, 500, 24), (512, 20, 2048), (7, 3, 40001), (300, 2049, 33)])
def test_gradient_of_few_entries(ops, dtype, n, rows, width):
    """Without the sort: ids all over the rows, of a few rows, of one, of the first and last row, ascending; strided, accumulated, with and without absent ones."""
    g = rng(n * 7 + width)
    whole = torch.randn(n, width + 3, generator=g, device="cuda").to(dtype)
    go, k = whole[:, 1:width + 1], torch.arange(n, device="cuda")
    for ids in (some_ids(g, n, rows, torch.int64), torch.randint(0, min(rows, 3), (n,), generator=g, device="cuda"), torch.full((n,), rows - 1, device="cuda"),
                (rows - 1) * (k % 2), k % rows, torch.where(k < n - 1, -1, rows // 2).int()):
        into = torch.full((rows, width + 5), 9.0, device="cuda", dtype=dtype)
        check_gradient(ops.embedding_gradient(go, ids, rows, scale=0.75, out=into[:, 2:width + 2]), go, ids, rows, 0.75)
        assert (into[:, :2] == 9).all() and (into[:, width + 2:] == 9).all()
        start = torch.randn(rows, width, generator=g, device="cuda")
        out = start.clone()
        ops.embedding_gradient(go, ids, rows, out=out, accumulate=True)
        check_gradient(out, go, ids, rows, 1.0, before=start)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_strides_and_alignment(ops, dtype):
    g = rng(6)
    whole = torch.randn(200, 90, generator=g, device="cuda").to(dtype)
    ids = some_ids(g, 200, 30, torch.int32)
    for first in range(4):
        go = whole[:, first:first + 77]
        into = torch.full((30, 85), 9.0, device="cuda", dtype=dtype)
        out = ops.embedding_gradient(go, ids, 30, out=into[:, first + 1:first + 78])
        check_gradient(out, go, ids, 30, 1.0)
        assert (into[:, :first + 1] == 9).all() and (into[:, first + 78:] == 9).all()
    wide = torch.randn(5000, 2100, generator=g, device="cuda").to(dtype)        # many entries of wide rows: rows with an id are spared the zeros
    many = some_ids(g, 5000, 3000, torch.int64)
    into = torch.full((3000, 2110), 9.0, device="cuda", dtype=dtype)
    check_gradient(ops.embedding_gradient(wide[:, 1:2090], many, 3000, out=into[:, 3:2092]), wide[:, 1:2090], many, 3000, 1.0)
    assert (into[:, :3] == 9).all() and (into[:, 2092:] == 9).all()
    same = whole[:1, :40].expand(200, 40)                                        # the gradient of a broadcast: one row for all entries
    check_gradient(ops.embedding_gradient(same, ids, 30), same, ids, 30, 1.0)


@gpu
def test_gradient_special_values_and_nothing(ops):
    go = torch.tensor([[1.0, math.inf], [math.nan, 2.0], [5.0, 6.0]], device="cuda")
    out = ops.embedding_gradient(go, torch.tensor([1, -1, 1], device="cuda"), 3)         # a NaN in an absent entry's row is not looked at
    assert torch.equal(out, torch.tensor([[0, 0], [6, math.inf], [0, 0]], device="cuda"))
    assert not ops.embedding_gradient(go[:0], torch.empty(0, dtype=torch.int32, device="cuda"), 3).any()
    assert ops.embedding_gradient(go, torch.tensor([1, -1, 1], device="cuda"), 0).shape == (0, 2)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.embedding_gradient(go, torch.tensor([1, -1, 1], device="cuda"), 3, out=go)


@gpu
def test_gradient_is_the_lookups_adjoint(ops):
    """<grad_out, lookup(E)> = <gradient(grad_out), E> for any E: the lookup is linear, its differences are exact. Whole numbers of few
    digits: every product and sum below is exact."""
    g = rng(9)
    go = torch.randint(-8, 9, (500, 24), generator=g, device="cuda").float()
    e = torch.randint(-8, 9, (60, 24), generator=g, device="cuda").float()
    ids = some_ids(g, 500, 60, torch.int64)
    a = (go.double() * ops.embedding_lookup(e, ids, scale=2.0).double()).sum()
    b = (ops.embedding_gradient(go, ids, 60, scale=2.0).double() * e.double()).sum()
    assert a == b


# ---------------------------------------------------------------------------------------------- log-likelihood
def exact_loglik(logits, target):
    """logp in 64 bits (0 where absent, -infinity for a row of nothing but -infinity), softmax, and a bound on the kernel's error in
    log p: with t = x - max, each term exp(t) is off by u (|t| for the difference, 2 |t| for its product with log2 e, 2 for exp2), the sum
    by u for each of a lane's additions and rescalings (at most 2 per element and 64 lanes share a row at least) and 64 more of joining."""
    x = logits.double()
    here = (target >= 0) & (target < x.shape[1])
    top = x.amax(1, keepdim=True)
    t = x - torch.where(top == -math.inf, torch.zeros_like(top), top)
    s = t.exp().sum(1, keepdim=True)
    p = torch.where(s > 0, t.exp() / s, torch.zeros_like(t))
    mean_t = (p * torch.where(p > 0, t.abs(), torch.zeros_like(t))).sum(1)
    logp = (t - s.log()).gather(1, target.long().clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    logp = torch.where(here, torch.where(top[:, 0] == -math.inf, torch.full_like(logp, -math.inf), logp), torch.zeros_like(logp))
    err = U * (3 * mean_t + 2 + 2 * math.ceil(x.shape[1] / 64) + 64)
    return logp, p, t, s.log(), err, here


def check_loglik(ops, logits, target, g=None, out=None):
    logp, p, t, log_s, err, here = exact_loglik(logits, target)
    got, stats = ops.token_loglik(logits, target)
    fine = torch.isfinite(logp)
    assert torch.equal(got[~fine].double(), logp[~fine])
    within(got[fine], logp[fine], (err + half_step(logp, torch.float32))[fine])
    if g is None:
        return got, stats
    # log p of every class: u for the difference t, the constant and the fma of its product; u for the stored logarithm, its constant, its
    # product and the fma; exp2 2 u
    delta = err[:, None] + U * (3 * t.abs().nan_to_num(0, posinf=0) + 4 * log_s.abs().nan_to_num(0, posinf=0) + 2)
    hit = torch.arange(logits.shape[1], device="cuda")[None, :] == target[:, None]
    lp = torch.where(p > 0, t - log_s, torch.full_like(t, -math.inf))
    want = torch.where(hit, -torch.expm1(lp), -p)
    some = here & (g != 0) & (logits.double().amax(1) > -math.inf)
    size = torch.where(some, g.double().abs(), torch.zeros_like(g.double()))[:, None]
    want = torch.where(some[:, None], g.double()[:, None] * want, torch.zeros_like(want))
    # the slope of exp and of expm1 is p; expm1 is off by 2 steps (4 u) of its value; exp2 of less than -126 gives 0: 2^-126 at most is lost
    tol = size * (1.01 * p * delta + 2.0 ** -126) + 5 * U * want.abs() + half_step(want, logits.dtype) * (1 + 1e-6)
    d = ops.token_loglik_gradient(logits, target, stats, g, out=out)
    within(d, want, tol)
    return got, stats


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,classes", [(1, 1), (1, 2), (5, 7), (3, 8), (17, 9), (4, 255), (2, 2048), (9, 2051), (1, 50021), (3, 131072), (300, 100), (6, 32000), (70, 4097), (2000, 33), (1, 300007), (2, 700001), (40, 20000), (300, 500), (300, 900)])
def test_loglik(ops, dtype, n, classes):
    g = rng(n + classes)
    logits = (4 * torch.randn(n, classes, generator=g, device="cuda")).to(dtype)
    for kind in (torch.int32, torch.int64):
        target = some_ids(g, n, classes, kind, absent=n > 4)
        w = torch.randn(n, generator=g, device="cuda")
        if n > 5:
            w[5] = 0
        check_loglik(ops, logits, target, w)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_loglik_strides_alignment_and_place(ops, dtype):
    g = rng(3)
    whole = torch.randn(12, 3100, generator=g, device="cuda").to(dtype)
    target = some_ids(g, 12, 3001, torch.int64)
    w = torch.randn(12, generator=g, device="cuda")
    for first in range(9):
        check_loglik(ops, whole[:, first:first + 3001], target, w)
    into = torch.full((12, 3050), 9.0, device="cuda", dtype=dtype)
    check_loglik(ops, whole[:, 5:3006], target, w, out=into[:, 3:3004])
    assert (into[:, :3] == 9).all() and (into[:, 3004:] == 9).all()
    one = whole[:1].expand(12, 3100)                                             # one row for all tokens
    check_loglik(ops, one, target, w)
    # in place: the same bits as beside it, and the columns behind the classes are left
    logits = whole[:, 1:3002]
    logp, stats = ops.token_loglik(logits, target)
    want, rest = ops.token_loglik_gradient(logits, target, stats, w), whole[:, 3002:].clone()
    got = ops.token_loglik_gradient(logits, target, stats, w, out=logits)
    assert torch.equal(got, want) and got.data_ptr() == logits.data_ptr() and torch.equal(whole[:, 3002:], rest)
    with pytest.raises(RuntimeError, match="overlaps logits"):
        ops.token_loglik_gradient(whole[:, :3000], target, stats, w, out=whole[:, 1:3001])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [5, 3001, 40000])
def test_loglik_masks_and_special_values(ops, dtype, classes):
    g = rng(classes)
    x = torch.randn(10, classes, generator=g, device="cuda").to(dtype)
    target = torch.arange(10, device="cuda") % 5
    low = torch.finfo(dtype).min
    x[0, 1:] = -math.inf                    # one class is left, and is the target: logp 0
    x[1] = -math.inf                        # nothing is left
    x[2, 2] = -math.inf                     # the target itself is excluded
    x[3, :2] = low                          # masked with the type's lowest value
    x[4] = low                              # ... all of them: uniform
    x[5] += 300 if dtype != torch.float16 else 60000
    x[6] = 0
    x[7, 2] = low
    x[7, 3:] = -math.inf
    w = torch.randn(10, generator=g, device="cuda")
    got, stats = check_loglik(ops, x, target, w)
    assert got[0] == 0 and got[1] == -math.inf and got[2] == -math.inf
    d = ops.token_loglik_gradient(x, target, stats, w)
    assert not d[0].any() and not d[1].any() and torch.isfinite(d).all()
    # NaN and +infinity make the row's values NaN; in a row that does not count they are not looked at
    y = x[:4].clone()
    y[0, 3] = math.nan
    y[1, 0] = math.inf
    y[2, 1] = math.nan
    y[3, 4] = math.nan
    t = torch.tensor([0, 1, -1, 2], device="cuda")
    g4 = torch.tensor([1.0, 1.0, 1.0, 0.0], device="cuda")
    got, stats = ops.token_loglik(y, t)
    assert got[0].isnan() and got[1].isnan() and got[2] == 0 and got[3].isnan()
    d = ops.token_loglik_gradient(y, t, stats, g4)
    assert d[0].isnan().all() and d[1].isnan().any() and not d[2:].any()
    # all rows NaN: still NaN
    nan = torch.full((1, classes), math.nan, device="cuda", dtype=dtype)
    got, stats = ops.token_loglik(nan, t[:1])
    assert got.isnan().all() and ops.token_loglik_gradient(nan, t[:1], stats, g4[:1]).isnan().all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [2, 4, 100, 3001, 32000, 200001])
def test_loglik_of_likely_targets(ops, dtype, classes):
    """Targets nearly certain: log p = -log(1 + R) keeps its digits, R being the others' sum. R is off by what any sum of exponentials is (as in
    exact_loglik, relative to the others' maximum) and by its rescaling to the target's logit."""
    g = rng(classes)
    x = torch.randn(12, classes, generator=g, device="cuda")
    target = torch.randint(0, classes, (12,), generator=g, device="cuda")
    rows = torch.arange(12, device="cuda")
    x[rows, target] = torch.linspace(4, 40, 12, device="cuda")
    x = x.to(dtype)
    v, at = x.double(), target[:, None]
    value = v.gather(1, at)
    others = v.scatter(1, at, -math.inf)
    top = others.amax(1, keepdim=True)
    e = (others - top).exp()
    mean_t = torch.where(e > 0, e * (others - top).abs(), 0.0).sum(1) / e.sum(1)
    R = (e.sum(1, keepdim=True) * (top - value).exp())[:, 0]
    want = -R.log1p()
    err = U * (3 * mean_t + 2 + 2 * math.ceil(classes / 64) + 64 + 3 * (top - value).abs()[:, 0] + 3)
    got, stats = ops.token_loglik(x, target)
    within(got, want, R / (1 + R) * err * 1.01 + half_step(want, torch.float32) * (1 + 1e-6) + 2.0 ** -126)
    d = ops.token_loglik_gradient(x, target, stats, torch.ones(12, device="cuda")).double().gather(1, at)[:, 0]
    p_not = -torch.expm1(want)
    within(d, p_not, p_not * (err * 1.01 + 8 * U) + half_step(p_not, dtype) * (1 + 1e-6) + 2.0 ** -126)


ONE_PART = 1.0 - 1.44269502162933 / 1.4426950408889634        # what log2 e as one 32-bit number lacks: 1.33e-8
MEAN_LOSS = 3.4e-9                                             # of a v_exp_f32, on average


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_loglik_of_targets_far_above(ops, dtype):
    """Two classes: log p = -log(1 + exp(-d)) with the digits of the one exponential that it is made of. That is off by 2 u (v_exp_f32: one step) and
    0.18 u (its argument of at most 1/2, rounded), the mean loss that is put back by 0.06 u, the logarithm by nothing, and the result is rounded: u."""
    g = rng(31)
    n = 100000
    x = torch.randn(n, 2, generator=g, device="cuda")
    target = torch.randint(0, 2, (n,), generator=g, device="cuda")
    x[torch.arange(n, device="cuda"), target] = torch.rand(n, generator=g, device="cuda") * 72 + 5
    x = x.to(dtype)
    v = x.double().gather(1, target[:, None])[:, 0] - x.double().gather(1, 1 - target[:, None])[:, 0]
    want = -torch.log1p(torch.exp(-v))
    got, stats = ops.token_loglik(x, target)
    within(got, want, want.abs() * 3.25 * U)
    within(stats[:, 1], -want, want.abs() * 3.25 * U)


@gpu
def test_loglik_has_no_bias_of_one_exponential(ops):
    """The mean of the relative error over 200000 rows of two classes, targets 1 to 12 above: 3.6e-8 rms (v_exp_f32 2.6e-8, rounding 2.5e-8) leave 8e-11;
    half the mean loss is allowed, so that its correction left out, or of the wrong sign, is seen."""
    g = rng(32)
    x = torch.zeros(200000, 2, device="cuda")
    x[:, 0] = torch.rand(200000, generator=g, device="cuda") * 11 + 1
    want = -torch.log1p(torch.exp(-x[:, 0].double()))
    off = ops.token_loglik(x, torch.zeros(200000, dtype=torch.int64, device="cuda"))[0].double() / want - 1
    assert off.pow(2).mean().sqrt() < 5e-8
    assert abs(off.mean()) < MEAN_LOSS / 2 < abs(off.mean() - MEAN_LOSS)


@gpu
@pytest.mark.parametrize("dtype,n,classes", [(torch.bfloat16, 8192, 32000), (torch.float32, 8192, 32000), (torch.bfloat16, 4096, 128000), (torch.float16, 4000, 200003)])
def test_loglik_sums_have_no_bias(ops, dtype, n, classes):
    """Likely targets of many classes, log p = -log(1 + R): relative errors of R are those of the others' sum. On average over thousands of rows they are off by
    two exponentials' mean loss at most (a term's own, its lane's rescaling and the joining of lanes, one of them put back: 7e-9), and, 16-bit logits near
    the maximum being a few dozen values, by the error of v_exp_f32 over those (2.6e-8 / sqrt(50)): 2e-8 are allowed. log2 e in one part is off by 1.33e-8
    of the mean distance to the maximum, more than twice that. The rms is that of a rounding, of v_exp_f32 and of the lanes' sums: u."""
    g = rng(classes)
    off, one_part = [], []
    for a in range(0, n, 512):
        x = torch.randn(min(512, n - a), classes, generator=g, device="cuda").mul_(2)
        x[:, 7] = -1e4
        x[:, 7] = torch.logsumexp(x, 1) + 6
        x = x.to(dtype)
        got = ops.token_loglik(x, torch.full((x.shape[0],), 7, device="cuda"))[0].double()
        for b in range(0, x.shape[0], 128):
            v = x[b:b + 128].double()
            value = v[:, 7:8].clone()
            v[:, 7] = -math.inf
            top = v.amax(1, keepdim=True)
            e = (v - top).exp()
            mean_t = torch.where(e > 0, e * (top - v), 0.0).sum(1) / e.sum(1)
            R = e.sum(1) * (top - value)[:, 0].exp()
            off.append(got[b:b + 128] / -torch.log1p(R) - 1)
            one_part.append(got[b:b + 128] / -torch.log1p(R * (1 + ONE_PART * mean_t)) - 1)       # (smaller |t| in the exponent: larger terms)
    off, one_part = torch.cat(off), torch.cat(one_part)
    assert off.pow(2).mean().sqrt() < U
    assert abs(off.mean()) < 2e-8 < abs(one_part.mean())


@gpu
@pytest.mark.parametrize("spread", [1.0, 2.0])
def test_loglik_gradient_has_no_bias(ops, spread):
    """What the gradient gives to all classes but the target is -(1 - p) of it on average: the stored logarithm's rounding (half a step of 4 to 16 at most, 2.8e-7
    rms) over 8192 rows leaves 3e-9, four times that and the mean loss of the exponentials are allowed; log2 e in one part is off by 1.33e-8 of the mean
    logarithm of 1 / p, more than twice as much."""
    g = rng(34)
    n, classes = 8192, 5000
    off, log_p = [], []
    for a in range(0, n, 1024):
        x = torch.randn(1024, classes, generator=g, device="cuda").mul_(spread)
        target = torch.randint(0, classes, (1024,), generator=g, device="cuda")
        _, stats = ops.token_loglik(x, target)
        d = ops.token_loglik_gradient(x, target, stats, torch.ones(1024, device="cuda")).double()
        p = x.double().softmax(1)
        log_p.append((p * p.log()).sum(1))
        d.scatter_(1, target[:, None], 0.0)
        p.scatter_(1, target[:, None], 0.0)
        off.append(-d.sum(1) / p.sum(1) - 1)
    bound = 4 * 2.8e-7 / math.sqrt(n) + MEAN_LOSS
    assert abs(torch.cat(off).mean()) < bound < -float(torch.cat(log_p).mean()) * ONE_PART / 2


@gpu
def test_margin_of_a_long_answer(ops):
    """One answer of 39000 tokens against one of 1000, from their logits, under a reference model that is near: the margin adds up the errors of 40000 log p. The
    roundings add like a random walk (4 of its deviations allowed), and what every row's sum has alike, 2e-8 at most, by the difference of the lengths."""
    g = rng(33)
    n, classes, beta = 40000, 4000, 0.125
    x = torch.randn(n, classes, generator=g, device="cuda").mul_(2).to(torch.bfloat16)
    target = torch.randint(0, classes, (n,), generator=g, device="cuda")
    logp, _ = ops.token_loglik(x, target)
    want, mean_t = torch.empty(n, dtype=torch.float64, device="cuda"), torch.empty(n, dtype=torch.float64, device="cuda")
    for a in range(0, n, 4000):
        v, at = x[a:a + 4000].double(), target[a:a + 4000, None]
        want[a:a + 4000] = (v.gather(1, at) - v.logsumexp(1, keepdim=True))[:, 0]
        p = v.softmax(1)
        mean_t[a:a + 4000] = (p * (v.amax(1, keepdim=True) - v)).sum(1)
    ref = (want + 0.1 * torch.randn(n, generator=g, device="cuda")).float()
    seq = torch.tensor([0, 39000, 40000], device="cuda")
    margin = float(ops.preference_loss(logp, ref, seq, beta=beta).margin)
    sign = torch.where(torch.arange(n, device="cuda") < 39000, 1.0, -1.0).double()
    exact = beta * float(((want - ref.double()) * sign).sum())
    allowed = beta * (4 * math.sqrt(n / 3) * float(half_step(want, torch.float32).pow(2).mean().sqrt()) + 38000 * 2e-8) + abs(exact) * U
    assert abs(margin - exact) <= allowed
    assert beta * ONE_PART * float((mean_t * sign).sum()) > allowed          # what log2 e in one part would add


@gpu
def test_loglik_of_nothing(ops):
    x = torch.zeros(0, 9, device="cuda")
    logp, stats = ops.token_loglik(x, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert logp.shape == (0,) and stats.shape == (0, 2)
    assert ops.token_loglik_gradient(x, torch.empty(0, dtype=torch.int64, device="cuda"), stats, logp).shape == (0, 9)


@gpu
@pytest.mark.parametrize("classes", [6, 1500])
def test_loglik_gradient_is_the_difference_quotient(ops, classes):
    """Central differences of logp in one logit, step d = 1/16: off by at most d^2 / 6 times the third derivative (below 1/6 in size for any
    p), and by the error of the two logp over 2 d."""
    g = rng(classes)
    x = torch.randn(4, classes, generator=g, device="cuda")
    target = torch.tensor([0, 1, 2, 3], device="cuda")
    logp, stats = ops.token_loglik(x, target)
    d = ops.token_loglik_gradient(x, target, stats, torch.ones(4, device="cuda"))
    for j in (0, 1, 2, 3, 5):
        h = 1 / 16
        up, down = x.clone(), x.clone()
        up[:, j] += h
        down[:, j] -= h
        q = (ops.token_loglik(up, target)[0].double() - ops.token_loglik(down, target)[0].double()) / ((up[:, j].double() - down[:, j].double()))
        err = exact_loglik(up, target)[4] + exact_loglik(down, target)[4] + 2 * half_step(logp.double().abs() + 1, torch.float32)
        within(d[:, j], q, h * h / 36 + err / (2 * h) + 1e-6)


@gpu
@pytest.mark.parametrize("dtype,n,classes", [(torch.bfloat16, 171, 160009), (torch.float32, 170, 160009), (torch.float16, 129, 160000), (torch.bfloat16, 511, 160001)])
def test_loglik_of_long_rows(ops, dtype, n, classes):
    """On both sides of the rule that cuts rows into parts: of 160000 classes and more, up to 170 rows and more than that."""
    need = ctypes.c_size_t()
    ops._ck(ops.L.mlx_token_loglik_workspace(n, classes, ctypes.byref(need)))
    assert (need.value > 0) == (n <= 170 and classes > 160000)
    g = rng(n)
    logits = (4 * torch.randn(n, classes, generator=g, device="cuda")).to(dtype)
    check_loglik(ops, logits, some_ids(g, n, classes, torch.int64))


# ---------------------------------------------------------------------------------------------- matrices beyond the memory-side cache
BEYOND = 256 << 20          # bytes from which on results are written past the caches


@gpu
@pytest.mark.parametrize("dtype,n,width", [(torch.float32, 33000, 2048), (torch.bfloat16, 40000, 3501), (torch.float16, 33001, 4097), (torch.float32, 5000011, 14), (torch.float32, 22400001, 3),
                                           (torch.bfloat16, 19300000, 7), (torch.float16, 16800000, 8)])
def test_lookup_beyond_the_cache(ops, dtype, n, width):
    assert n * width * dtype.itemsize > BEYOND
    g = rng(width)
    table = torch.randn(5003, width, generator=g, device="cuda").to(dtype)
    ids = some_ids(g, n, 5003, torch.int32)
    got, want = ops.embedding_lookup(table, ids, scale=1.7), plain_lookup(table, ids, 1.7)
    assert torch.equal(got, want)
    into = torch.full((n, width + 1), 9.0, device="cuda", dtype=dtype)
    ops.embedding_lookup(table, ids, scale=1.7, out=into[:, :width])
    assert torch.equal(into[:, :width], want) and (into[:, width] == 9).all()


@gpu
@pytest.mark.parametrize("dtype,grad_type", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
@pytest.mark.parametrize("n,width", [(1, 2049), (500, 2049), (3000, 2049), (5000, 1030), (70000, 2049), (300, 5), (9000, 3)])
def test_gradient_beyond_the_cache(ops, dtype, grad_type, n, width):
    """One launch, the sort in one workgroup and in many, rows with an id spared the zeros and not, one slot a row and many."""
    rows = BEYOND // (width * grad_type.itemsize) + 1000
    g = rng(n)
    go = torch.randn(n, width, generator=g, device="cuda").to(dtype)
    ids = torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, torch.randint(0, rows, (n,), generator=g, device="cuda"), torch.randint(rows - 50, rows + 3, (n,), generator=g, device="cuda"))
    got = ops.embedding_gradient(go, ids, rows, scale=1.5, dtype=grad_type)
    start = torch.randn(rows, 1, generator=g, device="cuda").to(grad_type).expand(rows, width).contiguous()
    out = start.clone()
    ops.embedding_gradient(go, ids, rows, scale=1.5, out=out, accumulate=True)
    used = torch.unique(ids[ids < rows])
    at = torch.where(ids < rows, torch.searchsorted(used, ids), torch.full_like(ids, -1))      # (in 64 bits the rows that have an id only)
    check_gradient(got[used], go, at, used.numel(), 1.5)
    check_gradient(out[used], go, at, used.numel(), 1.5, before=start[used])
    got[used] = 0
    assert not got.any()
    out[used] = start[used]
    assert torch.equal(out, start)


@gpu
@pytest.mark.parametrize("dtype,n", [(torch.float32, 700), (torch.float16, 1400), (torch.bfloat16, 1400)])
@pytest.mark.parametrize("classes", [50021, 50024])
def test_loglik_gradient_beyond_the_cache(ops, dtype, n, classes):
    assert 2 * n * classes * dtype.itemsize > BEYOND
    g = rng(n + classes)
    logits = (4 * torch.randn(n, classes, generator=g, device="cuda")).to(dtype)
    target = some_ids(g, n, classes, torch.int64)
    w = torch.randn(n, generator=g, device="cuda")
    w[5] = 0
    logp, stats = check_loglik(ops, logits, target, w)
    want = ops.token_loglik_gradient(logits, target, stats, w)
    assert torch.equal(ops.token_loglik_gradient(logits, target, stats, w, out=logits), want) and torch.equal(logits, want)


# ---------------------------------------------------------------------------------------------- preference
def exact_preference(logp, ref, seq_ptr, beta, smoothing, scale, mask, weight, offset, mean):
    """In 64 bits on the host, a loop over the sequences."""
    n, seq = logp.numel(), [int(v) for v in seq_ptr.cpu()]
    pairs = (len(seq) - 1) // 2
    x = logp.double().cpu() - (ref.double().cpu() if ref is not None else 0)
    on = mask.bool().cpu() if mask is not None else torch.ones(n, dtype=torch.bool)
    ratio, part = torch.zeros(2 * pairs, dtype=torch.float64), torch.ones(2 * pairs, dtype=torch.float64)
    for s in range(2 * pairs):
        v = x[seq[s]:seq[s + 1]][on[seq[s]:seq[s + 1]]]
        if mean:
            part[s] = 1.0 / len(v) if len(v) else 0.0
        ratio[s] = v.sum() * part[s] if len(v) else 0.0
    beta, scale, smoothing = (float(np.float32(v)) for v in (beta, scale, smoothing))
    h = beta * (ratio[:pairs] - ratio[pairs:]) + (offset.double().cpu() if offset is not None else 0.0)
    w = scale * (weight.double().cpu() if weight is not None else torch.ones(pairs, dtype=torch.float64))

    def sp(v):
        return v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))

    loss = torch.zeros_like(h)
    if smoothing < 1:
        loss = loss + (1 - smoothing) * sp(-h)
    if smoothing > 0:
        loss = loss + smoothing * sp(h)
    slope = torch.where(w == 0, torch.zeros_like(w), w * beta * (smoothing * torch.sigmoid(h) - (1 - smoothing) * torch.sigmoid(-h)))
    grad = torch.zeros(n, dtype=torch.float64)
    for s in range(2 * pairs):
        grad[seq[s]:seq[s + 1]] = torch.where(on[seq[s]:seq[s + 1]], (slope[s] if s < pairs else -slope[s - pairs]) * part[s], torch.zeros((), dtype=torch.float64))
    return torch.where(w == 0, torch.zeros_like(w), w * loss).sum(), loss, h, ratio, grad


def check_preference(ops, logp, ref, seq_ptr, beta=0.1, smoothing=0.0, scale=1.0, mask=None, weight=None, offset=None, mean=False):
    """Sums of n terms are in 64 bits (n 2^-53 of their sizes); what comes out is rounded to 32 bits once, the total loss from pair losses
    that were rounded once before."""
    r = ops.preference_loss(logp, ref, seq_ptr, beta=beta, smoothing=smoothing, scale=scale, mask=mask, weight=weight, offset=offset, mean=mean)
    want = exact_preference(logp, ref, seq_ptr, beta, smoothing, scale, mask, weight, offset, mean)
    n = logp.numel()
    size = float((logp.double().abs().nan_to_num(0, 0, 0).sum() + (0 if ref is None else ref.double().abs().nan_to_num(0, 0, 0).sum())))
    slack = (n + 8) * 2.0 ** -52 * size
    f32 = torch.float32
    for got, w, extra in ((r.pair_loss, want[1], beta * slack), (r.margin, want[2], beta * slack), (r.ratio, want[3], slack)):
        inf = torch.isinf(w)
        assert torch.equal(got.cpu()[inf].double(), w[inf])
        within(got.cpu()[~inf], w[~inf], half_step(w[~inf], f32) * (1 + 1e-6) + extra + w[~inf].abs() * 2.0 ** -50)
    within(r.grad, want[4], half_step(want[4], f32) * (1 + 1e-6) + want[4].abs() * (abs(beta) * slack + 2.0 ** -50))
    pairs = want[1].numel()
    if torch.isfinite(want[0]):
        w = scale * (weight.double().cpu() if weight is not None else torch.ones(pairs, dtype=torch.float64))
        terms = torch.where(w == 0, torch.zeros_like(w), (w * want[1]).abs()).sum()
        within(r.loss.view(1), want[0].view(1), terms * (2 * U + (pairs + 8) * 2.0 ** -52) * (1 + 1e-6) + beta * slack * pairs + 1e-45)
    return r


def pair_data(g, lengths, masked, behind=0, before=0):
    seq = torch.tensor([0] + list(lengths), device="cuda").cumsum(0) + before
    n = int(seq[-1]) + behind
    logp = torch.empty(n, device="cuda").exponential_(0.5, generator=g).neg_()
    ref = logp + 0.2 * torch.randn(n, generator=g, device="cuda")
    mask = (torch.rand(n, generator=g, device="cuda") < 0.6) if masked else None
    return logp, ref, seq, mask


LENGTHS = [[1, 1], [0, 0], [0, 5], [7, 0], [3, 4, 5, 6], [1000, 3, 0, 64, 65, 257], [5000, 70000], [40] * 200, [1] * 2002, [20000, 0, 7, 90001], [65] * 60, [600001, 300002],
           [9000, 8500, 8000, 10001, 1, 33000]]


@gpu
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda v: "%d_sequences_of_%d" % (len(v), sum(v)))
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("mean", [False, True])
def test_preference(ops, lengths, masked, mean):
    g = rng(sum(lengths) + 2 * masked)
    logp, ref, seq, mask = pair_data(g, lengths, masked, behind=3 * masked, before=2 * masked)
    pairs = len(lengths) // 2
    weight = torch.rand(pairs, generator=g, device="cuda") if masked else None
    offset = torch.randn(pairs, generator=g, device="cuda") if masked else None
    for smoothing in (0.0, 0.1, 1.0):
        check_preference(ops, logp, ref, seq, 0.3, smoothing, 1.0 / pairs, mask, weight, offset, mean)
    check_preference(ops, logp, None, seq, 0.01, 0.0, 1.0, mask, weight, offset, mean)
    if mask is not None:
        a = check_preference(ops, logp, ref, seq, 0.3, 0.0, 1.0, mask, None, None, mean)
        b = ops.preference_loss(logp, ref, seq, beta=0.3, mask=mask.to(torch.uint8) * 7, mean=mean)       # any byte but 0 counts
        c = ops.preference_loss(logp, ref, seq, beta=0.3, mask=mask, mean=mean, grad=False)
        assert all(torch.equal(x, y) for x, y in zip(a, b)) and c.grad is None and all(torch.equal(x, y) for x, y in zip(a[:4], c[:4]))


@gpu
def test_preference_special_values(ops):
    g = rng(1)
    logp, ref, seq, mask = pair_data(g, [4, 3, 5, 2, 6, 4], True)
    mask[:] = True
    mask[0], mask[5] = False, False
    logp[0], ref[5] = math.nan, math.inf                       # in masked places: not looked at
    check_preference(ops, logp, ref, seq, mask=mask)
    logp[1] = -math.inf                                        # the preferred answer is impossible: margin -infinity, loss infinity, gradient full
    r = check_preference(ops, logp, ref, seq, mask=mask)
    assert r.margin[0] == -math.inf and r.pair_loss[0] == math.inf and r.loss == math.inf and torch.isfinite(r.grad).all()
    r = check_preference(ops, logp, ref, seq, mask=mask, weight=torch.tensor([0.0, 1.0, 2.0], device="cuda"))
    assert torch.isfinite(r.loss) and not r.grad[:4].any()     # a pair of weight 0 adds nothing, whatever it holds
    logp[1] = -1
    s3 = int(seq[3])
    logp[s3] = -math.inf                                       # the other answer is impossible
    r = check_preference(ops, logp, ref, seq, mask=mask, smoothing=0.0)
    assert r.margin[0] == math.inf and r.pair_loss[0] == 0 and not r.grad[s3]
    r = check_preference(ops, logp, ref, seq, mask=mask, smoothing=0.2)
    assert r.pair_loss[0] == math.inf
    logp[s3] = -1
    for big in (800.0, -800.0, 1e30, -1e30):                   # margins far out: the loss is linear or 0, no overflow on the way
        check_preference(ops, logp, ref, seq, mask=mask, offset=torch.tensor([big, 0.0, big], device="cuda"))
    check_preference(ops, logp, ref, seq, beta=-2.0, mask=mask)
    check_preference(ops, logp, ref, seq, beta=0.0, mask=mask)


@gpu
def test_preference_of_nothing_and_bad_bounds(ops):
    z = torch.zeros(1, dtype=torch.int64, device="cuda")
    r = ops.preference_loss(torch.empty(0, device="cuda"), None, z)
    assert r.loss == 0 and r.pair_loss.shape == (0,) and r.ratio.shape == (0,) and r.grad.shape == (0,)
    r = ops.preference_loss(torch.full((50,), math.nan, device="cuda"), None, z)          # tokens of no sequence
    assert r.loss == 0 and not r.grad.any()
    # bounds outside the tokens are read as the nearest one, a sequence that ends before it begins as empty
    logp = -torch.rand(10, device="cuda")
    r = ops.preference_loss(logp, None, torch.tensor([-(2 ** 40), 4, 2 ** 40], device="cuda"))
    check = ops.preference_loss(logp, None, torch.tensor([0, 4, 10], device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(r, check))
    r = ops.preference_loss(logp, None, torch.tensor([6, 2, 10], device="cuda"))
    assert r.ratio[0] == 0 and torch.isfinite(r.loss)


@gpu
@pytest.mark.parametrize("n,pairs", [(40, 6), (40, 300), (3000, 7), (60000, 3)])
def test_preference_of_descending_bounds_stays_within_its_arrays(ops, n, pairs):
    """Bounds in any order and far outside: ratios are the sums between them, and nothing before or behind the outputs is written."""
    g = rng(n + pairs)
    logp = -torch.rand(n, generator=g, device="cuda")
    seq = torch.randint(-n // 4, n + n // 4, (2 * pairs + 1,), generator=g, device="cuda")
    seq[::5] *= 2 ** 40
    guard, need = 64, 16384 + 8 * pairs
    out = {k: torch.full((size + 2 * guard,), 9.0, device="cuda") for k, size in (("loss", 1), ("pair_loss", pairs), ("margin", pairs), ("ratio", 2 * pairs), ("grad", n))}
    keep = torch.empty(need, dtype=torch.uint8, device="cuda")
    ops._ck(ops.L.mlx_preference_loss(0, ops._stream(), logp.data_ptr(), None, n, seq.data_ptr(), pairs, 0.5, 0.0, 1.0, 0, None, None, None,
                                      *[out[k][guard:].data_ptr() for k in ("loss", "pair_loss", "margin", "ratio", "grad")], keep.data_ptr(), need))
    for x in out.values():
        assert (x[:guard] == 9).all() and (x[-guard:] == 9).all()
    bounds = [min(max(int(v), 0), n) for v in seq.cpu()]
    sums = torch.cat([torch.zeros(1, dtype=torch.float64), logp.double().cpu().cumsum(0)])
    want = torch.stack([sums[max(e, b)] - sums[b] for b, e in zip(bounds, bounds[1:])])
    within(out["ratio"][guard:-guard], want, half_step(want, torch.float32) + 4 * n * 2.0 ** -53 * n)


@gpu
def test_preference_gradient_is_the_difference_quotient(ops):
    """Central differences of the loss in one logp, step d: off by d^2 / 6 times the third derivative (beta^3 / 8 at most, times scale) and
    by the roundings of the two losses over 2 d."""
    g = rng(4)
    logp, ref, seq, mask = pair_data(g, [6, 4, 3, 8], True)
    args = dict(beta=0.5, smoothing=0.1, scale=0.5, mask=mask, mean=False)
    r = ops.preference_loss(logp, ref, seq, **args)
    for t in range(logp.numel()):
        d = 0.125
        up, down = logp.clone(), logp.clone()
        up[t] += d
        down[t] -= d
        q = (ops.preference_loss(up, ref, seq, **args).loss.double() - ops.preference_loss(down, ref, seq, **args).loss.double()) / (up[t].double() - down[t].double())
        assert abs(q - r.grad[t].double()) <= 0.5 * 0.5 ** 3 / 8 * d * d / 6 + 2 * 4 * U * float(r.loss + 0.1) / d, t


# ---------------------------------------------------------------------------------------------- together
def batch(g, pairs, length, vocabulary, width, dtype):
    n = 2 * pairs * length
    table = torch.randn(vocabulary, width, generator=g, device="cuda").mul_(0.3).to(dtype)
    head = torch.randn(width, vocabulary, generator=g, device="cuda").mul_(0.3).to(dtype)
    ids = torch.randint(0, vocabulary, (n,), generator=g, device="cuda")
    target = torch.where(torch.rand(n, generator=g, device="cuda") < 0.2, -1, ids.roll(-1))
    seq = torch.arange(0, n + 1, length, device="cuda")
    return table, head, ids, target, seq


def training_step(ops, table, head, ids, target, seq, ref):
    """Ids, rows of the table, logits, pairs' loss, and back to the table's gradient."""
    x = ops.embedding_lookup(table, ids, scale=2.0)
    logits = x @ head
    logp, stats = ops.token_loglik(logits, target)
    r = ops.preference_loss(logp, ref, seq, beta=0.2, scale=2.0 / (seq.numel() - 1), mask=target >= 0)
    dlogits = ops.token_loglik_gradient(logits, target, stats, r.grad, out=logits)
    dx = dlogits @ head.t().contiguous()
    return r.loss, logp, r.margin, dx, ops.embedding_gradient(dx, ids, table.shape[0], scale=2.0)


@gpu
def test_training_step_on_pairs(ops):
    """The whole run in 32 bits against automatic differentiation in 64: products over 24 and 60 terms and logits below 10 leave 1e-5 of the
    largest gradient."""
    g = rng(11)
    table, head, ids, target, seq = batch(g, 3, 40, 60, 24, torch.float32)
    ref = -4 * torch.rand(ids.numel(), generator=g, device="cuda")
    loss, logp, margin, dx, grad = training_step(ops, table, head, ids, target, seq, ref)
    t = table.double().cpu().requires_grad_()
    lp = torch.log_softmax((t[ids.cpu()] * 2.0) @ head.double().cpu(), 1)
    tc = target.cpu()
    on = tc >= 0
    lp = torch.where(on, lp.gather(1, tc.clamp(0)[:, None])[:, 0], 0.0)
    ratio = torch.where(on, lp - ref.double().cpu(), 0.0).view(6, 40).sum(1)
    h = float(np.float32(0.2)) * (ratio[:3] - ratio[3:])
    want = torch.nn.functional.softplus(-h).mean()
    want.backward()
    within(logp, lp.detach(), 1e-5)
    within(margin, h.detach(), 1e-4)
    within(loss.view(1), want.detach().view(1), 1e-4)
    within(grad, t.grad, 1e-5 * float(t.grad.abs().max()))


@gpu
def test_pairs_of_scored_rows(ops):
    """The trainer's own scores as log ratios: rows scored under a model and under the one it is compared with (mlx_score_rows), one token
    to a sequence, offset and weight as a training row has them: the logistic loss on differences of rows."""
    from mlease_amd.hip_engine import HipScorer
    r = np.random.RandomState(0)
    n, rows, per = 101, 64, 7
    rp = np.arange(0, (rows + 1) * per, per, dtype=np.int64)
    gi = r.randint(-1, n - 1, rows * per).astype(np.int32)
    model, other = r.randn(n).astype(np.float32), r.randn(n).astype(np.float32)
    sc = HipScorer(0)
    a, b = sc.score_rows(model, rp, gi, None), sc.score_rows(other, rp, gi, None)
    sc.close()
    weight, offset = torch.rand(rows // 2, device="cuda"), torch.randn(rows // 2, device="cuda")
    check_preference(ops, torch.from_numpy(a).cuda(), torch.from_numpy(b).cuda(), torch.arange(rows + 1, device="cuda"), 1.0, 0.0, 1.0, None, weight, offset)


@gpu
def test_captured_step_replays(ops):
    """The whole run in a graph, replayed on new inputs with eager work in between: the same bits as eager calls."""
    g = rng(12)
    table, head, ids, target, seq = batch(g, 2, 30, 500, 64, torch.bfloat16)
    ref = -4 * torch.rand(ids.numel(), generator=g, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        training_step(ops, table, head, ids, target, seq, ref)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = training_step(ops, table, head, ids, target, seq, ref)
    for k in range(4):
        ids.copy_(torch.randint(0, 500, ids.shape, generator=g, device="cuda"))
        target.copy_(ids.roll(-1))
        target[::7] = -1
        table.copy_(torch.randn(500, 64, generator=g, device="cuda").mul_(0.3))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        want = training_step(ops, table, head, ids, target, seq, ref)
        assert all(torch.equal(x, y) for x, y in zip(got, want)), k


@gpu
def test_two_captured_graphs_and_accumulation(ops):
    """Gradients of two batches added to one table in two graphs, replayed in turn with eager work between: every replay adds what an eager
    call adds, in the same bits."""
    g = rng(13)
    n, rows, width = 6000, 900, 72
    batches = [(torch.randn(n, width, generator=g, device="cuda").to(torch.bfloat16), some_ids(g, n, rows, torch.int64)) for _ in range(2)]
    acc = torch.zeros(rows, width, device="cuda")
    for go, ids in batches:
        ops.embedding_gradient(go, ids, rows, out=acc, accumulate=True)
    graphs = []
    for go, ids in batches:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.embedding_gradient(go, ids, rows, out=acc, accumulate=True)
        graphs.append(graph)
    acc.zero_()
    want = torch.zeros_like(acc)
    for k in range(5):
        go, ids = batches[k % 2]
        go.copy_(torch.randn(n, width, generator=g, device="cuda"))
        graphs[k % 2].replay()
        ops.embedding_gradient(go, ids, rows, out=want, accumulate=True)
        torch.cuda.synchronize()
        assert torch.equal(acc, want), k


@gpu
def test_streams_and_threads(ops):
    """Calls of several threads, each on a stream of its own, give what they give alone; another operators object is another caller."""
    data = []
    for k in range(4):
        g = rng(20 + k)
        table, head, ids, target, seq = batch(g, 2, 50, 700, 40, torch.float32)
        data.append((table, head, ids, target, seq, -4 * torch.rand(ids.numel(), generator=g, device="cuda")))
    want = [training_step(ops, *d) for d in data]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(k):
        try:
            mine = HipOperators(0)
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[k] = training_step(mine, *data[k])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    for k in range(4):
        assert all(torch.equal(x, y) for x, y in zip(got[k], want[k]))


@gpu
def test_other_devices_are_refused(ops):
    with pytest.raises(RuntimeError, match="out of range"):
        HipOperators(torch.cuda.device_count())
    t, i = torch.zeros(4, 6), torch.zeros(5, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="is on cpu"):
        ops.embedding_lookup(t, i)
    with pytest.raises(ValueError, match="is on cpu"):
        ops.embedding_lookup(t.cuda(), i.cpu())
    with pytest.raises(ValueError, match="is on cpu"):
        ops.embedding_lookup(t.cuda(), i, out=torch.zeros(5, 6))
    x = torch.empty(1, device="cuda").data_ptr()
    assert ops.L.mlx_embedding_lookup(torch.cuda.device_count(), None, 0, x, 1, 1, 1, 1, x + 512, 1, 1.0, x + 1024, 1) == -3
    assert torch.cuda.current_device() == 0


@gpu
def test_offsets_beyond_32_bits(ops):
    """Matrices of more than 2^31 elements: the last rows, against the same rows alone."""
    n, width = 70001, 32768
    big = torch.empty(n, width, device="cuda", dtype=torch.bfloat16)
    g = rng(2)
    tail = torch.randn(5, width, generator=g, device="cuda").to(torch.bfloat16)
    big.fill_(0.25)
    big[-5:] = tail
    ids = torch.tensor([n - 1, n - 5, 0, n - 3], device="cuda")
    assert torch.equal(ops.embedding_lookup(big, ids), big[ids])
    # gradient: entries far behind, ids far behind
    where = torch.full((n,), -1, device="cuda", dtype=torch.int32)
    where[-5:] = torch.tensor([n - 1, n - 1, 3, n - 1, 3], device="cuda", dtype=torch.int32)
    grad = ops.embedding_gradient(big, where, n)
    small = ops.embedding_gradient(tail, torch.tensor([1, 1, 0, 1, 0], device="cuda"), 2)
    assert torch.equal(grad[n - 1], small[1]) and torch.equal(grad[3], small[0]) and not grad[:3].any() and not grad[4:n - 1].any()
    del grad
    target = torch.full((n,), -1, device="cuda")
    target[-5:] = torch.arange(5, device="cuda") * 6000
    g5 = torch.randn(5, generator=g, device="cuda")
    w = torch.ones(n, device="cuda")
    w[-5:] = g5
    logp, stats = ops.token_loglik(big, target)
    logp5, stats5 = ops.token_loglik(tail, target[-5:].clone())
    within(logp[-5:], logp5, U * 600 + half_step(logp5.double(), torch.float32))
    assert not logp[:-5].any()
    d5 = ops.token_loglik_gradient(tail, target[-5:].clone(), stats[-5:].clone(), g5)
    d = ops.token_loglik_gradient(big, target, stats, w, out=big)
    assert torch.equal(d[-5:], d5) and not d[:-5].any()
