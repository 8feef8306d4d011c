"""CPU checks of the tuning operators (layer norm, policy / preference loss, gradient clipping): the C entry points and
the tensor wrappers refuse what the kernels do not take, before anything is launched; struct layouts."""
import ctypes as C
import os
import subprocess

import pytest
import torch

import ldrs_amd  # noqa: F401
from ldrs_amd.hip import _lib, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD = _lib.CGN_ERR_INVALID_ARG
P = C.c_void_p(4096)  # never dereferenced: every call below is refused or has nothing to do


@pytest.fixture
def host(monkeypatch):
    """The wrappers with their device checks off and the launch replaced by a record: host validation alone runs."""
    calls = []

    def f32(t, name):
        if not (isinstance(t, torch.Tensor) and t.dtype == torch.float32):
            raise TypeError(name)

    def any16(t, name):
        if not (isinstance(t, torch.Tensor) and t.dtype in (torch.float32, torch.bfloat16)):
            raise TypeError(name)
        return t.dtype == torch.bfloat16

    def i64(t, name):
        if not (isinstance(t, torch.Tensor) and t.dtype == torch.int64 and t.is_contiguous()):
            raise TypeError(name)

    monkeypatch.setattr(ops, "_chk_f32", f32)
    monkeypatch.setattr(ops, "_chk_f32_or_bf16", any16)
    monkeypatch.setattr(ops, "_chk_i64", i64)
    monkeypatch.setattr(ops, "_call", lambda name, dev, *a: calls.append(name))
    return calls


def test_wrappers_refuse_cpu_tensors():
    x, i = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    v = torch.zeros(4)
    for call in (lambda: ops.layer_norm_fwd(x), lambda: ops.token_logp(x, i), lambda: ops.policy_loss(x, i, v),
                 lambda: ops.preference_loss(x, i, v.view(2, 2), v[:2], beta=0.1), lambda: ops.grad_norm([x]),
                 lambda: ops.clip_grad_norm([x], 1.0), lambda: ops.layer_norm_bwd(x, x, None, v, v)):
        with pytest.raises(TypeError, match="HIP"):
            call()


def test_layer_norm_refusals(host):
    x = torch.zeros(4, 8)
    v = torch.zeros(4)
    buf = torch.zeros(64)
    bad = [
        lambda: ops.layer_norm_fwd(torch.zeros(4, 0)),
        lambda: ops.layer_norm_fwd(torch.zeros(1, ops.LAYER_NORM_MAX_COLS + 1)),
        lambda: ops.layer_norm_fwd(torch.zeros(8, 4).t()),
        lambda: ops.layer_norm_fwd(torch.zeros(1, 8).expand(4, 8)),
        lambda: ops.layer_norm_fwd(torch.zeros(2, 4, 8).transpose(0, 1)),
        lambda: ops.layer_norm_fwd(x, torch.zeros(7)),
        lambda: ops.layer_norm_fwd(x, torch.zeros(16)[::2]),
        lambda: ops.layer_norm_fwd(x, eps=-1.0),
        lambda: ops.layer_norm_fwd(x, out=torch.zeros(4, 9)),
        lambda: ops.layer_norm_fwd(x, out=torch.zeros(4, 8, dtype=torch.bfloat16)),
        lambda: ops.layer_norm_bwd(torch.zeros(4, 9), x, None, v, v),
        lambda: ops.layer_norm_bwd(x.bfloat16(), x, None, v, v),
        lambda: ops.layer_norm_bwd(x, x, None, torch.zeros(3), v),
        lambda: ops.layer_norm_bwd(x, x, None, v, v, beta=1.0),
        lambda: ops.layer_norm_bwd(x, x, torch.zeros(8), v, v, dbias=torch.zeros(8), beta=1.0),
        lambda: ops.layer_norm_bwd(x, x, None, v, v, dbias=torch.zeros(8), params=False),
        lambda: ops.layer_norm_bwd(x, x, None, v, v, dx=torch.zeros(4, 7)),
        # a destination that overlaps its source without being its buffer
        lambda: ops.layer_norm_fwd(buf[:32].view(4, 8), out=buf[8:40].view(4, 8)),
        lambda: ops.layer_norm_fwd(buf.view(4, 16)[:, :8], out=buf[:32].view(4, 8)),
        lambda: ops.layer_norm_bwd(buf[:32].view(4, 8), x, None, v, v, dx=buf[4:36].view(4, 8)),
        lambda: ops.layer_norm_bwd(x, buf[:32].view(4, 8), None, v, v, dx=buf[4:36].view(4, 8)),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    with pytest.raises(TypeError):
        ops.layer_norm_fwd(x.half())
    with pytest.raises(TypeError):
        ops.layer_norm_fwd(x, torch.zeros(8, dtype=torch.bfloat16))
    assert not host
    ops.layer_norm_fwd(torch.zeros(4, 16)[:, :8], torch.zeros(8))
    ops.layer_norm_bwd(x, x, None, v, v, dx=False)
    ops.layer_norm_fwd(x, out=x)
    ops.layer_norm_bwd(x, torch.zeros(4, 8), None, v, v, dx=x)
    assert len(host) == 4


def test_layer_norm_parameter_destinations_lie_apart(host):
    """dweight and dbias are written by threads of their own while the operands are read: given destinations overlap
    neither each other nor an operand nor dx."""
    x, dy, v, w = torch.zeros(4, 8), torch.zeros(4, 8), torch.zeros(8), torch.ones(8)
    mean, rstd, buf, wide = torch.zeros(4), torch.zeros(4), torch.zeros(64), torch.zeros(4, 16)
    stats = torch.zeros(16)
    call = lambda dweight, dbias, **k: ops.layer_norm_bwd(k.pop("dy", dy), k.pop("x", x), k.pop("w", w),  # noqa: E731
                                                          k.pop("mean", mean), k.pop("rstd", rstd), dweight=dweight,
                                                          dbias=dbias, **k)
    bad = [
        lambda: call(v, v),                                            # one tensor for both
        lambda: call(buf[:8], buf[7:15]),
        lambda: call(w, v),
        lambda: call(None, w),
        lambda: call(buf[4:12], None, w=buf[:8]),
        lambda: call(x.view(-1)[:8], v),
        lambda: call(v, dy.view(-1)[24:]),
        lambda: call(v, buf[31:39], dy=buf[:32].view(4, 8)),
        lambda: call(wide.view(-1)[48:56], None, x=wide[:, :8]),
        lambda: call(v, stats[2:10], mean=stats[:4]),
        lambda: call(stats[6:14], v, rstd=stats[4:8]),
        lambda: call(buf[:8], v, dx=buf[:32].view(4, 8)),
    ]
    for k, f in enumerate(bad):
        with pytest.raises(ValueError, match="overlap"):
            f()
            raise AssertionError("case %d was taken" % k)
    assert not host
    call(buf[:8], buf[8:16])
    call(buf[32:40], buf[40:48], x=buf[:32].view(4, 8), dx=dy)
    call(None, v)
    call(v, None, dx=x)
    assert len(host) == 4


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are dummies: only where nothing can be launched")
def test_layer_norm_entry_point_refuses_one_destination_for_both():
    lib, nb = _lib.load(), C.c_int64()
    for R in (3, 2000):  # one workgroup, many
        assert lib.cgn_layer_norm_bwd_workspace(R, 8, 0, C.byref(nb)) == _lib.CGN_OK
        for off in (-28, -4, 0, 4, 28):
            assert lib.cgn_layer_norm_bwd(None, P, 8, P, 8, R, 8, 0, None, P, P, None, 8, C.c_void_p(8192),
                                          C.c_void_p(8192 + off), 0.0, P, nb.value) == BAD, (R, off)


def test_token_loss_refusals(host):
    x, i = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    v, w = torch.zeros(4), torch.ones(2, 2)
    buf = torch.zeros(64)
    inf, nan = float("inf"), float("nan")
    pref = lambda **k: ops.preference_loss(k.pop("x", x), k.pop("i", i), k.pop("w", w), k.pop("r", v[:2]),  # noqa: E731
                                           **{"beta": 0.1, **k})
    bad = [
        lambda: ops.token_logp(torch.zeros(8), i),
        lambda: ops.token_logp(torch.zeros(4, 0), i),
        lambda: ops.token_logp(torch.zeros(8, 4).t(), i),
        lambda: ops.token_logp(torch.zeros(1, 8).expand(4, 8), i),
        lambda: ops.token_logp(x, i[:3]),
        lambda: ops.token_logp(x, i, torch.zeros(5)),
        lambda: ops.token_logp(x, i, torch.zeros(8)[::2]),
        lambda: ops.token_logp(x, i, inv_tau=0.0),
        lambda: ops.token_logp(x, i, inv_tau=-1.0),
        lambda: ops.token_logp(x, i, inv_tau=inf),
        lambda: ops.token_logp(x, i, inv_tau=nan),
        lambda: ops.token_logp_bwd(x, i, torch.zeros(4), v),
        lambda: ops.token_logp_bwd(x, i, torch.zeros(4, 2), v, scale=torch.zeros(2)),
        lambda: ops.policy_loss(x, i, v[:3]),
        lambda: ops.policy_loss(x, i, v, old_logp=v[:3]),
        lambda: ops.policy_loss(x, i, v, kl_coef=0.1),
        lambda: ops.policy_loss(x, i, v, clip=(-0.1, 0.2)),
        lambda: ops.policy_loss(x, i, v, clip=(0.1, nan)),
        lambda: ops.policy_loss(x, i, v, dlogits=torch.zeros(4, 9)),
        lambda: ops.policy_loss(x, i, v, dlogits=x.bfloat16()),
        lambda: ops.policy_loss(x, i, v, dlogits=torch.zeros(8, 4).t()),
        # a destination that overlaps the logits without being their buffer
        lambda: ops.policy_loss(buf[:32].view(4, 8), i, v, dlogits=buf[8:40].view(4, 8)),
        lambda: ops.policy_loss(buf.view(4, 16)[:, :8], i, v, dlogits=buf[:32].view(4, 8)),
        lambda: pref(w=torch.ones(4)),
        lambda: pref(w=torch.ones(1, 4)),
        lambda: pref(w=torch.ones(2, 3)),
        lambda: pref(w=None),
        lambda: pref(r=v),
        lambda: pref(beta=0.0),
        lambda: pref(beta=inf),
        lambda: pref(label_smoothing=0.5),
        lambda: pref(label_smoothing=-0.1),
        lambda: pref(x=torch.zeros(0, 8), i=i[:0], w=torch.ones(0, 2), r=v[:0]),
    ]
    for k, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            raise AssertionError("case %d was taken" % k)
    with pytest.raises(TypeError):
        ops.token_logp(x, i.int())
    with pytest.raises(TypeError):
        ops.policy_loss(x, i, v.double())
    assert not host
    ops.policy_loss(x, i, v, dlogits=x)
    ops.policy_loss(buf[:32].view(4, 8), i, v, dlogits=buf[32:].view(4, 8))
    pref()
    assert len(host) == 3


def test_vocabularies_past_32_bits_are_refused(host):
    """The library counts a row's columns in 32 bits: 2^32 + 5 of them would pass for 5."""
    x = torch.empty(1, 2 ** 32 + 5, dtype=torch.bfloat16)  # (8.6 GB that nothing touches)
    i, v = torch.zeros(1, dtype=torch.int64), torch.zeros(1)
    for f in (lambda: ops.token_logp(x, i), lambda: ops.policy_loss(x, i, v),
              lambda: ops.token_logp_bwd(x, i, torch.zeros(1, 2), v, dlogits=x)):
        with pytest.raises(ValueError, match="2\\^31"):
            f()
    assert not host


def test_clip_refusals(host):
    x = torch.zeros(6, 4)
    bad = [
        lambda: ops.grad_norm([]),
        lambda: ops.clip_grad_norm([], 1.0),
        lambda: ops.grad_norm([x], norm_type=1.0),
        lambda: ops.clip_grad_norm([x], -1.0),
        lambda: ops.clip_grad_norm([x], float("nan")),
        lambda: ops.clip_grad_norm([x], 1.0, out=[x, x]),
        lambda: ops.clip_grad_norm([x], 1.0, out=[x[:, :3]]),
        lambda: ops.clip_grad_norm([x], 1.0, out=[x.bfloat16()]),
        lambda: ops.clip_grad_norm([x], 1.0, out=[torch.zeros(4, 6).t()]),
        lambda: ops.clip_grad_norm([x, x], 1.0),                       # the same tensor twice
        lambda: ops.clip_grad_norm([x, x[2:]], 1.0),
        lambda: ops.clip_grad_norm([x[:3], x[2:]], 1.0),
        lambda: ops.clip_grad_norm([x], 1.0, out=[x.view(-1)[:24].view(4, 6).t()]),
        lambda: ops.clip_grad_norm([x[:4]], 1.0, out=[x[1:5]]),        # overlaps its own gradient
        lambda: ops.grad_norm([x[:, ::2]]),
        lambda: ops.grad_norm([torch.zeros(1, 4).expand(6, 4)]),
        lambda: ops.grad_norm([torch.zeros(2, 6, 4)[:, :3]]),
    ]
    for k, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            raise AssertionError("case %d was taken" % k)
    with pytest.raises(TypeError):
        ops.grad_norm([x.double()])
    assert not host
    ops.grad_norm([x, x])                                              # reading one tensor twice is fine
    ops.clip_grad_norm([x[:3], x[3:]], 1.0)
    ops.clip_grad_norm([x.t(), torch.zeros(0)], 1.0)
    assert len(host) == 3


@pytest.mark.skipif(torch.cuda.is_available(), reason="the pointers are dummies: only where nothing can be launched")
def test_entry_points_refuse_bad_arguments():
    lib = _lib.load()
    ln = lambda **k: lib.cgn_layer_norm_fwd(None, k.get("x", P), k.get("ldx", 8), k.get("R", 2), k.get("C", 8),  # noqa: E731
                                            0, None, None, k.get("eps", 1e-5), P, k.get("ldy", 8), k.get("mean", P), P)
    for k in (dict(R=-1), dict(C=0), dict(C=8193, ldx=9000, ldy=9000), dict(ldx=7), dict(ldy=7), dict(x=None),
              dict(mean=None), dict(eps=-1.0)):
        assert ln(**k) == BAD, k
    assert ln(R=0) == _lib.CGN_OK
    lb = lambda **k: lib.cgn_layer_norm_bwd(None, P, 8, P, 8, 2000, 8, 0, None, k.get("mean", P), P, P, k.get("lddx", 8),  # noqa: E731
                                            P, P, 0.0, k.get("ws", P), k.get("bytes", 1 << 20))
    assert lb(mean=None) == BAD and lb(lddx=7) == BAD and lb(ws=None) == BAD
    nb = C.c_int64()
    assert lib.cgn_layer_norm_bwd_workspace(2000, 8, 0, C.byref(nb)) == _lib.CGN_OK and nb.value > 0
    assert lb(bytes=nb.value - 1) == _lib.CGN_ERR_WORKSPACE and lb(ws=None, bytes=0) == _lib.CGN_ERR_WORKSPACE
    assert lib.cgn_layer_norm_bwd_workspace(3, 8, 0, C.byref(nb)) == _lib.CGN_OK and nb.value == 0
    assert lib.cgn_layer_norm_bwd_workspace(0, 8, 0, C.byref(nb)) == _lib.CGN_OK and nb.value == 0
    for k in ((-1, 8), (2, 0), (2, 8193)):
        assert lib.cgn_layer_norm_bwd_workspace(*k, 0, C.byref(nb)) == BAD

    def rows(**k):
        r = _lib.TokenRows()
        r.logits, r.ld, r.M, r.target, r.V, r.inv_tau = 4096, 8, 4, 4096, 8, 1.0
        r.weight = 4096
        for n, v in k.items():
            setattr(r, n, v)
        return C.byref(r)

    for k in (dict(M=-1), dict(V=0), dict(ld=7), dict(inv_tau=0.0), dict(inv_tau=float("nan")), dict(logits=None),
              dict(target=None), dict(M=1 << 31), dict(logits=4098), dict(logits=4097, bf16=1)):
        assert lib.cgn_token_logp(None, rows(**k), P, P) == BAD, k
        assert lib.cgn_token_logp_bwd(None, rows(**k), P, P, None, P, 8) == BAD, k
    assert lib.cgn_token_logp(None, rows(), None, P) == BAD
    assert lib.cgn_token_logp(None, rows(M=0), P, P) == _lib.CGN_OK
    assert lib.cgn_token_logp_bwd(None, rows(), P, P, None, P, 7) == BAD
    pl = lambda r, **k: lib.cgn_policy_loss(None, r, k.get("A", P), None, None, k.get("lo", 0.2), 0.2, 0.0,  # noqa: E731
                                            k.get("loss", P), P, None, None, P, k.get("ldd", 8), k.get("ws", P),
                                            k.get("bytes", 1 << 20))
    for k in (dict(A=None), dict(lo=-0.1), dict(loss=None), dict(ldd=7), dict(ws=None), dict(ws=C.c_void_p(4100))):
        assert pl(rows(), **k) == BAD, k
    assert pl(rows(), bytes=32) == _lib.CGN_ERR_WORKSPACE
    pr = lambda r, **k: lib.cgn_preference_loss(None, r, k.get("T", 2), k.get("ref", P), k.get("beta", 0.1),  # noqa: E731
                                                k.get("smooth", 0.0), P, P, P, None, None, P, k.get("ldd", 8), P,
                                                k.get("bytes", 1 << 20))
    for k in (dict(T=0), dict(T=3), dict(ref=None), dict(beta=0.0), dict(beta=float("nan")), dict(smooth=0.5), dict(ldd=7)):
        assert pr(rows(), **k) == BAD, k
    assert pr(rows(weight=None)) == BAD and pr(rows(M=0)) == BAD
    assert pr(rows(), bytes=32) == _lib.CGN_ERR_WORKSPACE

    def table(*rows_):
        flat = [v for r in rows_ for v in r]
        return (C.c_int64 * max(1, len(flat)))(*flat), len(rows_)

    nb = C.c_int64()
    for t in ((0, 0, 1, 4, 0, 0, 0), (4096, 0, -1, 4, 0, 0, 0), (4096, 0, 2, 4, 3, 4, 0), (4098, 0, 1, 4, 0, 0, 0),
              (4097, 0, 1, 4, 0, 0, 1)):
        tb, n = table(t)
        assert lib.cgn_grad_norm_workspace(tb, n, 0, C.byref(nb)) == BAD, t
    tb, n = table((4096, 4096, 1, 10 ** 9, 0, 0, 0), (4096, 4096, 300, 825, 828, 828, 0), (0, 0, 1, 0, 0, 0, 0))
    assert lib.cgn_grad_norm_workspace(tb, n, 0, C.byref(nb)) == _lib.CGN_OK and 8 * 1000 < nb.value < 8 * 2000
    assert lib.cgn_grad_norm(None, tb, n, 0, 1.0, P, P, 8) == _lib.CGN_ERR_WORKSPACE
    assert lib.cgn_grad_norm(None, tb, n, 0, 1.0, None, P, nb.value) == BAD
    assert lib.cgn_clip_grads(None, tb, n, 0, 1.0, float("nan"), P, P, nb.value) == BAD
    assert lib.cgn_clip_grads(None, tb, n, 0, 1.0, 1.0, None, P, nb.value) == BAD
    tb, n = table((4096, 0, 1, 4, 0, 0, 0))
    assert lib.cgn_clip_grads(None, tb, n, 0, 1.0, 1.0, P, P, 1 << 20) == BAD  # no destination
    for one in (1, 4096, 4097, 1 << 20, (1 << 22) + 1, (1 << 25) + 1, 64000000):  # one tensor: at most 1024 partials
        tb, n = table((4096, 4096, 1, one, 0, 0, 0))
        assert lib.cgn_grad_norm_workspace(tb, n, 0, C.byref(nb)) == _lib.CGN_OK and nb.value <= 8 * 1024 + 8
    for second, ok in ((4096 + 16, True), (4096 + 12, False), (4096, False)):  # two tensors of 4, apart or not
        tb, n = table((4096, 4096, 1, 4, 0, 0, 0), (second, second, 1, 4, 0, 0, 0))
        assert lib.cgn_grad_norm_workspace(tb, n, 1, C.byref(nb)) == (_lib.CGN_OK if ok else BAD)
        assert lib.cgn_grad_norm_workspace(tb, n, 0, C.byref(nb)) == _lib.CGN_OK
    tb, n = table((4096, 4112, 1, 4, 0, 0, 0))
    assert lib.cgn_grad_norm_workspace(tb, n, 1, C.byref(nb)) == _lib.CGN_OK
    tb, n = table((4096, 4108, 1, 4, 0, 0, 0))
    assert lib.cgn_grad_norm_workspace(tb, n, 1, C.byref(nb)) == BAD
    ad = lambda **k: lib.cgn_adam_clipped_f32(None, P, k.get("g", P), P, P, k.get("n", 4), 1e-3, 0.9, 0.999, 1e-8,  # noqa: E731
                                              k.get("step", 1), None, 1.0, k.get("max_norm", 1.0), k.get("norm", P),
                                              k.get("ws", P), k.get("bytes", _lib.ADAM_CLIP_WORKSPACE))
    for k in (dict(g=None), dict(n=0), dict(n=-1), dict(step=0), dict(max_norm=-1.0), dict(max_norm=float("nan")),
              dict(norm=None), dict(ws=None), dict(ws=C.c_void_p(4100))):
        assert ad(**k) == BAD, k
    assert ad(bytes=_lib.ADAM_CLIP_WORKSPACE - 1) == _lib.CGN_ERR_WORKSPACE
    header = open(os.path.join(ROOT, "include", "cgn_hip.h")).read()
    assert "#define CGN_ADAM_CLIP_WORKSPACE %d " % _lib.ADAM_CLIP_WORKSPACE in header


def test_struct_layouts_match_header(tmp_path):
    structs = {"cgn_token_rows": _lib.TokenRows, "cgn_grad_tensor": _lib.GradTensor}
    lines = ['#include <stdio.h>', '#include "cgn_hip.h"', "int main(void){"]
    for cname, cls in structs.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (cname, cname))
        lines += ['printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (cname, f, cname, f) for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0;}"]))
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o",
                           str(exe)])
    got = dict(l.split() for l in subprocess.check_output([str(exe)]).decode().splitlines())
    for cname, cls in structs.items():
        assert int(got[cname]) == C.sizeof(cls), cname
        for f, _ in cls._fields_:
            assert int(got["%s.%s" % (cname, f)]) == getattr(cls, f).offset, (cname, f)
    assert C.sizeof(_lib.GradTensor) == 7 * 8  # hip/ops.py packs the table as plain int64 values


def test_layer_norm_module_refuses():
    from ldrs_amd.hip import nn
    with pytest.raises(ValueError):
        nn.LayerNorm(0)
    with pytest.raises(ValueError):
        nn.LayerNorm(8193)
    m = nn.LayerNorm(8)
    assert sorted(m.state_dict()) == ["bias", "weight"] == sorted(torch.nn.LayerNorm(8).state_dict())
    assert list(nn.LayerNorm(8, bias=False).state_dict()) == ["weight"]
    assert not nn.LayerNorm(8, elementwise_affine=False).state_dict()
    with pytest.raises(ValueError):
        m(torch.zeros(2, 7))
    with pytest.raises(RuntimeError, match="MI355X"):
        m(torch.zeros(2, 8))
