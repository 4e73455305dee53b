"""The operators' library without a GPU: what it exports is what its header declares, bad arguments are refused before anything could be launched
(the pointers here are fakes that are never read), and the Python entry points refuse what the kernels cannot take."""
import copy
import ctypes as C
import os
import re
import subprocess

import pytest
import torch

import hsenet_amd as H
from hsenet_amd import _lib as L
from hsenet_amd import _ops as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 0x10000
no_gpu_only = pytest.mark.skipif(torch.cuda.is_available(), reason="fake pointers: only where nothing can be launched")


def test_library_header_and_binding_agree():
    from hsenet_amd.build import OPS_LIB, build
    build()
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "hsenet_ops.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(hs_[a-z0-9_]+)\s*\(", src)))
    out = subprocess.run(["nm", "-D", "--defined-only", OPS_LIB], capture_output=True, text=True, check=True).stdout
    assert names == sorted(set(re.findall(r" T (hs_[a-z0-9_]+)", out))) == sorted(O.SIGNATURES)
    assert O.load().hs_ops_version() == O.ABI_VERSION and O.check_fresh() == O.load().hs_ops_build_id().decode()
    assert b"gfx950" in open(OPS_LIB, "rb").read()


@pytest.mark.parametrize("name", sorted(n for n in O.SIGNATURES if n not in ("hs_ops_version", "hs_ops_build_id")))
def test_null_arguments_are_refused(name):
    args = [None if a is C.c_void_p or hasattr(a, "contents") else a(0) for a in O.SIGNATURES[name]]
    rc = getattr(O.load(), name)(*args)
    assert rc == 0 if name.endswith("_ws_bytes") else rc in (L.HS_ERR_ARG, L.HS_ERR_SHAPE)


def _rot(**kw):
    d = O.RotaryDesc(2, 3, 64, 32, 3)
    d.heads[0], d.heads[1] = 4, 2
    for i in range(2):
        d.x_b[i], d.x_n[i], d.x_h[i] = 3 * 4 * 64, 4 * 64, 64
        d.y_b[i], d.y_n[i], d.y_h[i] = 3 * 4 * 64, 4 * 64, 64
    for k, v in kw.items():
        if k == "heads1":
            d.heads[1] = v
        else:
            setattr(d, k, v)
    return d


@no_gpu_only
@pytest.mark.parametrize("kw,want", [(dict(B=0), "s"), (dict(N=0), "s"), (dict(pairs=0), "s"), (dict(pairs=33), "s"), (dict(pairs=600, dh=2000), "s"),
                                     (dict(dtype=3), "a"), (dict(pos_dtype=-1), "a"), (dict(axes=0), "s"), (dict(heads1=-1), "s"),
                                     (dict(heads1=5000), "s"), (dict(dh=5000), "s"), (dict(struct_size=8), "a"), (dict(B=1 << 20, N=1 << 20), "s")])
def test_rotary_refusals(kw, want):
    rc = O.load().hs_rotary_axes(C.byref(_rot(**kw)), P, P, P, P, P, P, P, None)
    assert rc == (L.HS_ERR_SHAPE if want == "s" else L.HS_ERR_ARG)


def _diff(**kw):
    d = O.DiffAttnDesc(2, 5, 7, 4, 2, 64, L.PREC_BF16, 0, 0, 1, 0.125)
    d.q_b, d.q_n, d.q_h, d.k_b, d.k_n, d.k_h, d.v_b, d.v_n, d.v_h = 5 * 512, 512, 64, 7 * 256, 256, 64, 7 * 256, 256, 128
    d.go_b, d.go_n, d.go_h = 5 * 512, 512, 128
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@no_gpu_only
@pytest.mark.parametrize("kw,want", [(dict(B=0), "s"), (dict(Nq=0), "s"), (dict(Nk=0), "s"), (dict(H=3), "s"), (dict(Hkv=0), "s"), (dict(d=48), "s"),
                                     (dict(d=256), "s"), (dict(dtype=L.PREC_F32), "a"), (dict(scale=0.0), "a"), (dict(scale=float("nan")), "a"),
                                     (dict(q_n=511), "s"), (dict(k_h=-64), "s"), (dict(v_b=4), "s"), (dict(go_n=3), "s"), (dict(lam_stride=-1), "a"),
                                     (dict(struct_size=0), "a"), (dict(Nk=1 << 29), "s")])
def test_diff_attention_refusals(kw, want):
    lib, bad, code = O.load(), _diff(**kw), L.HS_ERR_SHAPE if want == "s" else L.HS_ERR_ARG
    if "go_n" not in kw:
        assert lib.hs_diff_attn_fwd(C.byref(bad), P, P, P, P, None, None, P, None, None, P, 1 << 40, None) == code
        assert lib.hs_diff_attn_fwd_ws_bytes(C.byref(bad)) == lib.hs_diff_attn_bwd_ws_bytes(C.byref(bad)) == 0
    assert lib.hs_diff_attn_bwd(C.byref(bad), P, P, P, P, None, None, P, P, P, P, P, P, P, P, 1 << 40, None) == code


@no_gpu_only
def test_diff_attention_pointers_and_workspace():
    lib, d = O.load(), _diff()
    assert lib.hs_diff_attn_fwd(C.byref(d), P + 8, P, P, P, None, None, P, None, None, None, 0, None) == L.HS_ERR_SHAPE
    assert lib.hs_diff_attn_fwd(C.byref(d), P, P, P, P, None, None, P, P, None, None, 0, None) == L.HS_ERR_ARG       # maps without statistics
    need = lib.hs_diff_attn_bwd_ws_bytes(C.byref(d))
    assert need == 2 * 4 * (5 * 12 + 512)                  # three numbers a row, and the rows' constants by whole tiles of 32
    assert lib.hs_diff_attn_bwd(C.byref(d), P, P, P, P, None, None, P, P, P, P, P, P, P, P, need - 1, None) == L.HS_ERR_SHAPE
    long = _diff(Nq=1, Nk=100000)
    need = lib.hs_diff_attn_fwd_ws_bytes(C.byref(long))
    assert need > 0
    assert lib.hs_diff_attn_fwd(C.byref(long), P, P, P, P, None, None, P, None, None, P, need - 1, None) == L.HS_ERR_SHAPE
    assert lib.hs_diff_attn_fwd(C.byref(long), P, P, P, P, None, None, P, None, None, None, 0, None) == L.HS_ERR_SHAPE


@pytest.mark.filterwarnings("ignore:optimizer contains a parameter group with duplicate")
def test_adamw_takes_a_parameter_once():
    p = torch.zeros(3, requires_grad=True)
    with pytest.raises(ValueError, match="twice"):
        H.AdamW([p, p])


def test_sizes_that_do_not_fit_are_errors():
    with pytest.raises(L.HsError, match="32 bits"):
        O.DIFF_PACK.pack(O.DIFF_PACK.size, 1, 1 << 31, *[1] * 8, 1.0, *[0] * 12)


@no_gpu_only
def test_adamw_refusals():
    lib = O.load()
    def call(entry=(P, P, P, P, P, P, P, 64), count=1, dtype=L.PREC_F32, bits=8, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.0):
        words = (C.c_int64 * 8)(*entry)
        return lib.hs_adamw_multi(words, count, dtype, bits, lr, b1, b2, eps, wd, None)
    for kw in (dict(count=0), dict(dtype=3), dict(bits=16), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(entry=(0, P, P, P, P, P, P, 64)),
               dict(entry=(P, P, P, P, 0, P, P, 64)), dict(entry=(P, P, P, P, P, P, 0, 64)), dict(entry=(P, P, P, P, P, P, P + 4, 64)),
               dict(entry=(P + 2, P, P, P, P, P, P, 64)), dict(entry=(P, P, P + 2, P, 0, 0, P, 64), bits=32)):
        assert call(**kw) == L.HS_ERR_ARG
    assert call(entry=(P, P, P, P, P, P, P, -1)) == L.HS_ERR_SHAPE
    assert lib.hs_adamw_moments((C.c_int64 * 8)(P, P, P, P, P, P, P, 64), 1, L.PREC_F16, None) == L.HS_ERR_ARG


def test_entry_points_refuse_host_tensors_and_bad_plans():
    q = torch.zeros(1, 2, 4, 32, dtype=torch.bfloat16)
    with pytest.raises(L.HsError, match="no CPU fallback"):
        H.rotary_axes(q, None, torch.zeros(3, 2, dtype=torch.int32), H.RotaryAxes((4, 6, 6), device="cpu"))
    with pytest.raises(L.HsError, match="no CPU fallback"):
        H.diff_attention(q, q, torch.zeros(1, 2, 2, 64, dtype=torch.bfloat16), torch.ones(2))
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.zeros(4)
    with pytest.raises(L.HsError, match="no CPU fallback"):
        H.AdamW([p]).step()
    for kw in (dict(sections=()), dict(sections=(4, -1)), dict(sections=(0, 0)), dict(sections=(600,)), dict(sections=(4,), ladder="x"),
               dict(sections=(4,), theta=0.0)):
        with pytest.raises(ValueError):
            H.RotaryAxes(**kw, device="cpu")
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(lr=torch.tensor(1.0))):
        with pytest.raises(ValueError):
            H.AdamW([p], **kw)
    with pytest.raises(ValueError, match="bf16, fp16 or fp32"):
        H.AdamW([torch.nn.Parameter(torch.zeros(4, dtype=torch.float64))])


def test_rotary_ladders():
    shared, per = H.RotaryAxes((2, 3, 3), 100.0, "shared", device="cpu"), H.RotaryAxes((2, 3, 3), 100.0, "per_axis", device="cpu")
    assert shared.axis.tolist() == per.axis.tolist() == [0, 0, 1, 1, 1, 2, 2, 2] and shared.freq.dtype == torch.float64
    assert torch.allclose(shared.freq, 100.0 ** (-torch.arange(8, dtype=torch.float64) / 8), rtol=1e-14)
    assert torch.allclose(per.freq, 100.0 ** -torch.tensor([0, 1 / 2, 0, 1 / 3, 2 / 3, 0, 1 / 3, 2 / 3], dtype=torch.float64), rtol=1e-14)


def test_diff_attention_workspace_beyond_2_31_bytes_of_rows():
    """twelve bytes a query pass 2^31 from 178956971 queries on"""
    for Nq in (178956970, 178956971, 200_000_000, 1 << 28):
        need = O.load().hs_diff_attn_bwd_ws_bytes(C.byref(_diff(B=1, Nq=Nq, Nk=40, H=1, Hkv=1, d=32)))
        assert need >= Nq * 12 + -(-Nq // 32) * 512, Nq


@no_gpu_only
def test_sizes_whose_products_wrap_are_refused():
    lib, big = O.load(), _diff(B=1 << 30, H=1 << 16, Hkv=1 << 16, Nq=1 << 28, Nk=1 << 28)
    assert lib.hs_diff_attn_fwd(C.byref(big), P, P, P, P, None, None, P, None, None, P, (1 << 63) - 1, None) == L.HS_ERR_SHAPE
    assert lib.hs_diff_attn_bwd(C.byref(big), P, P, P, P, None, None, P, P, P, P, P, P, P, P, (1 << 63) - 1, None) == L.HS_ERR_SHAPE
    heads = _rot()
    heads.heads[0] = heads.heads[1] = (1 << 31) - 1
    assert lib.hs_rotary_axes(C.byref(heads), P, P, P, P, P, P, P, None) == L.HS_ERR_SHAPE


def _launches(monkeypatch):
    """the launches of what follows, recorded instead of made, with host tensors that pass for tensors of device 0"""
    seen = []
    monkeypatch.setattr(O, "call", lambda dev, name, *a: seen.append(name))
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    return seen


def _state(p, bits, step=1):
    n = -(-p.numel() // 256)
    m = torch.zeros_like(p, dtype=torch.int8 if bits == 8 else torch.float32, requires_grad=False)
    v = torch.zeros_like(p, dtype=torch.uint8 if bits == 8 else torch.float32, requires_grad=False)
    return dict(step=step, exp_avg=m, exp_avg_sq=v, **(dict(exp_avg_scale=torch.zeros(n), exp_avg_sq_scale=torch.zeros(n)) if bits == 8 else {}))


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_states_that_no_longer_fit_are_not_read(monkeypatch, bits):
    """neither a step nor a reading of the moments hands a kernel a state that another size, type or order of the parameter needs"""
    seen = _launches(monkeypatch)
    p = torch.nn.Parameter(torch.zeros(6, 4))
    opt = H.AdamW([p], state_bits=bits)
    opt.set_state(p, **_state(p, bits))
    p.grad = torch.zeros(6, 4)
    opt.step()
    opt.moments(p)
    assert seen == ["hs_adamw_multi"] + ["hs_adamw_moments"] * (bits == 8)
    seen.clear()
    def refused(calls=(opt.step, lambda: opt.moments(p))):
        p.grad = torch.zeros_like(p)
        for f in calls:
            with pytest.raises(L.HsError):
                f()
        assert not seen
    for data in (torch.zeros(600, 400), torch.zeros(0), torch.zeros(4, 6).t(), torch.zeros(6, 8)[:, :4]):
        p.grad = None
        p.data = data
        refused()
    p.grad = None
    p.data = torch.zeros(6, 4)
    opt.param_groups[0]["state_bits"] = 40 - bits
    refused()
    opt.param_groups[0]["state_bits"] = bits
    for name in ("exp_avg", "exp_avg_sq", "step", *(("exp_avg_scale", "exp_avg_sq_scale") if bits == 8 else ())):
        held = opt.state[p][name]
        opt.state[p][name] = held.flatten()[:0]
        refused((opt.step,) if name == "step" else (opt.step, lambda: opt.moments(p)))      # (a count is not read with the moments)
        opt.state[p][name] = held
    opt.step()
    assert seen == ["hs_adamw_multi"]


def test_adamw_states_on_another_device_are_not_read(monkeypatch):
    seen = _launches(monkeypatch)
    p = torch.nn.Parameter(torch.zeros(6, 4))
    opt = H.AdamW([p], state_bits=8)
    opt.set_state(p, **_state(p, 8))
    p.grad = torch.zeros(6, 4)
    for name in list(opt.state[p]):
        held = opt.state[p][name]
        opt.state[p][name] = torch.empty_like(held, device="meta")
        monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 1 if t.is_meta else 0)
        for f in (opt.step, *[lambda: opt.moments(p)] * (name != "step")):
            with pytest.raises(L.HsError, match="device"):
                f()
        opt.state[p][name] = held
    assert not seen


@pytest.mark.parametrize("order", [lambda t: t.contiguous(memory_format=torch.channels_last), lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)])
def test_adamw_codes_are_loaded_in_their_memory_order_alone(order):
    """a scale belongs to 256 neighbours in memory: codes of another order would be read with others' scales"""
    g = torch.Generator().manual_seed(1)
    def made(data, bits):
        p = torch.nn.Parameter(data)
        opt = H.AdamW([p], state_bits=bits)
        st = _state(p, bits)
        st["exp_avg"].copy_(torch.randint(-127, 128, p.shape, generator=g))
        opt.set_state(p, **st)
        return opt, p
    plain, other = torch.zeros(4, 16, 3, 8), order(torch.zeros(4, 16, 3, 8))
    for bits in (8, 32):
        (a, p), (b, q), (c, r) = made(other, bits), made(plain, bits), made(other.clone(memory_format=torch.preserve_format), bits)
        want = a.state[p]["exp_avg"]
        c.load_state_dict(a.state_dict())                     # the same order: taken over as it is
        assert torch.equal(c.state[r]["exp_avg"], want) and c.state[r]["exp_avg"].stride() == r.stride()
        if bits == 8:
            there, back = a.state_dict(), b.state_dict()
            for opt, saved in ((b, there), (a, back)):
                with pytest.raises(L.HsError, match="memory order"):
                    opt.load_state_dict(saved)
        else:
            b.load_state_dict(a.state_dict())
            assert torch.equal(b.state[q]["exp_avg"], want) and b.state[q]["exp_avg"].is_contiguous()


def test_adamw_states_of_another_shape_are_not_spread():
    p, q = torch.nn.Parameter(torch.zeros(8, 6)), torch.nn.Parameter(torch.zeros(6))
    a, b = H.AdamW([p]), H.AdamW([q])
    b.set_state(q, **_state(q, 32))
    with pytest.raises(L.HsError, match="shape"):
        a.load_state_dict(b.state_dict())


def test_adamw_that_refuses_a_state_dict_is_as_before():
    ps = [torch.nn.Parameter(torch.zeros(6, 4)), torch.nn.Parameter(torch.zeros(300))]
    opt = H.AdamW(ps, lr=0.25, state_bits=8)
    for p in ps:
        opt.set_state(p, **_state(p, 8, step=7))
    good = opt.state_dict()
    def bad(where, what):
        d = copy.deepcopy(good)
        d["param_groups"][0]["lr"] = 0.5
        where(d).update(what) if isinstance(what, dict) else where(d).pop(what)
        return d
    first, second, group = lambda d: d["state"][0], lambda d: d["state"][1], lambda d: d["param_groups"][0]
    cases = [bad(second, dict(exp_avg=torch.zeros(299, dtype=torch.int8))), bad(second, dict(exp_avg=torch.zeros(300))), bad(second, "exp_avg_sq_scale"),
             bad(second, dict(step=torch.tensor(3.0))), bad(first, "exp_avg_sq"), bad(group, "state_bits"), bad(group, dict(state_bits=16)),
             bad(group, dict(lr=-1.0)), bad(group, dict(params=[0])), torch.optim.AdamW(ps).state_dict()]
    held = [{k: t for k, t in opt.state[p].items()} for p in ps]
    for d in cases:
        with pytest.raises((L.HsError, ValueError)):
            opt.load_state_dict(d)
        assert opt.param_groups[0]["lr"] == 0.25 and opt.param_groups[0]["state_bits"] == 8 and len(opt.state) == 2
        for p, st in zip(ps, held):
            assert list(opt.state[p]) == list(st) and all(opt.state[p][k] is t for k, t in st.items())
    opt.load_state_dict(good)
    assert all(int(opt.state[p]["step"][0]) == 7 and opt.state[p]["exp_avg"].dtype == torch.int8 for p in ps)


def test_adamw_step_that_is_refused_for_one_is_taken_for_none(monkeypatch):
    seen = _launches(monkeypatch)
    p, q = torch.nn.Parameter(torch.zeros(6, 4)), torch.nn.Parameter(torch.zeros(5))
    opt = H.AdamW([{"params": [p]}, {"params": [q], "lr": 0.1}])
    for x in (p, q):
        opt.set_state(x, **_state(x, 32))
        x.grad = torch.zeros_like(x)
    q.data, versions = torch.zeros(7), (p._version, q._version)
    with pytest.raises(L.HsError):
        opt.step()
    q.data = torch.zeros(5)
    opt.param_groups[1]["lr"] = -0.1
    with pytest.raises(ValueError):
        opt.step()
    assert not seen and p._version == versions[0]
    opt.param_groups[1]["lr"] = 0.1
    opt.step()
    assert seen == ["hs_adamw_multi"] * 2 and p._version > versions[0]


def test_adamw_refuses_bad_counts_and_strangers():
    p, q = torch.nn.Parameter(torch.zeros(6, 4)), torch.nn.Parameter(torch.zeros(6, 4))
    opt = H.AdamW([p])
    for step in (-1, 1 << 31):                                # (with -1 the next step would divide by 1 - beta^0)
        with pytest.raises(L.HsError, match="step"):
            opt.set_state(p, **_state(p, 32, step=step))
    for f in (lambda: opt.set_state(q, **_state(q, 32)), lambda: opt.moments(q)):
        with pytest.raises(L.HsError, match="not a parameter"):
            f()


def test_tensors_that_share_memory_are_found():
    """against the places of all elements, one by one"""
    import random
    from hsenet_amd.rotary import _apart, _share_memory
    def quick(xs):
        return _apart(*xs[0].shape[:2], xs[0].shape[3], [(x.shape[2], x, O.bnh(x.shape, x.stride()), None, None) for x in xs])
    rng, room, found, proved = random.Random(5), torch.zeros(4096, dtype=torch.bfloat16), [0, 0], 0
    def places(x):
        at = x.storage_offset() + sum(torch.arange(n).view([-1 if i == a else 1 for i in range(4)]) * s for a, (n, s) in enumerate(zip(x.shape, x.stride())))
        return at.flatten().tolist()
    def one():
        shape = [rng.choice([1, 2, 3]), rng.choice([1, 2, 4]), rng.choice([1, 2, 3]), 4]
        strides = rng.choice([[shape[1] * shape[2] * 4, shape[2] * 4, 4], [96, 24, 8], [96, 24, 4], [48, 12, 4], [rng.choice([8, 60, 100]), rng.choice([4, 12, 50]), rng.choice([2, 4, 6, 16])],
                              [24, 96, 8], [128, 32, 16]])
        return room.as_strided(shape, [*strides, 1], rng.choice([0, 4, 8, 12, 16, 24, 3, 200, 400]))
    for i in range(4000):
        xs = [one() for _ in range(1 + i % 4 // 2)]
        if len(xs) == 2:
            xs[1] = room.as_strided([*xs[0].shape[:2], *xs[1].shape[2:]], xs[1].stride(), xs[1].storage_offset())
        all_ = sum((places(x) for x in xs), [])
        want = len(set(all_)) < len(all_)
        assert _share_memory(xs) == want and not (want and quick(xs)), [(x.shape, x.stride(), x.storage_offset()) for x in xs]
        found[want] += 1
        proved += quick(xs)
    assert min(found) > 500 and proved > 500
    qkv = torch.zeros(2, 1000, 36, 64)                         # the thirds of a projection, heads of q and k in turn, another tensor
    for q, k in ((qkv[:, :, :12], qkv[:, :, 12:24]), (qkv[:, :, 0::3], qkv[:, :, 1::3]), (qkv[:1], qkv[1:]), (qkv[:, :, :3], torch.zeros(2, 1000, 3, 64))):
        assert not _share_memory([q, k]) and (quick([q, k]) or q.stride(2) == 192)
    for q, k in ((qkv[:, :1, :12], qkv[:, :1, 12:24]), (qkv[:1, :1, :12], qkv[:1, :1, 12:24])):
        assert quick([q, k]) and quick([k, q])
    for q, k in ((qkv[:, :, :12], qkv[:, :, 11:24]), (qkv[:, :-1], qkv[:, 1:]), (qkv[..., :40], qkv[..., 24:])):
        assert _share_memory([q, k])


def test_tensors_with_tangents_are_refused():
    """a result without a tangent would read as a derivative of zero"""
    from torch.autograd import forward_ad
    plan, pos = H.RotaryAxes((4, 6, 6), device="cpu"), torch.zeros(3, 2)
    args = [torch.zeros(1, 2, 4, 32), torch.zeros(1, 2, 4, 32), torch.zeros(1, 2, 2, 64), torch.ones(2)]
    with forward_ad.dual_level():
        for i in range(4):
            dual = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(L.HsError, match="forward-mode"):
                H.diff_attention(*dual)
        q, k, p = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (args[0], args[1], pos))
        for call in ((q, None, pos), (args[0], k, pos), (args[0], None, p)):
            for inplace in (False, True):
                with pytest.raises(L.HsError, match="forward-mode"):
                    H.rotary_axes(*call, plan, inplace=inplace)
        with pytest.raises(L.HsError, match="no CPU fallback"):                  # (without one the call goes on)
            H.rotary_axes(args[0], None, pos, plan)


def test_adamw_gradients_of_another_shape_are_not_read(monkeypatch):
    """a gradient that was there before p.data was replaced, with a state of the new size"""
    seen = _launches(monkeypatch)
    p = torch.nn.Parameter(torch.zeros(6, 4))
    opt = H.AdamW([p], state_bits=8)
    for grad, data in ((torch.zeros(6, 4), torch.zeros(600, 400)), (torch.zeros(1, 4), torch.zeros(6, 4)), (torch.zeros(4, 1).t(), torch.zeros(4, 6).t()),
                       (torch.zeros(6, 4), torch.zeros(6, 4).t())):
        p.data = torch.zeros(grad.shape)
        p.grad = grad
        p.data = data
        opt.set_state(p, **_state(p, 8))
        with pytest.raises(L.HsError, match="gradient"):
            opt.step()
    assert not seen


@no_gpu_only
@pytest.mark.parametrize("scale", [1e-38, 1e-31, 1e6, float("inf")])
def test_diff_attention_refuses_scales_out_of_range(scale):
    """the backward pass divides a row's statistics by the scale: of 1e-38 they would be infinite, and dv zero"""
    lib, bad = O.load(), _diff(scale=scale)
    assert lib.hs_diff_attn_fwd(C.byref(bad), P, P, P, P, None, None, P, None, None, P, 1 << 40, None) == L.HS_ERR_ARG
    assert lib.hs_diff_attn_bwd(C.byref(bad), P, P, P, P, None, None, P, P, P, P, P, P, P, P, 1 << 40, None) == L.HS_ERR_ARG
