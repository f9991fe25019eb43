"""The routing matrix and the experts' products (alphasparseRouting*, alphasparseExpert*) against plain 64-bit
implementations, and their refusals.

Tolerances count roundings.  u(t) = finfo(t).eps / 2 is a rounding to t, U = 2^-24 one to fp32.  An fp32 sum of n products
is off by at most n * 2U * (sum of the products' absolute values): a step of 2U covers sums that cut off instead of
rounding.  An activation's or slope's own evaluation (a handful of fp32 operations, exp and erfc within a few ulp) is
given 16 roundings.  |gelu'| <= 1.13 and |silu'| <= 1.1 carry an error of Z to Y.
"""
import ctypes as C
import math
import os
import subprocess
import sys

import pytest
import torch

from library_b200 import api

U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
D16 = [torch.bfloat16, torch.float16]
ACTS = [api.ACT_NONE, api.ACT_RELU, api.ACT_GELU, api.ACT_SILU]


def u(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    """Half the smallest subnormal: the absolute part of a rounding."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def act64(z, act):
    if act == api.ACT_RELU:
        return z.clamp(min=0)
    if act == api.ACT_GELU:
        return z * torch.special.ndtr(z)
    if act == api.ACT_SILU:
        return z * torch.sigmoid(z)
    return z


def slope64(z, act):
    if act == api.ACT_RELU:
        return (z > 0).double()
    if act == api.ACT_GELU:
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == api.ACT_SILU:
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    return torch.ones_like(z)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def strided(t, pad=0, shift=0):
    """The same values with a leading dimension of cols + pad, ``shift`` elements into an allocation; what lies around
    them is NaN (a read of it would show) and is returned to check that it stays."""
    rows, cols = t.shape
    ld = cols + pad
    flat = torch.full((rows * ld + shift + 16,), float("nan"), dtype=t.dtype, device=t.device)
    view = flat[shift:shift + rows * ld].view(rows, ld)[:, :cols] if rows else flat[:0].view(0, max(cols, 1))[:, :cols]
    view.copy_(t)
    return flat, view


def untouched(flat, view, before):
    """Whether everything of the allocation outside the view is as it was."""
    mask = torch.ones(flat.shape, dtype=torch.bool, device=flat.device)
    if view.numel():
        start = (view.data_ptr() - flat.data_ptr()) // flat.element_size()
        for_rows = torch.arange(view.shape[0], device=flat.device)[:, None] * view.stride(0)
        mask[(start + for_rows + torch.arange(view.shape[1], device=flat.device)[None, :]).reshape(-1)] = False
    it = torch.int16 if flat.element_size() == 2 else torch.int32
    return torch.equal(flat.view(it)[mask], before.view(it)[mask])


def close(got, want, bound):
    got = got.double()
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), float((got - want).abs().max()), float(((got - want).abs() / bound).max()))


def places(ids, experts):
    """The definition: offsets and positions of the stable sort, slot by slot."""
    flat = ids.reshape(-1).tolist()
    counts = [0] * experts
    for e in flat:
        if 0 <= e < experts:
            counts[e] += 1
    off = [0]
    for c in counts:
        off.append(off[-1] + c)
    nxt, pos = list(off), []
    for e in flat:
        if 0 <= e < experts:
            pos.append(nxt[e])
            nxt[e] += 1
        else:
            pos.append(-1)
    return torch.tensor(off, dtype=torch.int32), torch.tensor(pos, dtype=torch.int32).reshape(ids.shape)


def offsets_of(counts):
    off = [0]
    for c in counts:
        off.append(off[-1] + c)
    return torch.tensor(off, dtype=torch.int32, device="cuda")


def buffer(size):
    return torch.empty(size, dtype=torch.uint8, device="cuda") if size else None


@pytest.fixture
def h(handle):
    handle.use_torch_stream()
    yield handle
    assert api.device_error(handle) == 0


# ---- refusals, without a GPU ------------------------------------------------------------------
# The checks come before any CUDA call, so a zeroed handle structure and descriptors over addresses that are never read do.

FAKE = C.create_string_buffer(1024)


def dn(rows, cols, dt=api.R_16BF, ld=None, order=0, ptr=0x1000):
    d = C.c_void_p()
    st = api.load().alphasparseCreateDnMat(C.byref(d), C.c_int64(rows), C.c_int64(cols), C.c_int64(cols if ld is None else ld),
                                           C.c_void_p(ptr), dt, order)
    assert st == 0
    return d


def routing(tokens=4, topk=2, experts=8, ids=0x1000, it=api.INDEX_I32, off=0x1000, pos=0x1000):
    d = C.c_void_p()
    st = api.load().alphasparseCreateRouting(C.byref(d), C.c_int64(tokens), C.c_int64(topk), C.c_int64(experts), C.c_void_p(ids), it,
                                             C.c_void_p(off), C.c_void_p(pos))
    return st, d


def test_routing_descriptor_refusals():
    assert routing()[0] == 0
    assert routing(tokens=0, ids=None, pos=None)[0] == 0
    assert api.load().alphasparseCreateRouting(None, C.c_int64(1), C.c_int64(1), C.c_int64(1), None, 2, None, None) == 7
    for bad in (dict(tokens=-1), dict(topk=0), dict(topk=api.MAX_TOPK + 1), dict(experts=0), dict(experts=api.MAX_EXPERTS + 1),
                dict(tokens=2 ** 30, topk=2), dict(tokens=2 ** 62, topk=64)):
        assert routing(**bad)[0] == 10, bad
    assert routing(tokens=2 ** 30 - 1, topk=2)[0] == 0
    assert routing(it=1)[0] == 6
    assert routing(off=None)[0] == 7
    assert routing(pos=None)[0] == 7
    assert api.load().alphasparseDestroyRouting(None) == 7


def test_routing_call_refusals():
    lib = api.load()
    r, r_none = routing()[1], routing(ids=None)[1]
    size = C.c_size_t()
    assert lib.alphasparseRoutingSort(None, r, None) == 8
    assert lib.alphasparseRoutingSort(FAKE, None, None) == 7
    assert lib.alphasparseRoutingSort(FAKE, r_none, None) == 7
    assert lib.alphasparseRoutingSort(FAKE, routing(tokens=2 ** 20)[1], None) == 7      # long: needs its buffer
    assert lib.alphasparseRoutingSort_bufferSize(FAKE, r, None) == 7
    assert lib.alphasparseRoutingSort_bufferSize(FAKE, r, C.byref(size)) == 0 and size.value == 0
    x, xs = dn(4, 16), dn(8, 16)
    assert lib.alphasparseRoutingDispatch(None, r, x, xs) == 8
    assert lib.alphasparseRoutingDispatch(FAKE, None, x, xs) == 7
    assert lib.alphasparseRoutingDispatch(FAKE, r, None, xs) == 7
    assert lib.alphasparseRoutingDispatch(FAKE, r, x, None) == 7
    assert lib.alphasparseRoutingDispatch(FAKE, r, dn(5, 16), xs) == 10                 # not the routing's tokens
    assert lib.alphasparseRoutingDispatch(FAKE, r, x, dn(8, 17)) == 10
    assert lib.alphasparseRoutingDispatch(FAKE, r, x, dn(8, 16, api.R_16F)) == 6
    assert lib.alphasparseRoutingDispatch(FAKE, r, dn(4, 16, api.R_64F), dn(8, 16, api.R_64F)) == 6
    assert lib.alphasparseRoutingDispatch(FAKE, r, dn(4, 16, order=1, ld=16), xs) == 6  # column-major
    assert lib.alphasparseRoutingDispatch(FAKE, r, dn(4, 16, ptr=0x1001), xs) == 7      # off its type's alignment
    w = C.c_void_p(0x1000)
    assert lib.alphasparseRoutingCombine(None, r, xs, w, None, x) == 8
    assert lib.alphasparseRoutingCombine(FAKE, r, None, w, None, x) == 7
    assert lib.alphasparseRoutingCombine(FAKE, r, xs, w, None, None) == 7
    assert lib.alphasparseRoutingCombine(FAKE, r, xs, w, dn(4, 16, api.R_32F), x) == 6
    assert lib.alphasparseRoutingCombine(FAKE, r, xs, w, dn(3, 16), x) == 10
    assert lib.alphasparseRoutingCombine(FAKE, r, xs, w, None, dn(4, 15)) == 10
    assert lib.alphasparseRoutingCombineGrad(None, r, x, xs, w, xs, w) == 8
    assert lib.alphasparseRoutingCombineGrad(FAKE, r, None, xs, w, xs, w) == 7
    assert lib.alphasparseRoutingCombineGrad(FAKE, r, x, None, w, xs, w) == 7           # dweights need Ys
    assert lib.alphasparseRoutingCombineGrad(FAKE, r, x, xs, w, None, None) == 7        # nothing wanted
    assert lib.alphasparseRoutingCombineGrad(FAKE, r, x, xs, w, dn(9, 16), w) == 10
    assert lib.alphasparseRoutingCombineGrad(FAKE, r, x, xs, w, dn(8, 16, api.R_16F), w) == 6


def test_expert_product_refusals():
    lib = api.load()
    off, size = C.c_void_p(0x1000), C.c_size_t()
    x, w, y, b = dn(10, 32), dn(3 * 24, 32), dn(10, 24), dn(3, 24)

    def mm(h=FAKE, op=1, e=3, off=off, x=x, w=w, b=b, act=0, r=None, z=None, y=y):
        return lib.alphasparseExpertMM(h, op, C.c_int64(e), off, x, w, b, act, r, z, y, None)

    assert mm(h=None) == 8
    for name in ("x", "w", "y"):
        assert mm(**{name: None}) == 7
    assert mm(op=2) == 6
    assert mm(act=4) == 3 and mm(act=-1) == 3
    assert mm(e=0) == 10 and mm(e=api.MAX_EXPERTS + 1) == 10
    assert mm(off=None) == 7                                                              # several segments need offsets
    assert mm(x=dn(10, 32, api.R_32F), w=dn(72, 32, api.R_32F)) == 6                      # fp32 operands: no instance
    assert mm(w=dn(72, 32, api.R_16F)) == 6
    assert mm(y=dn(10, 24, api.R_16F)) == 6
    assert mm(w=dn(71, 32)) == 10 and mm(w=dn(72, 31)) == 10 and mm(op=0) == 10
    assert mm(y=dn(11, 24)) == 10 and mm(b=dn(2, 24)) == 10 and mm(b=dn(3, 23)) == 10
    assert mm(r=dn(10, 23)) == 10 and mm(z=dn(9, 24)) == 10
    assert mm(r=dn(10, 24, api.R_32F)) == 6 and mm(z=dn(10, 24, api.R_32F)) == 6 and mm(b=dn(3, 24, api.R_16F)) == 6
    assert mm(x=dn(10, 32, order=1)) == 6
    assert mm(x=dn(2 ** 31 - 1, 32), y=dn(2 ** 31 - 1, 24)) == 10
    assert lib.alphasparseExpertMM_bufferSize(FAKE, 1, C.c_int64(3), off, x, w, y, None) == 7
    assert lib.alphasparseExpertMM_bufferSize(None, 1, C.c_int64(3), off, x, w, y, C.byref(size)) == 8
    assert lib.alphasparseExpertMM_bufferSize(FAKE, 1, C.c_int64(3), off, x, w, y, C.byref(size)) == 0 and size.value == 0

    def gw(h=FAKE, op=1, e=3, off=off, x=x, dz=y, dw=w):
        return lib.alphasparseExpertMM_gradW(h, op, C.c_int64(e), off, x, dz, dw, None)

    assert gw(h=None) == 8
    for name in ("x", "dz", "dw"):
        assert gw(**{name: None}) == 7
    assert gw(op=2) == 6 and gw(op=0) == 10 and gw(dw=dn(72, 32, api.R_16F)) == 6 and gw(dz=dn(10, 24, api.R_32F)) == 6
    assert gw(dz=dn(9, 24)) == 10 and gw(e=2) == 10 and gw(off=None) == 7
    assert lib.alphasparseExpertMM_gradW_bufferSize(FAKE, 1, C.c_int64(3), off, x, y, w, None) == 7
    assert lib.alphasparseExpertMM_gradW_bufferSize(FAKE, 1, C.c_int64(3), off, x, y, w, C.byref(size)) == 0 and size.value == 0


def test_act_grad_refusals():
    lib = api.load()
    off, buf, size = C.c_void_p(0x1000), C.c_void_p(0x1000), C.c_size_t()
    dy, db = dn(10, 24), dn(3, 24, api.R_32F)

    def ag(h=FAKE, e=3, off=off, act=2, dy=dy, z=dy, dz=dy, db=db, buf=buf):
        return lib.alphasparseExpertActGrad(h, C.c_int64(e), off, act, dy, z, dz, db, buf)

    assert ag(h=None) == 8 and ag(dy=None) == 7 and ag(z=None) == 7 and ag(buf=None) == 7
    assert ag(dz=None, db=None) == 7
    assert ag(act=4) == 3 and ag(e=0) == 10 and ag(off=None) == 7
    assert ag(db=dn(3, 24)) == 6 and ag(db=dn(2, 24, api.R_32F)) == 10
    assert ag(z=dn(10, 24, api.R_16F)) == 6 and ag(z=dn(10, 23)) == 10 and ag(dz=dn(11, 24)) == 10
    assert lib.alphasparseExpertActGrad_bufferSize(FAKE, C.c_int64(3), off, 2, dy, db, None) == 7
    assert lib.alphasparseExpertActGrad_bufferSize(FAKE, C.c_int64(3), off, 2, dy, None, C.byref(size)) == 0 and size.value == 0
    assert lib.alphasparseExpertActGrad_bufferSize(FAKE, C.c_int64(3), off, 2, dy, db, C.byref(size)) == 0 and size.value > 0
    assert lib.alphasparseGetDeviceError(None, None) == 8


def test_workspace_sizes_follow_the_operands_addresses():
    """The same descriptor, asked again after its values moved off 16 bytes, needs room for a copy: rows x cols rounded up to 8, and 256
    bytes to align."""
    lib = api.load()
    x, w, y, dz, dw = dn(10, 24), dn(3 * 40, 24), dn(10, 40), dn(10, 40), dn(3 * 40, 24)
    off, size = C.c_void_p(0x1000), C.c_size_t()

    def mm():
        assert lib.alphasparseExpertMM_bufferSize(FAKE, api.OP_T, C.c_int64(3), off, x, w, y, C.byref(size)) == 0
        return size.value

    def grad():
        assert lib.alphasparseExpertMM_gradW_bufferSize(FAKE, api.OP_T, C.c_int64(3), off, x, dz, dw, C.byref(size)) == 0
        return size.value

    assert mm() == 0 and grad() == 0
    assert lib.alphasparseDnMatSetValues(x, C.c_void_p(0x1002)) == 0
    assert mm() >= 10 * 24 * 2 and grad() >= 10 * 24 * 2
    alone = mm()
    assert lib.alphasparseDnMatSetValues(w, C.c_void_p(0x1008)) == 0
    assert mm() >= alone + 3 * 40 * 24 * 2
    assert lib.alphasparseExpertMM(FAKE, api.OP_T, C.c_int64(3), off, x, w, None, 0, None, None, y, None) == 7
    for d in (x, w):
        assert lib.alphasparseDnMatSetValues(d, C.c_void_p(0x1000)) == 0
    assert mm() == 0 and grad() == 0


ARGUMENTS = """
import torch
from library_b200 import api

class Stand:  # a device tensor's attributes, without a device
    is_cuda, dtype, device = True, torch.int32, None
    def __init__(self, n, contiguous=True): self.n, self.c = n, contiguous
    def is_contiguous(self): return self.c
    def numel(self): return self.n
    def element_size(self): return 4
    def data_ptr(self): return 4096

class Shape: tokens, topk = 4, 2

host = torch.zeros(4, 2, dtype=torch.int32)
assert_ran = [False]
assert assert_ran.__setitem__(0, True) is None
refused = [lambda: api._workspace(Stand(63), lambda: 256), lambda: api._workspace(Stand(64, False), lambda: 256),
           lambda: api._workspace(host, lambda: 1), lambda: api._segments(host[0]), lambda: api._segments(Stand(4, False)),
           lambda: api._gates(Shape, host.float()), lambda: api._gates(Shape, Stand(8)), lambda: api.Routing(host, 4), lambda: api.DnMat(host.float()),
           lambda: api.DnVec(host.float()), lambda: api.CsrMatrix(4, 2, host, host, host), lambda: api.coo2csr(host, 4)]
for i, call in enumerate(refused):
    try:
        call()
    except api.ArgumentError:
        continue
    raise SystemExit(f"call {i} was not refused")
if api._workspace(Stand(64), lambda: 256) != 4096 or api._workspace(None, None) is not None:
    raise SystemExit("a workspace that fits was refused")
print(assert_ran[0])
"""


@pytest.mark.parametrize("flag", ["-O", "-B"])
def test_tensors_are_refused_with_and_without_assertions(flag):
    """The bindings' checks of tensors (host memory, short workspaces, wrong types) hold under python -O."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, flag, "-c", ARGUMENTS], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == str(flag != "-O"), r.stdout + r.stderr[-800:]


# ---- the sort ---------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("tokens,topk,experts,dtype", [
    (0, 2, 8, torch.int32), (1, 1, 1, torch.int64), (1, 8, 64, torch.int32), (3, 5, 7, torch.int64), (33, 2, 1024, torch.int32),
    (1000, 3, 61, torch.int64), (4096, 8, 256, torch.int32), (40000, 6, 1000, torch.int64), (70001, 4, 1024, torch.int32),
    (300007, 1, 3, torch.int64), (9, 64, 70, torch.int32),
    (8192, 2, 64, torch.int32), (16385, 1, 65, torch.int64), (128, 2, 5, torch.int64)])
def test_sort(h, tokens, topk, experts, dtype):
    g = gen(tokens + topk)
    skew = (torch.rand(tokens, topk, device="cuda", generator=g) ** 2 * (experts + 2)).to(dtype) - 1   # -1 .. experts: both ends drop
    if tokens > 4 and dtype == torch.int64:
        skew[2, 0] = 2 ** 40 + 1                    # low 32 bits would be a valid expert
        skew[3, 0] = -2 ** 40 + 1
    r = api.Routing(skew, experts)
    r.position.fill_(-7)
    api.routing_sort(h, r, buffer(api.routing_buffer_size(h, r)))
    off, pos = places(skew, experts)
    assert torch.equal(r.offsets.cpu(), off) and torch.equal(r.position.cpu(), pos)


@pytest.mark.gpu
@pytest.mark.parametrize("fill", [0, 5, -1, 6])
def test_sort_all_slots_alike(h, fill):
    ids = torch.full((20000, 2), fill, dtype=torch.int32, device="cuda")
    r = api.Routing(ids, 6)
    api.routing_sort(h, r, buffer(api.routing_buffer_size(h, r)))
    off, pos = places(ids, 6)
    assert torch.equal(r.offsets.cpu(), off) and torch.equal(r.position.cpu(), pos)


# ---- dispatch and combine ----------------------------------------------------------------------

def routed(tokens, topk, experts, seed, dropped=0.2):
    g = gen(seed)
    ids = torch.randint(0, experts, (tokens, topk), device="cuda", generator=g, dtype=torch.int32)
    ids[torch.rand(tokens, topk, device="cuda", generator=g) < dropped] = -1
    if tokens > 2:
        ids[1] = -1                                # a token without any expert
    off, pos = places(ids, experts)
    return api.Routing(ids, experts, off.cuda(), pos.cuda())


SHAPES = [(1, 1, 1, 0, 0), (1, 8, 4096, 0, 0), (5, 2, 64, 8, 8), (37, 3, 1003, 0, 0), (37, 3, 1000, 24, 0), (64, 33, 7, 5, 3),
          (300, 8, 520, 8, 1), (129, 6, 2048, 0, 0), (2, 64, 40, 0, 0), (3, 4, 20000, 0, 0), (50, 3, 1258, 0, 0), (41, 2, 90, 2, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("tokens,topk,width,pad,shift", SHAPES)
def test_dispatch_and_combine(h, tokens, topk, width, pad, shift, dt):
    r = routed(tokens, topk, 9, tokens + width)
    g = gen(width)
    pos, kept = r.position.long(), r.position >= 0
    _, x = strided(torch.randn(tokens, width, device="cuda", generator=g).to(dt), pad, shift)
    xs_flat, xs = strided(torch.full((tokens * topk, width), 7.0, dtype=dt, device="cuda"), pad, shift)
    before = xs_flat.clone()
    api.routing_dispatch(h, r, api.DnMat(x), api.DnMat(xs))
    want = torch.full((tokens * topk, width), 7.0, dtype=dt, device="cuda")
    want[pos[kept]] = x[torch.nonzero(kept)[:, 0]]
    assert torch.equal(xs, want) and untouched(xs_flat, xs, before)

    # combine: rows behind the kept ones are NaN and must not be used
    ys0 = torch.randn(tokens * topk, width, device="cuda", generator=g).to(dt)
    ys0[int(kept.sum()):] = float("nan")
    _, ys = strided(ys0, pad, shift)
    w = torch.randn(tokens, topk, device="cuda", generator=g)
    w[~kept] = float("nan")
    res = torch.randn(tokens, width, device="cuda", generator=g).to(dt)
    y64, mag = torch.zeros(tokens, width, dtype=torch.float64, device="cuda"), torch.zeros(tokens, width, dtype=torch.float64, device="cuda")
    one64, one_mag = y64.clone(), mag.clone()
    for j in range(topk):
        row = torch.where(kept[:, j:j + 1], ys.double()[pos[:, j].clamp(min=0)], 0.0)
        wj = torch.where(kept[:, j:j + 1], w[:, j:j + 1].double(), 0.0)
        y64, mag, one64, one_mag = y64 + wj * row, mag + (wj * row).abs(), one64 + row, one_mag + row.abs()
    for weights, residual, want, m in ((w, res, y64 + res.double(), mag + res.double().abs()), (w, None, y64, mag), (None, None, one64, one_mag)):
        y_flat, y = strided(torch.full((tokens, width), 3.0, dtype=dt, device="cuda"), pad, shift)
        before = y_flat.clone()
        api.routing_combine(h, r, api.DnMat(ys), api.DnMat(y), weights, api.DnMat(residual) if residual is not None else None)
        close(y, want, u(dt) * want.abs() + (topk + 1) * 2 * U * m + tiny(dt))
        assert untouched(y_flat, y, before)
    y = res.clone()                                 # in place on the residual
    api.routing_combine(h, r, api.DnMat(ys), api.DnMat(y), w, api.DnMat(y))
    want = y64 + res.double()
    close(y, want, u(dt) * want.abs() + (topk + 1) * 2 * U * (mag + res.double().abs()) + tiny(dt))

    # gradient of combine
    _, dy = strided(torch.randn(tokens, width, device="cuda", generator=g).to(dt), pad, shift)
    dys_flat, dys = strided(torch.full((tokens * topk, width), 5.0, dtype=dt, device="cuda"), pad, shift)
    before = dys_flat.clone()
    dw = torch.full((tokens, topk), 11.0, device="cuda")
    api.routing_combine_grad(h, r, api.DnMat(dy), api.DnMat(ys), api.DnMat(dys), w, dw)
    t = torch.nonzero(kept)[:, 0]
    want = torch.full((tokens * topk, width), 5.0, dtype=dt, device="cuda")
    want[pos[kept]] = (w[kept][:, None] * dy.float()[t]).to(dt)     # one fp32 product, one rounding: bit for bit
    assert torch.equal(dys, want) and untouched(dys_flat, dys, before)
    prod = dy.double()[t] * ys.double()[pos[kept]]
    want_w, bound = torch.zeros(tokens, topk, dtype=torch.float64, device="cuda"), torch.zeros(tokens, topk, dtype=torch.float64, device="cuda")
    want_w[kept], bound[kept] = prod.sum(1), (width + 8) * 2 * U * prod.abs().sum(1)
    close(dw, want_w, bound)
    only = torch.full((tokens, topk), 11.0, device="cuda")
    api.routing_combine_grad(h, r, api.DnMat(dy), api.DnMat(ys), None, w, only)
    assert torch.equal(only, dw)
    alone = torch.full_like(dys, 5.0)
    api.routing_combine_grad(h, r, api.DnMat(dy), None, api.DnMat(alone), w)
    assert torch.equal(alone, dys)
    own = ys.clone()                                # dYs in place of Ys
    dw2 = torch.zeros(tokens, topk, device="cuda")
    api.routing_combine_grad(h, r, api.DnMat(dy), api.DnMat(own), api.DnMat(own), w, dw2)
    n = int(kept.sum())
    assert torch.equal(own[:n], dys[:n])
    if (width * dys.element_size()) % 16 == 0 and pad % 8 == 0 and shift % 8 == 0:
        assert torch.equal(dw2, dw)                 # the same kernel: the same order of sums


@pytest.mark.gpu
def test_dispatch_passes_over_bad_positions(h):
    """Positions outside Xs (a routing array that was never sorted, a short Xs) are neither written nor read."""
    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    pos = torch.tensor([[0, 5], [-9, 2 ** 31 - 1], [3, 4], [1, 2]], dtype=torch.int32, device="cuda")
    r = api.Routing(ids, 2, torch.zeros(3, dtype=torch.int32, device="cuda"), pos)
    x = torch.randn(4, 24, device="cuda")
    xs_flat, xs = strided(torch.zeros(5, 24, device="cuda"))
    before = xs_flat.clone()
    api.routing_dispatch(h, r, api.DnMat(x), api.DnMat(xs))
    assert torch.equal(xs, torch.stack([x[0], x[3], x[3], x[2], x[2]])) and untouched(xs_flat, xs, before)
    y = torch.zeros(4, 24, device="cuda")
    api.routing_combine(h, r, api.DnMat(xs), api.DnMat(y))
    assert torch.equal(y, torch.stack([x[0], torch.zeros_like(x[0]), x[2] + x[2], x[3] + x[3]]))
    dw = torch.ones(4, 2, device="cuda")
    api.routing_combine_grad(h, r, api.DnMat(x), api.DnMat(xs), None, None, dw)
    assert dw[0, 1] == 0 and dw[1].eq(0).all() and dw[2, 0] != 0


# ---- the products -------------------------------------------------------------------------------

# counts per segment, K, N: one row; one token's choice of experts; ragged with empty segments at both ends; a plain dense
# layer; tiles cut in every direction; K from nothing up; many segments, as many as there may be; nothing but empty ones; more tiles
# than the device holds at once; both kernels for few rows, with and without a shared contraction; long segments of small products
PRODUCTS = [([1], 64, 64), ([0, 1, 0, 1, 1], 256, 200), ([0, 130, 1, 0, 257, 64, 0], 192, 136), ([300], 512, 384), ([17], 1024, 640),
            ([5, 9], 8, 8), ([3, 0, 2], 1, 1), ([70, 3], 0, 24), ([33, 40], 1000, 515), ([129, 255, 256], 72, 264),
            ([2] * 200 + [0] * 100 + [3] * 57, 40, 24), ([600, 1], 2048, 128), ([0, 0, 0], 64, 40), ([20] * 1023 + [40], 24, 16),
            ([10] * 33, 136, 72), ([700, 900, 257, 0, 1200], 320, 2000), ([64, 50, 1], 1096, 3000), ([48] * 40, 128, 1032),
            ([1100], 200, 136), ([1300, 0, 900], 72, 40)]


def product_inputs(counts, k, n, op, dt, seed, pad, shift, tail):
    g = gen(seed)
    e, rows = len(counts), sum(counts) + tail
    x0 = torch.randn(rows, k, device="cuda", generator=g).to(dt)
    if tail:
        x0[sum(counts):] = float("nan")            # rows behind the last segment
    w0 = (torch.randn(e, n, k, device="cuda", generator=g) * max(k, 1) ** -0.5).to(dt)
    for i, c in enumerate(counts):
        if c == 0:
            w0[i] = float("nan")                    # an expert without rows: its weights must not matter
    stacked = (w0 if op == api.OP_T else w0.transpose(1, 2)).reshape((e * n, k) if op == api.OP_T else (e * k, n)).contiguous()
    _, x = strided(x0, pad, shift)
    _, w = strided(stacked, pad, shift)
    return g, e, rows, x, w0, w


@pytest.mark.gpu
@pytest.mark.parametrize("op", [api.OP_T, api.OP_N])
@pytest.mark.parametrize("case", range(len(PRODUCTS)))
@pytest.mark.parametrize("dt,pad,shift", [(torch.bfloat16, 0, 0), (torch.float16, 8, 8), (torch.bfloat16, 3, 1), (torch.float16, 2, 2)])
def test_expert_mm(h, case, op, dt, pad, shift):
    counts, k, n = PRODUCTS[case]
    tail = 5 if case % 2 == 0 and case else 0
    g, e, rows, x, w0, w = product_inputs(counts, k, n, op, dt, case, pad, shift, tail)
    off = None if e == 1 and not tail else offsets_of(counts)
    live = sum(counts)
    act = ACTS[(case + op) % 4]
    out_dt = torch.float32 if case % 3 == 1 else dt
    b = (torch.randn(e, n, device="cuda", generator=g) * 0.5).to(dt if case % 2 else torch.float32)
    r0 = torch.randn(rows, n, device="cuda", generator=g).to(out_dt)
    r0[live:] = float("nan")
    z64 = torch.zeros(rows, n, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(z64)
    for i in range(e):
        lo, hi = int(sum(counts[:i])), int(sum(counts[:i + 1]))
        if hi > lo:
            z64[lo:hi] = x[lo:hi].double() @ w0[i].double().t()
            mag[lo:hi] = x[lo:hi].double().abs() @ w0[i].double().abs().t()
    seg = torch.repeat_interleave(torch.arange(e, device="cuda"), torch.tensor(counts, device="cuda"))
    for bias, residual, preact in ((True, True, True), (False, False, False)):
        zb, m = z64.clone(), mag.clone()
        if bias:
            zb[:live] += b.double()[seg]
            m[:live] += b.double()[seg].abs()
        ez = (k + 2) * 2 * U * m
        y64 = act64(zb, act).clone()
        bound = 1.13 * ez + 16 * U * zb.abs()
        if residual:
            y64[:live] = y64[:live] + r0[:live].double()
            bound[:live] += 2 * U * (r0[:live].double().abs() + y64[:live].abs())
        y_flat, y = strided(torch.full((rows, n), 9.0, dtype=out_dt, device="cuda"), pad, shift)
        z_flat, z = strided(torch.full((rows, n), 8.0, dtype=out_dt, device="cuda"), pad, shift)
        y_before, z_before = y_flat.clone(), z_flat.clone()
        X, W, Y = api.DnMat(x), api.DnMat(w), api.DnMat(y)
        api.expert_mm(h, X, W, Y, off, op, api.DnMat(b) if bias else None, act, api.DnMat(r0) if residual else None,
                      api.DnMat(z) if preact else None, buffer(api.expert_mm_buffer_size(h, X, W, Y, off, op)))
        close(y[:live], y64[:live], (u(out_dt) * y64.abs() + bound * (1 + u(out_dt)) + tiny(out_dt))[:live])
        assert untouched(y_flat, y, y_before) and y[live:].eq(9.0).all()
        if preact:
            close(z[:live], zb[:live], (u(out_dt) * zb.abs() + ez * (1 + u(out_dt)) + tiny(out_dt))[:live])
            assert untouched(z_flat, z, z_before) and z[live:].eq(8.0).all()
            y2 = r0.clone()                         # Y in place of the residual
            api.expert_mm(h, X, W, api.DnMat(y2), off, op, api.DnMat(b), act, api.DnMat(y2), None,
                          buffer(api.expert_mm_buffer_size(h, X, W, api.DnMat(y2), off, op)))
            assert torch.equal(y2[:live], y[:live])


@pytest.mark.gpu
@pytest.mark.parametrize("op", [api.OP_T, api.OP_N])
@pytest.mark.parametrize("case", range(len(PRODUCTS)))
@pytest.mark.parametrize("dt,pad,shift", [(torch.bfloat16, 0, 0), (torch.float16, 8, 8), (torch.bfloat16, 3, 1), (torch.float16, 2, 2)])
def test_expert_mm_grad_weight(h, case, op, dt, pad, shift):
    counts, k, n = PRODUCTS[case]
    tail = 5 if case % 2 == 0 and case else 0
    g, e, rows, x, _, _ = product_inputs(counts, k, n, op, dt, case, pad, shift, tail)
    off = None if e == 1 and not tail else offsets_of(counts)
    dz0 = torch.randn(rows, n, device="cuda", generator=g).to(dt)
    dz0[sum(counts):] = float("inf")
    _, dz = strided(dz0, pad, shift)
    out_dt = torch.float32 if case % 3 == 2 else dt
    shape = (e * n, k) if op == api.OP_T else (e * k, n)
    flat, dw = strided(torch.full(shape, 6.0, dtype=out_dt, device="cuda"), pad, shift)
    before = flat.clone()
    X, D, G = api.DnMat(x), api.DnMat(dz), api.DnMat(dw)
    api.expert_mm_grad_weight(h, X, D, G, off, op, buffer(api.expert_mm_grad_weight_buffer_size(h, X, D, G, off, op)))
    want, mag = torch.zeros(e, n, k, dtype=torch.float64, device="cuda"), torch.zeros(e, n, k, dtype=torch.float64, device="cuda")
    for i in range(e):
        lo, hi = int(sum(counts[:i])), int(sum(counts[:i + 1]))
        want[i] = dz[lo:hi].double().t() @ x[lo:hi].double()
        mag[i] = dz[lo:hi].double().abs().t() @ x[lo:hi].double().abs()
    terms = torch.tensor(counts, dtype=torch.float64, device="cuda")[:, None, None] + 2
    bound = u(out_dt) * want.abs() + terms * 2 * U * mag * (1 + u(out_dt)) + tiny(out_dt)
    if op == api.OP_N:
        want, bound = want.transpose(1, 2), bound.transpose(1, 2)
    close(dw, want.reshape(shape), bound.reshape(shape))
    assert untouched(flat, dw, before)


@pytest.mark.gpu
def test_non_finite_values_stay_in_their_rows(h):
    """An infinity or NaN in one row of X, or in one segment, reaches that row's (that segment's) results only."""
    counts, k, n = [40, 30, 50], 136, 72
    off = offsets_of(counts)
    for op in (api.OP_T, api.OP_N):
        g, e, rows, x, w0, w = product_inputs(counts, k, n, op, torch.bfloat16, 3, 0, 0, 0)
        clean = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
        api.expert_mm(h, api.DnMat(x), api.DnMat(w), api.DnMat(clean), off, op)
        x2, w2 = x.clone(), w.clone()
        x2[41] = float("nan")
        x2[69, 3] = float("inf")
        size = n if op == api.OP_T else k
        w2[2 * size:] = float("nan")
        got = torch.empty_like(clean)
        api.expert_mm(h, api.DnMat(x2), api.DnMat(w2), api.DnMat(got), off, op)
        same = torch.ones(rows, dtype=torch.bool, device="cuda")
        same[41] = same[69] = False
        same[70:] = False
        assert torch.equal(got[same], clean[same])
        assert got[41].isnan().all() and got[70:].isnan().all() and not got[69].isfinite().any()
        dz = torch.randn(rows, n, device="cuda", generator=g).to(torch.bfloat16)
        shape = (e * n, k) if op == api.OP_T else (e * k, n)
        a, b = torch.empty(shape, dtype=torch.bfloat16, device="cuda"), torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        api.expert_mm_grad_weight(h, api.DnMat(x), api.DnMat(dz), api.DnMat(a), off, op)
        api.expert_mm_grad_weight(h, api.DnMat(x2), api.DnMat(dz), api.DnMat(b), off, op)
        assert torch.equal(a[:size], b[:size]) and torch.equal(a[2 * size:], b[2 * size:]) and not torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("op", [api.OP_T, api.OP_N])
@pytest.mark.parametrize("rows,n,k", [(5, 200, 64), (16, 64, 200), (41, 392, 64), (2305, 1288, 64), (7, 136, 2048), (35, 72, 1100)])
def test_a_row_has_the_same_bits_whatever_its_neighbours_hold(h, rows, n, k, op, act):
    """Rows are independent: with every odd row and every row behind the last segment replaced (by other numbers, infinities, NaN),
    the even rows of Y and Z keep their bits, in fp32 so that a difference in the last place shows.  The sizes run the kernel
    for few rows with tiles of 16 and 64, alone and with a shared contraction, and the pair kernel."""
    g = gen(rows + n)
    x = torch.randn(rows + 9, k, device="cuda", generator=g).to(torch.bfloat16)
    w = (torch.randn(n, k, device="cuda", generator=g) * k ** -0.5).to(torch.bfloat16)
    w = w if op == api.OP_T else w.t().contiguous()
    off = offsets_of([rows])
    first = None
    for scale in (1.0, 0.5, 40.0, float("inf"), float("nan")):
        x2 = x.clone()
        x2[1::2] *= scale
        x2[rows:] *= scale
        y, z = torch.zeros(rows + 9, n, device="cuda"), torch.zeros(rows + 9, n, device="cuda")
        X, W, Y = api.DnMat(x2), api.DnMat(w), api.DnMat(y)
        api.expert_mm(h, X, W, Y, off, op, None, act, None, api.DnMat(z), buffer(api.expert_mm_buffer_size(h, X, W, Y, off, op)))
        got = [t[:rows:2].clone().view(torch.int32) for t in (y, z)]
        first = got if first is None else first
        assert torch.equal(got[1], first[1])
        assert torch.equal(got[0], first[0]), int((got[0] != first[0]).sum())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 31, 33, 127, 130, 257, 1300])
@pytest.mark.parametrize("rows", [3, 50, 2400])
def test_residual_where_the_last_warp_is_part_full(h, rows, n):
    """Columns that end inside a warp's 32: only some of its lanes have a residual to read before the accumulator is read by all."""
    k, g = 96, gen(rows + n)
    x = torch.randn(rows, k, device="cuda", generator=g).to(torch.float16)
    w = (torch.randn(n, k, device="cuda", generator=g) * k ** -0.5).to(torch.float16)
    y_flat, y = strided(torch.zeros(rows, n, device="cuda"), 3, 1)
    r = torch.randn(rows, n, device="cuda", generator=g)
    before = y_flat.clone()
    api.expert_mm(h, api.DnMat(x), api.DnMat(w), api.DnMat(y), None, api.OP_T, None, api.ACT_RELU, api.DnMat(r))
    z, mag = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    want = z.clamp(min=0) + r.double()
    close(y, want, (k + 2) * 2 * U * mag + 2 * U * (want.abs() + r.double().abs()))
    assert untouched(y_flat, y, before)


@pytest.mark.gpu
def test_offsets_outside_the_rows(h):
    """Offsets are clamped to the rows; descending ones give an empty segment."""
    off = torch.tensor([-5, 3, 2, 900], dtype=torch.int32, device="cuda")
    x = torch.randn(10, 64, device="cuda").to(torch.bfloat16)
    w = torch.randn(3 * 32, 64, device="cuda").to(torch.bfloat16)
    y_flat, y = strided(torch.zeros(10, 32, dtype=torch.bfloat16, device="cuda"))
    before = y_flat.clone()
    api.expert_mm(h, api.DnMat(x), api.DnMat(w), api.DnMat(y), off)
    want = torch.cat([x[:2].double() @ w[:32].double().t(), x[2:].double() @ w[64:].double().t()])
    rows = [0, 1] + list(range(3, 10))              # row 2 lies in two segments: either may win
    assert untouched(y_flat, y, before) and (y.double() - want)[rows].abs().max() < 0.2
    dw = torch.empty(96, 64, dtype=torch.bfloat16, device="cuda")
    api.expert_mm_grad_weight(h, api.DnMat(x), api.DnMat(y), api.DnMat(dw), off)
    assert dw[32:64].eq(0).all()
    db = torch.empty(3, 32, device="cuda")
    api.expert_act_grad(h, api.DnMat(y), None, None, off, api.ACT_NONE, api.DnMat(db),
                        buffer(api.expert_act_grad_buffer_size(h, api.DnMat(y), off, api.ACT_NONE, api.DnMat(db))))
    assert db[1].eq(0).all()


@pytest.mark.gpu
def test_waits_that_run_out_are_reported(monkeypatch):
    """Failure detection without a fault: the producers announce their copies and do not issue them, so every role's bounded
    wait runs out, the blocks raise the handle's flag, free their tensor memory and leave.  A fresh handle computes."""
    x = torch.randn(600, 256, device="cuda").to(torch.bfloat16)
    w = torch.randn(512, 256, device="cuda").to(torch.bfloat16)
    y = torch.zeros(600, 512, dtype=torch.bfloat16, device="cuda")
    dw = torch.zeros(512, 256, dtype=torch.bfloat16, device="cuda")

    def calls(h):
        api.expert_mm(h, api.DnMat(x), api.DnMat(w), api.DnMat(y))                         # the pair kernel
        api.expert_mm(h, api.DnMat(x[:5]), api.DnMat(w), api.DnMat(y[:5]))                 # few rows
        api.expert_mm_grad_weight(h, api.DnMat(x[:500]), api.DnMat(y[:500]), api.DnMat(dw))  # with a tail to clear

    monkeypatch.setenv("ASP_TEST_DROP_COPY", "1")
    monkeypatch.setenv("ASP_WAIT_POLLS", "64")
    flags = []
    for i in range(3):
        broken = api.Handle()
        (lambda: api.expert_mm(broken, api.DnMat(x), api.DnMat(w), api.DnMat(y)),
         lambda: api.expert_mm(broken, api.DnMat(x[:5]), api.DnMat(w), api.DnMat(y[:5])),
         lambda: api.expert_mm_grad_weight(broken, api.DnMat(x[:500]), api.DnMat(y[:500]), api.DnMat(dw)))[i]()
        flags.append(api.device_error(broken))
    monkeypatch.delenv("ASP_TEST_DROP_COPY")
    monkeypatch.delenv("ASP_WAIT_POLLS")
    assert flags == [1, 1, 1]
    fresh = api.Handle()
    calls(fresh)
    want = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    close(y, want, u(torch.bfloat16) * want.abs() + 256 * 2 * U * mag)
    assert api.device_error(fresh) == 0


# rows, N, K of few-row products whose CTAs share the contraction (from 8 chunks of 64 on, 2 to 8 to a cluster; tiles of 16 and
# of 64 rows), and of weight gradients that do (more than 512 rows, few tiles)
SHARED = [("mm", 5, 512, 1024), ("mm", 40, 136, 2048), ("mm", 16, 72, 4104), ("grad", 1100, 64, 96), ("grad", 4133, 200, 72)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,rows,n,k", SHARED)
def test_a_shared_contraction_whose_wait_runs_out_is_reported(monkeypatch, kind, rows, n, k):
    """One CTA of every cluster gives up while its peers have their sums: the flag is raised, the peers wait for the one that
    gave up, and all leave together.  A fresh handle computes the same shapes."""
    g = gen(rows)
    x = torch.randn(rows, k, device="cuda", generator=g).to(torch.bfloat16)
    w = (torch.randn(n, k, device="cuda", generator=g) * k ** -0.5).to(torch.bfloat16)
    dz = torch.randn(rows, n, device="cuda", generator=g).to(torch.bfloat16)
    out = torch.zeros((rows, n) if kind == "mm" else (n, k), device="cuda")

    def call(h):
        if kind == "mm":
            api.expert_mm(h, api.DnMat(x), api.DnMat(w), api.DnMat(out))
        else:
            api.expert_mm_grad_weight(h, api.DnMat(x), api.DnMat(dz), api.DnMat(out))
        return api.device_error(h)

    monkeypatch.setenv("ASP_TEST_DROP_COPY", "1")
    for polls in ("1", "64", "1000"):
        monkeypatch.setenv("ASP_WAIT_POLLS", polls)
        assert call(api.Handle()) == 1
    monkeypatch.delenv("ASP_TEST_DROP_COPY")
    monkeypatch.delenv("ASP_WAIT_POLLS")
    out.fill_(float("nan"))
    assert call(api.Handle()) == 0
    a, b = (x, w.t()) if kind == "mm" else (dz.t(), x)
    close(out, a.double() @ b.double(), 2 * U * a.shape[1] * (a.double().abs() @ b.double().abs()))


# ---- the epilogue's gradient ---------------------------------------------------------------------

ACT_SHAPES = [([1], 1, 0, 0), ([0, 5, 0], 64, 0, 0), ([127, 2, 128, 300, 0, 1], 264, 8, 8), ([1000], 520, 0, 0), ([40, 260], 1003, 5, 1),
              ([1] * 700 + [0] * 50, 24, 0, 0), ([128, 128, 0, 128], 2048, 0, 0), ([0, 0], 40, 0, 0), ([3000, 1], 8, 0, 0),
              ([33, 7, 64, 0, 31, 32, 200], 1258, 0, 0), ([9000, 1, 400], 300, 2, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("case", range(len(ACT_SHAPES)))
def test_act_grad(h, case, act, dt):
    counts, n, pad, shift = ACT_SHAPES[case]
    tail, live, e = case % 3, sum(counts), len(counts)
    rows, off, g = live + tail, offsets_of(counts), gen(case)
    _, dy = strided(torch.randn(rows, n, device="cuda", generator=g).to(dt), pad, shift)
    z0 = (torch.randn(rows, n, device="cuda", generator=g) * 3).to(dt)
    if rows * n > 50:                               # far out and on the border
        z0.view(-1)[:8] = torch.tensor([0.0, -0.0, 30.0, -30.0, 200.0, -200.0, 19.9, -19.9], device="cuda").to(dt)
    z0[live:] = float("nan")
    _, z = strided(z0, pad, shift)
    dz_flat, dz = strided(torch.full((rows, n), 4.0, dtype=dt, device="cuda"), pad, shift)
    db_flat, db = strided(torch.full((e, n), 2.0, device="cuda"), pad, shift)
    before, db_before = dz_flat.clone(), db_flat.clone()
    DY, Z, DZ, DB = api.DnMat(dy), api.DnMat(z), api.DnMat(dz), api.DnMat(db)
    buf = buffer(api.expert_act_grad_buffer_size(h, DY, off, act, DB))
    api.expert_act_grad(h, DY, Z if act else None, DZ, off, act, DB, buf)
    s = slope64(z.double(), act) if act else torch.ones(rows, n, dtype=torch.float64, device="cuda")
    want = dy.double() * s
    err = 16 * U * dy.double().abs()
    close(dz[:live], want[:live], (u(dt) * want.abs() + err + tiny(dt))[:live])
    assert untouched(dz_flat, dz, before) and dz[live:].eq(4.0).all()
    lo = 0
    for i, c in enumerate(counts):
        if i < 20 or c:
            part = want[lo:lo + c]
            close(db[i], part.sum(0), (c + 2) * 2 * U * part.abs().sum(0) + err[lo:lo + c].sum(0))
        lo += c
    assert untouched(db_flat, db, db_before)
    only = torch.empty(e, n, device="cuda")         # the bias gradient alone, and dZ alone in place of dY
    api.expert_act_grad(h, DY, Z, None, off, act, api.DnMat(only), buf)
    assert torch.equal(only, db)
    own = dy.clone()
    api.expert_act_grad(h, api.DnMat(own), Z, api.DnMat(own), off, act)
    assert torch.equal(own[:live], dz[:live]) and torch.equal(own[live:], dy[live:])


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[1] * 700 + [0] * 50, [0] * 300 + [9] + [0] * 300, [0] * 1024, [0] * 40 + [700] + [0] * 40 + [3]])
def test_act_grad_of_empty_segments(h, counts):
    """dBias of every empty segment is zero, wherever it lies, and dZ may take the place of Z."""
    n, e, rows, off = 24, len(counts), sum(counts), offsets_of(counts)
    g = gen(len(counts))
    dy, z = torch.randn(rows, n, device="cuda", generator=g), torch.randn(rows, n, device="cuda", generator=g)
    db = torch.full((e, n), float("nan"), device="cuda")
    dz = torch.zeros(rows, n, device="cuda")
    DY, Z, DB = api.DnMat(dy), api.DnMat(z), api.DnMat(db)
    buf = buffer(api.expert_act_grad_buffer_size(h, DY, off, api.ACT_GELU, DB))
    api.expert_act_grad(h, DY, Z, api.DnMat(dz), off, api.ACT_GELU, DB, buf)
    c = torch.tensor(counts, device="cuda")
    assert db[c == 0].eq(0).all()
    seg = torch.repeat_interleave(torch.arange(e, device="cuda"), c)
    want = dy.double() * slope64(z.double(), api.ACT_GELU)
    sums, mag = (torch.zeros(e, n, dtype=torch.float64, device="cuda").index_add_(0, seg, t) for t in (want, want.abs()))
    err = torch.zeros_like(sums).index_add_(0, seg, 16 * U * dy.double().abs())
    close(db, sums, (c[:, None] + 2) * 2 * U * mag + err)
    again = torch.full_like(db, float("nan"))
    api.expert_act_grad(h, DY, Z, Z, off, api.ACT_GELU, api.DnMat(again), buf)
    assert torch.equal(z, dz) and torch.equal(again, db)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTS[1:])
def test_act_grad_against_differences(h, act):
    """Central differences of the 64-bit activation: step 1e-4, their error (1e-8 / 6) max|act'''| < 1e-8; away from relu's kink."""
    z = torch.linspace(-6, 6, 997 * 8, device="cuda").reshape(997, 8).contiguous()
    z = torch.where(z.abs() < 1e-3, torch.full_like(z, 0.5), z)
    dy = torch.ones_like(z)
    dz = torch.empty_like(z)
    api.expert_act_grad(h, api.DnMat(dy), api.DnMat(z), api.DnMat(dz), None, act)
    step = 1e-4
    diff = (act64(z.double() + step, act) - act64(z.double() - step, act)) / (2 * step)
    close(dz, diff, 1e-8 + 17 * U * torch.ones_like(diff))


# ---- a layer, forwards and backwards ---------------------------------------------------------------

class Layer:
    """A two-product expert layer on the library's calls: sort, dispatch, act(X W1^T + b1), H W2^T + b2, combine + residual."""

    def __init__(self, h, tokens, topk, experts, width, inner, dt, act):
        dev = "cuda"
        self.h, self.act, self.dt = h, act, dt
        self.ids = torch.zeros(tokens, topk, dtype=torch.int64, device=dev)
        self.r = api.Routing(self.ids, experts)
        slots = tokens * topk

        def t(rows, cols, dtype=dt):
            return torch.zeros(rows, cols, dtype=dtype, device=dev)

        self.x, self.y, self.xs, self.z, self.hid, self.ys = t(tokens, width), t(tokens, width), t(slots, width), t(slots, inner), t(slots, inner), t(slots, width)
        self.w1, self.b1, self.w2, self.b2 = t(experts * inner, width), t(experts, inner), t(experts * width, inner), t(experts, width)
        self.gate = torch.zeros(tokens, topk, device=dev)
        self.dy, self.dys, self.dhid, self.dz, self.dxs, self.dx = t(tokens, width), t(slots, width), t(slots, inner), t(slots, inner), t(slots, width), t(tokens, width)
        self.dgate = torch.zeros(tokens, topk, device=dev)
        self.dw1, self.dw2 = t(experts * inner, width), t(experts * width, inner)
        self.db1, self.db2 = t(experts, inner, torch.float32), t(experts, width, torch.float32)
        self.m = {k: api.DnMat(v) for k, v in vars(self).items() if isinstance(v, torch.Tensor) and v.dim() == 2 and v.dtype in (dt, torch.float32)
                  and k not in ("gate", "dgate")}
        m, off = self.m, self.r.offsets
        sizes = [api.routing_buffer_size(h, self.r), api.expert_mm_buffer_size(h, m["xs"], m["w1"], m["hid"], off),
                 api.expert_mm_buffer_size(h, m["hid"], m["w2"], m["ys"], off), api.expert_mm_buffer_size(h, m["dys"], m["w2"], m["dhid"], off, api.OP_N),
                 api.expert_mm_buffer_size(h, m["dz"], m["w1"], m["dxs"], off, api.OP_N),
                 api.expert_mm_grad_weight_buffer_size(h, m["hid"], m["dys"], m["dw2"], off), api.expert_mm_grad_weight_buffer_size(h, m["xs"], m["dz"], m["dw1"], off),
                 api.expert_act_grad_buffer_size(h, m["dhid"], off, act, m["db1"]), api.expert_act_grad_buffer_size(h, m["dys"], off, api.ACT_NONE, m["db2"])]
        self.buf = torch.empty(max(sizes) + 16, dtype=torch.uint8, device=dev)

    def fill(self, seed):
        g = gen(seed)
        tokens, topk = self.ids.shape
        experts = self.r.experts
        for name, scale in (("x", 1.0), ("w1", self.x.shape[1] ** -0.5), ("b1", 0.3), ("w2", self.z.shape[1] ** -0.5), ("b2", 0.3), ("dy", 0.3)):
            v = getattr(self, name)
            v.copy_((torch.randn(v.shape, device="cuda", generator=g) * scale).to(v.dtype))
        self.ids.copy_(torch.topk(torch.rand(tokens, experts, device="cuda", generator=g), topk, dim=1).indices)
        self.ids[::7] = -1                         # padding tokens
        self.gate.copy_(torch.softmax(torch.randn(tokens, topk, device="cuda", generator=g), 1))

    def run(self):
        h, m, off, r, buf = self.h, self.m, self.r.offsets, self.r, self.buf
        api.routing_sort(h, r, buf)
        api.routing_dispatch(h, r, m["x"], m["xs"])
        api.expert_mm(h, m["xs"], m["w1"], m["hid"], off, api.OP_T, m["b1"], self.act, preact=m["z"], buffer=buf)
        api.expert_mm(h, m["hid"], m["w2"], m["ys"], off, api.OP_T, m["b2"], buffer=buf)
        api.routing_combine(h, r, m["ys"], m["y"], self.gate, m["x"])
        api.routing_combine_grad(h, r, m["dy"], m["ys"], m["dys"], self.gate, self.dgate)
        api.expert_act_grad(h, m["dys"], None, None, off, api.ACT_NONE, m["db2"], buf)
        api.expert_mm_grad_weight(h, m["hid"], m["dys"], m["dw2"], off, buffer=buf)
        api.expert_mm(h, m["dys"], m["w2"], m["dhid"], off, api.OP_N, buffer=buf)
        api.expert_act_grad(h, m["dhid"], m["z"], m["dz"], off, self.act, m["db1"], buf)
        api.expert_mm_grad_weight(h, m["xs"], m["dz"], m["dw1"], off, buffer=buf)
        api.expert_mm(h, m["dz"], m["w1"], m["dxs"], off, api.OP_N, buffer=buf)
        api.routing_combine(h, r, m["dxs"], m["dx"], None, m["dy"])    # the residual's gradient added

    def outputs(self):
        return [self.y, self.dx, self.dgate, self.dw1, self.db1, self.dw2, self.db2]

    def reference(self):
        """The same layer in 64 bits, gradients by autograd over its formula."""
        leaves = [v.double().detach().requires_grad_() for v in (self.x, self.gate, self.w1, self.b1, self.w2, self.b2)]
        x, gate, w1, b1, w2, b2 = leaves
        experts, inner, width = self.r.experts, self.z.shape[1], self.x.shape[1]
        rows = [x * 1.0]
        for j in range(self.ids.shape[1]):
            e = self.ids[:, j].clamp(min=0)
            z = torch.einsum("th,tih->ti", x, w1.view(experts, inner, width)[e]) + b1[e]
            o = torch.einsum("ti,thi->th", act64(z, self.act), w2.view(experts, width, inner)[e]) + b2[e]
            rows.append(gate[:, j:j + 1] * o * (self.ids[:, j] >= 0)[:, None])
        y = sum(rows)
        y.backward(self.dy.double())
        return [y.detach()] + [leaves[i].grad for i in (0, 1, 2, 3, 4, 5)]


def rel(a, b):
    return float((a.double() - b).norm() / b.norm())


# Every 16-bit array between two calls carries a relative rounding of at most u; errors of separate elements add up like their
# squares at worst to u of the array's norm each.  The longest chain (dw1: x, z and hid forwards, dys, dhid, dz backwards, dw1
# itself) passes 7 roundings; norms of products grow an error by less than a factor of two here.
@pytest.mark.gpu
@pytest.mark.parametrize("dt", D16)
@pytest.mark.parametrize("act,shape", [(api.ACT_GELU, (96, 4, 8, 128, 200)), (api.ACT_SILU, (61, 2, 5, 72, 104)), (api.ACT_SILU, (1, 2, 4, 64, 128))])
def test_layer_forwards_and_backwards(h, act, shape, dt):
    layer = Layer(h, *shape, dt, act)
    layer.fill(5)
    if shape[0] == 1:
        layer.ids[0] = torch.tensor([3, 0], device="cuda")
    layer.run()
    for got, want in zip(layer.outputs(), layer.reference()):
        assert rel(got, want) <= 14 * u(dt), (rel(got, want), got.shape)


@pytest.mark.gpu
def test_product_gradients_against_differences(h):
    """A directional difference of L = sum(dZ * (X W^T)) (linear in X and in W: a difference is exact up to rounding)."""
    counts, k, n = [19, 0, 45], 80, 56
    off, dt = offsets_of(counts), torch.bfloat16
    g, e, rows, x, w0, w = product_inputs([max(c, 0) for c in counts], k, n, api.OP_T, dt, 1, 0, 0, 0)
    w = torch.nan_to_num(w, nan=0.5)
    w0 = w.view(e, n, k)
    dz = torch.randn(rows, n, device="cuda", generator=g).to(dt)
    dx, dw = torch.empty(rows, k, device="cuda"), torch.empty(e * n, k, device="cuda")
    api.expert_mm(h, api.DnMat(dz), api.DnMat(w), api.DnMat(dx), off, api.OP_N)
    api.expert_mm_grad_weight(h, api.DnMat(x), api.DnMat(dz), api.DnMat(dw), off)

    def loss(x, w):
        return sum((dz.double()[a:b] * (x[a:b] @ w[i].t())).sum() for i, (a, b) in enumerate(zip(off.tolist(), off.tolist()[1:])))

    vx, vw = torch.randn(rows, k, device="cuda", generator=g).double(), torch.randn(e, n, k, device="cuda", generator=g).double()
    for got, v, hi, lo in ((dx, vx, loss(x.double() + vx, w0.double()), loss(x.double() - vx, w0.double())),
                           (dw.view(e, n, k), vw, loss(x.double(), w0.double() + vw), loss(x.double(), w0.double() - vw))):
        mag = (got.double().abs() * v.abs()).sum()
        # every element's fp32 sum of at most 64 (dx: 56, dw: 45) products; |sum of products' sizes| < 16 |element| in the mean
        assert abs(float((hi - lo) / 2 - (got.double() * v).sum())) <= float(64 * 2 * U * 16 * mag)


@pytest.mark.gpu
def test_combine_gradient_against_differences(h):
    """L = sum(dY * combine(Ys, w)) is linear in Ys and in w: a directional difference is exact up to rounding."""
    tokens, topk, width = 40, 3, 88
    r = routed(tokens, topk, 6, 4)
    g = gen(8)
    ys, dy = torch.randn(tokens * topk, width, device="cuda", generator=g), torch.randn(tokens, width, device="cuda", generator=g)
    w = torch.randn(tokens, topk, device="cuda", generator=g)
    dys, dw = torch.zeros_like(ys), torch.zeros_like(w)
    api.routing_combine_grad(h, r, api.DnMat(dy), api.DnMat(ys), api.DnMat(dys), w, dw)
    pos, kept = r.position.long(), (r.position >= 0).double()

    def loss(ys, w):
        rows = ys[pos.clamp(min=0)] * (w * kept)[:, :, None]
        return (dy.double() * rows.sum(1)).sum()

    vy, vw = torch.randn_like(ys).double(), torch.randn_like(w).double()
    for got, v, diff in ((dys, vy, loss(ys.double() + vy, w.double()) - loss(ys.double() - vy, w.double())),
                         (dw, vw, loss(ys.double(), w.double() + vw) - loss(ys.double(), w.double() - vw))):
        # dys: one rounding an element; dw: fp32 sums of 88 products whose sizes add up to less than 16 times their sum in the mean
        assert abs(float(diff / 2 - (got.double() * v).sum())) <= float(96 * 2 * U * 16 * (got.double() * v).abs().sum())


@pytest.mark.gpu
def test_a_workspace_that_is_too_small_is_refused(h):
    x, w = torch.zeros(9, 33, device="cuda", dtype=torch.float16), torch.zeros(20, 33, device="cuda", dtype=torch.float16)
    y, dw = torch.zeros(9, 20, device="cuda", dtype=torch.float16), torch.zeros(20, 33, device="cuda", dtype=torch.float16)
    X, W, Y, D = api.DnMat(x), api.DnMat(w), api.DnMat(y), api.DnMat(dw)
    small = torch.zeros(16, dtype=torch.uint8, device="cuda")
    for call in (lambda b: api.expert_mm(h, X, W, Y, buffer=b), lambda b: api.expert_mm_grad_weight(h, X, Y, D, buffer=b)):
        with pytest.raises(AssertionError):
            call(small)
        with pytest.raises(api.AlphaSparseError) as e:
            call(None)
        assert e.value.status == 7
    db = torch.zeros(1, 20, device="cuda")
    with pytest.raises(AssertionError):
        api.expert_act_grad(h, Y, None, None, None, api.ACT_NONE, api.DnMat(db), small)
    r = api.Routing(torch.zeros(20000, 2, dtype=torch.int32, device="cuda"), 6)
    with pytest.raises(AssertionError):
        api.routing_sort(h, r, small)


@pytest.mark.gpu
def test_captured_layer_and_other_streams(h):
    """The whole layer captured into a graph and replayed on new inputs, and run on a stream of its own, gives the bits of the
    plain call; a second layer with its own workspace runs beside it."""
    args = (160, 4, 16, 128, 136, torch.bfloat16, api.ACT_GELU)
    layer, other = Layer(h, *args), Layer(h, *args)
    want = {}
    for seed in (1, 2):
        layer.fill(seed)
        layer.run()
        torch.cuda.synchronize()
        want[seed] = [t.clone() for t in layer.outputs()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        h.use_torch_stream()
        layer.run()                                 # warm-up on the capture stream
        s.synchronize()
        graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            h.use_torch_stream()
            layer.run()
        with torch.cuda.graph(graph2, stream=s):
            h.use_torch_stream()
            other.run()
    torch.cuda.synchronize()
    h.use_torch_stream()
    for seed in (2, 1, 2):
        layer.fill(seed)
        other.fill(3 - seed)
        for t in layer.outputs():
            t.fill_(77.0)
        torch.cuda.synchronize()
        t2 = torch.cuda.Stream()
        with torch.cuda.stream(s):
            graph.replay()
        with torch.cuda.stream(t2):
            graph2.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(layer.outputs(), want[seed]))
        assert all(torch.equal(a, b) for a, b in zip(other.outputs(), want[3 - seed]))
    del graph, graph2


@pytest.mark.gpu
def test_repeated_calls_give_the_same_bits(h):
    layer = Layer(h, 700, 3, 12, 264, 520, torch.float16, api.ACT_SILU)
    layer.fill(9)
    layer.run()
    first = [t.clone() for t in layer.outputs()]
    for _ in range(3):
        layer.run()
        assert all(torch.equal(a, b) for a, b in zip(layer.outputs(), first))


@pytest.mark.gpu
def test_offsets_past_32_bits(h):
    """Element offsets beyond 2^31 (rows x leading dimension): the last rows of a tall matrix."""
    rows, k = 70000, 32768
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.randn(3, k, device="cuda").to(torch.bfloat16)
    w = (torch.randn(64, k, device="cuda") * k ** -0.5).to(torch.bfloat16)
    y = torch.empty(rows, 64, dtype=torch.bfloat16, device="cuda")
    api.expert_mm(h, api.DnMat(x), api.DnMat(w), api.DnMat(y))
    want = x[-3:].double() @ w.double().t()
    mag = x[-3:].double().abs() @ w.double().abs().t()
    close(y[-3:], want, u(torch.bfloat16) * want.abs() + k * 2 * U * mag)
    assert y[:-3].eq(0).all()
    ids = torch.zeros(3, 1, dtype=torch.int32, device="cuda")
    pos = torch.tensor([[rows - 1], [rows - 2], [5]], dtype=torch.int32, device="cuda")
    r = api.Routing(ids, 1, torch.zeros(2, dtype=torch.int32, device="cuda"), pos)
    out = torch.empty(3, k, dtype=torch.bfloat16, device="cuda")
    api.routing_combine(h, r, api.DnMat(x), api.DnMat(out))
    assert torch.equal(out, torch.stack([x[-1], x[-2], x[5]]))
    api.routing_dispatch(h, r, api.DnMat(out), api.DnMat(x))
    assert torch.equal(x[-1], out[0]) and torch.equal(x[-2], out[1])
    z = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    api.expert_act_grad(h, api.DnMat(x), api.DnMat(z), api.DnMat(x), None, api.ACT_SILU)
    assert torch.equal(x[-1], (out[0].float() * 0.5).to(torch.bfloat16))


ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def python(code):
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr[-800:]


def test_the_stream_is_asked_of_torch_where_the_short_way_is_missing():
    python("""
import torch
for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
class Stream: cuda_stream = 77
torch.cuda.current_stream = lambda: Stream
from library_b200 import api
assert api._stream_number() == 77
""")


@pytest.mark.gpu
@pytest.mark.parametrize("short", [True, False])
def test_a_handle_follows_torchs_stream(short):
    """A program whose first call is the library's: torch's own state of the device is set up, and the handle takes the
    current stream, with the short way of asking for it and without."""
    python(f"""
import ctypes as C
import torch
from library_b200 import api
h = api.Handle()
assert torch.cuda.is_initialized() and (api._raw_stream is not None or not {short})
if not {short}:
    api._raw_stream = None
def stream():
    p = C.c_void_p()
    assert api.load().alphasparseGetStream(h.h, C.byref(p)) == 0
    return p.value or 0
assert stream() == torch.cuda.current_stream().cuda_stream
s = torch.cuda.Stream()
with torch.cuda.stream(s):
    h.use_torch_stream()
assert stream() == s.cuda_stream != 0
h.use_torch_stream()
assert stream() == torch.cuda.current_stream().cuda_stream
""")
