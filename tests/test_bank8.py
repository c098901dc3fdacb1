"""The paged 8-bit bank (rmem_amd/bank8.py, include/rmem_hip.h): plan, append, gather and attend against plain implementations --
codes, slots and tables exactly, attention in 64 bits with tolerances derived beside them -- and their refusals."""
import ctypes as C
import math
import os
import subprocess
import tempfile

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
TOP = {"int8": 127.0, "e4m3": 448.0}
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------------- plain reference
def e4m3_values():
    """The 256 values of the 8-bit float, from its definition (NaN at 0x7f / 0xff)."""
    out = np.zeros(256)
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        x = (8 + m) * 2.0 ** (e - 10) if e else m * 2.0 ** -9
        out[b] = math.nan if b & 127 == 127 else -x if b > 127 else x
    return out


E4M3 = e4m3_values()


def decode(b, code):
    return b.astype(np.float64) - 128 if code == "int8" else E4M3[b]


def encode(x, code):
    """fp32 array in units of the scale -> bytes, round to nearest even, saturating, NaN -> 0."""
    x = np.where(np.isnan(x), np.float32(0), x).astype(np.float32)
    if code == "int8":
        return (np.rint(np.clip(x, -127, 127)) + 128).astype(np.uint8)
    x = np.clip(x, -448, 448).astype(np.float64)
    e = np.clip(np.floor(np.log2(np.maximum(np.abs(x), 1e-30))), -6, None)
    step = 2.0 ** (e - 3)
    v = np.rint(x / step) * step
    pos = E4M3[:127]
    return np.where(np.signbit(v) | (x < 0), 128, 0).astype(np.uint8) + np.searchsorted(pos, np.abs(v)).astype(np.uint8)


class PlainPool:
    """Codes by (page, token, head, dim) and scales by (page, head), in numpy."""

    def __init__(self, pages, heads, dim, page, code):
        self.page, self.code, self.pages, self.heads, self.dim = page, code, pages, heads, dim
        zero = 128 if code == "int8" else 0
        self.codes = {w: np.full((pages, page, heads, dim), zero, np.uint8) for w in "kv"}
        self.scale = {w: np.ones((pages, heads), np.float32) for w in "kv"}

    def append(self, k, v, slots):
        """k, v: fp32 numpy [rows, heads, dim]"""
        place = {}                                   # page -> {offset: row}, the last row of several
        for i, s in enumerate(int(x) for x in slots):
            if 0 <= s < self.pages * self.page:
                place.setdefault(s // self.page, {})[s % self.page] = i
        top = np.float32(TOP[self.code])
        zero = 128 if self.code == "int8" else 0
        for pg, at in place.items():
            offs, lo, hi = np.array(sorted(at)), min(at), max(at) + 1
            rows = np.array([at[o] for o in offs])
            rest = np.array([o for o in range(hi) if o not in at], int)
            for w, x in (("k", k[rows]), ("v", v[rows])):
                with np.errstate(invalid="ignore"):
                    mx = np.where(np.isfinite(x), np.abs(x), np.float32(0)).max(axis=(0, 2)).astype(np.float32)
                fresh = np.maximum(mx, np.float32(1e-30)) / top
                for h in range(self.heads):
                    was = self.scale[w][pg, h]
                    grown = lo > 0 and fresh[h] > was
                    new = was if lo and not grown else fresh[h]
                    if grown:
                        old = decode(self.codes[w][pg, rest, h], self.code).astype(np.float32)
                        self.codes[w][pg, rest, h] = encode(old * (was / new), self.code)
                    elif not lo:
                        self.codes[w][pg, rest, h] = zero
                    with np.errstate(invalid="ignore", over="ignore"):
                        self.codes[w][pg, offs, h] = encode(x[:, h] * (np.float32(1) / new), self.code)
                    self.scale[w][pg, h] = new
                if w == "v":      # the rest of the last 32-token tile
                    self.codes[w][pg, hi:-(-hi // 32) * 32] = zero

    def values(self, w):
        return decode(self.codes[w], self.code) * self.scale[w].astype(np.float64)[:, None, :, None]

    def tokens(self, values, table_row, length):
        """[length, heads, dim] of a request, from values(w)"""
        t = np.arange(length)
        return values[np.asarray(table_row)[t // self.page], t % self.page]

    def to_device(self, B):
        p = B.Pool.empty(self.pages, self.heads, self.dim, self.page, self.code, DEV)
        p.k.copy_(torch.from_numpy(store_keys(self.codes["k"])))
        p.v.copy_(torch.from_numpy(store_values(self.codes["v"])))
        p.k_scale.copy_(torch.from_numpy(self.scale["k"]))
        p.v_scale.copy_(torch.from_numpy(self.scale["v"]))
        return p


def store_keys(c):
    n, p, h, d = c.shape
    out = np.zeros((n, h, d // 16, p, 16), np.uint8)
    for t in range(p):
        for b in range(d // 16):
            out[:, :, b, t] = c[:, t, :, 16 * b:16 * b + 16]
    return out


def store_values(c):
    n, p, h, d = c.shape
    out = np.zeros((n, h, p // 32, 2, d, 16), np.uint8)
    for t in range(p):
        q = t % 32
        out[:, :, t // 32, (q // 4) % 2, :, 4 * (q // 8) + q % 4] = c[:, t]
    return out


def load_keys(x):
    n, h, b, p, _ = x.shape
    return x.transpose(0, 3, 1, 2, 4).reshape(n, p, h, b * 16)


def load_values(x):
    n, h, tiles, _, d, _ = x.shape
    out = np.zeros((n, tiles * 32, h, d), np.uint8)
    for t in range(tiles * 32):
        q = t % 32
        out[:, t] = x[:, :, t // 32, (q // 4) % 2, :, 4 * (q // 8) + q % 4]
    return out


def random_pool(rs, pages, heads, dim, page, code):
    p = PlainPool(pages, heads, dim, page, code)
    for w in "kv":
        x = rs.standard_normal(p.codes[w].shape).astype(np.float32) * (TOP[code] / 4)
        p.codes[w] = encode(x, code)
        p.scale[w] = ((rs.rand(pages, heads) * 0.6 + 0.7) * 4 / TOP[code]).astype(np.float32)
    return p


def make_table(rs, lens, page, pages, cols=None):
    held = [-(-n // page) for n in lens]
    cols = cols or max(1, max(held) + 1)
    ids = rs.permutation(pages)[:sum(held)]
    t = np.full((len(lens), cols), -1, np.int32)
    at = 0
    for r, n in enumerate(held):
        t[r, :n] = ids[at:at + n]
        at += n
    return t


def attend64(pool, q, cu, lens, table, causal, scale):
    """Reference output and lse in 64 bits, and per element the weighted mean of |v| and per row the largest sum of |q k| scale
    (what the tolerances are made of).  q: numpy float64 [rows, heads_q, dim]."""
    rows, hq, dim = q.shape
    out, mean = np.zeros((rows, hq, dim)), np.zeros((rows, hq, dim))
    lse, most = np.full((rows, hq), -np.inf), np.zeros((rows, hq))
    group = hq // pool.heads
    all_k, all_v = pool.values("k"), pool.values("v")
    for r in range(len(lens)):
        ln, n = int(lens[r]), int(cu[r + 1] - cu[r])
        k, v = pool.tokens(all_k, table[r], ln), pool.tokens(all_v, table[r], ln)
        if not n or not ln:
            continue
        rows = slice(int(cu[r]), int(cu[r]) + n)
        sees = np.arange(ln)[None] < (ln - n + np.arange(n) + 1 if causal else np.full(n, ln))[:, None]
        on = sees.any(1)
        for h in range(hq):
            qq, kk, vv = q[rows, h], k[:, h // group], v[:, h // group]
            s = np.where(sees, qq @ kk.T * scale, -np.inf)
            m = np.where(on, s.max(1), 0.0)
            p = np.exp(s - m[:, None])
            total = np.where(on, p.sum(1), 1.0)
            out[rows, h] = p @ vv / total[:, None]
            mean[rows, h] = p @ np.abs(vv) / total[:, None]
            lse[rows, h] = np.where(on, m + np.log(total), -np.inf)
            most[rows, h] = np.where(sees, np.abs(qq) @ np.abs(kk).T, 0.0).max(1) * scale
    return out, lse, mean, most


def attend_tolerance(kind, dim, out, lse, mean, most):
    """Per element.  A weight is off by a factor of e^d, d being the score's error: the product sums `dim` terms in fp32 (each
    addition at most 2^-24 of the sum of |q k|, in MFMA blocks: dim of them at worst), fp32 queries count with 22 bits (2^-22),
    the scaled score, the sum with the maximum and the exponent are rounded a few times (2^-24 of numbers below |score| + 150 in
    the log2 domain, value scales being within 2^-88 .. 2^20) and 2^x is good to 2^-22.  Both sums see it: 2 d.  Weights are
    rounded once (2^-11; fp32 calls 2^-22, or 2^-25 of the largest weight 2^10 below the normal range), sums of weights and of
    products add fp32 roundings that are below the same terms.  Then the output's own rounding, half a step."""
    d = 2.0 ** -24 * (dim + 8) * most + (2.0 ** -22 * most if kind == "fp32" else 0) + 2.0 ** -24 * 4 * (1.4427 * np.abs(np.where(np.isfinite(lse), lse, 0)) + 20) + 2.0 ** -22
    w = 2.0 ** -22 if kind == "fp32" else 2.0 ** -11
    eps = torch.finfo(TYPES[kind]).eps / 2
    tol = eps * np.abs(out) + (1.01 * (2 * d + 2.0 ** -20) + w)[..., None] * mean if np.ndim(w) else \
        eps * np.abs(out) + (1.01 * (2 * d + 2.0 ** -20))[..., None] * mean + w * mean
    # values below the type's normal range: half a step there
    tol = tol + {"fp32": 0.0, "fp16": 2.0 ** -25, "bf16": 0.0}[kind]
    return tol, np.where(np.isfinite(lse), 1.01 * d + 2.0 ** -22 * (np.abs(np.where(np.isfinite(lse), lse, 0)) + 20), 0.0)


def to_np(t):
    return t.detach().float().cpu().numpy()


@pytest.fixture(scope="module")
def B():
    from rmem_amd import bank8, hip
    hip.load()
    return bank8


# ----------------------------------------------------------------------------------------------------------------- refusals
def test_struct_sizes_match_the_header():
    from rmem_amd import hip
    src = r'''
    #include "rmem_hip.h"
    #include <stdio.h>
    int main(){ printf("%zu %zu %zu %zu %zu\n", sizeof(rmem_bank8), sizeof(rmem_bank8_plan_args), sizeof(rmem_bank8_append_args),
                       sizeof(rmem_bank8_gather_args), sizeof(rmem_bank8_attn_args)); return 0; }'''
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "s.c"), "w").write(src)
        subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), os.path.join(d, "s.c"), "-o", os.path.join(d, "s")])
        sizes = [int(x) for x in subprocess.check_output([os.path.join(d, "s")]).split()]
    assert sizes == [C.sizeof(x) for x in (hip.Bank8Args, hip.Bank8PlanArgs, hip.Bank8AppendArgs, hip.Bank8GatherArgs, hip.Bank8AttnArgs)]


def _addr(i):
    return (i + 1) << 20


def _bank(hip, **kw):
    d = dict(k=_addr(0), v=_addr(1), k_scale=_addr(2), v_scale=_addr(3), pages=10, heads=2, page=64, dim=64, code=0)
    d.update(kw)
    return hip.Bank8Args(*(d[n] for n, _ in hip.Bank8Args._fields_))


BAD_BANKS = [dict(k=0), dict(v=0), dict(k_scale=0), dict(v_scale=0), dict(pages=0), dict(pages=-1), dict(heads=0), dict(page=16),
             dict(page=48), dict(page=256), dict(dim=16), dict(dim=48), dict(dim=256), dict(code=2), dict(code=-1), dict(k=_addr(0) + 8),
             dict(v=_addr(1) + 1), dict(pages=1 << 25, page=64)]


@pytest.mark.parametrize("bad", BAD_BANKS, ids=str)
def test_c_abi_refuses_bad_banks(bad):
    """Argument checks come before any HIP call."""
    from rmem_amd import hip
    lib = hip.load()
    b = _bank(hip, **bad)
    ap = hip.Bank8AppendArgs(b, _addr(4), _addr(5), 1, 128, 64, 128, 64, _addr(6), 4, None, 0)
    assert lib.rmem_bank8_append_workspace(C.byref(ap)) == -1
    ga = hip.Bank8GatherArgs(b, _addr(4), 4, _addr(5), _addr(6), 0)
    at = hip.Bank8AttnArgs(b, _addr(4), _addr(5), None, 1, 128, 64, 128, 64, _addr(6), _addr(7), 1, 4, _addr(8), 4, 4, 2, 1, 1, 0.1,
                           _addr(20), 1 << 40)
    assert lib.rmem_bank8_append(C.byref(ap), None) == -1
    assert lib.rmem_bank8_gather(C.byref(ga), None) == -1
    assert lib.rmem_bank8_attn(C.byref(at), None) == -1
    assert lib.rmem_bank8_attn_workspace(C.byref(at)) == -1


def test_c_abi_refuses_bad_arguments():
    from rmem_amd import hip
    lib = hip.load()
    good = dict(ctx=_addr(0), add=_addr(1), had=0, reqs=2, table=_addr(2), ld_table=8, cols=8, page=64, free_ring=_addr(3), ring=16,
                state_in=_addr(4), state_out=_addr(5), cu=_addr(6), lens=_addr(7), start=_addr(8), slots=_addr(9), rows=4, status=_addr(10))
    for bad in (dict(ctx=0), dict(add=0), dict(reqs=0), dict(reqs=-3), dict(table=0), dict(ld_table=7), dict(cols=0), dict(page=16), dict(page=96),
                dict(free_ring=0), dict(ring=0), dict(state_in=0), dict(state_out=0), dict(cu=0), dict(lens=0), dict(start=0), dict(slots=0),
                dict(rows=-1), dict(status=0), dict(cols=1 << 25, ld_table=1 << 25)):
        a = hip.Bank8PlanArgs()
        for n, _ in hip.Bank8PlanArgs._fields_:
            val = {**good, **bad}[n]
            setattr(a, n, val)
        assert lib.rmem_bank8_plan(C.byref(a), None) == -1, bad
    assert lib.rmem_bank8_plan(None, None) == -1 and lib.rmem_bank8_append(None, None) == -1
    assert lib.rmem_bank8_gather(None, None) == -1 and lib.rmem_bank8_attn(None, None) == -1 and lib.rmem_bank8_attn_workspace(None) == -1

    b = _bank(hip)
    good = dict(bank=b, k=_addr(4), v=_addr(5), type=1, k_row=128, k_head=64, v_row=128, v_head=64, slots=_addr(6), rows=4)
    for bad in (dict(k=0), dict(v=0), dict(slots=0), dict(type=3), dict(type=-1), dict(rows=-1), dict(rows=1 << 24), dict(rows=5000),
                dict(rows=5000, workspace=_addr(7), workspace_bytes=79), dict(rows=5000, workspace=_addr(7) + 4, workspace_bytes=80)):
        a = hip.Bank8AppendArgs()
        for n, val in {**good, **bad}.items():
            setattr(a, n, val)
        assert lib.rmem_bank8_append(C.byref(a), None) == -1, bad
    good = dict(bank=b, slots=_addr(4), rows=4, ko=_addr(5), vo=_addr(6), type=0)
    for bad in (dict(slots=0), dict(ko=0), dict(vo=0), dict(ko=_addr(5) + 4), dict(vo=_addr(6) + 8), dict(type=3), dict(rows=-1)):
        a = hip.Bank8GatherArgs()
        for n, val in {**good, **bad}.items():
            setattr(a, n, val)
        assert lib.rmem_bank8_gather(C.byref(a), None) == -1, bad
    good = dict(bank=b, q=_addr(4), out=_addr(5), lse=0, type=1, q_row=256, q_head=64, o_row=256, o_head=64, cu=_addr(6), lens=_addr(7),
                reqs=2, rows=4, table=_addr(8), ld_table=16, cols=16, heads_q=4, max_rows=2, causal=1, scale=0.125, workspace=_addr(20),
                workspace_bytes=1 << 40)
    for bad in (dict(q=0), dict(out=0), dict(cu=0), dict(lens=0), dict(table=0), dict(workspace=0), dict(workspace=_addr(20) + 4),
                dict(workspace_bytes=16), dict(type=3), dict(reqs=0), dict(rows=-1), dict(cols=0), dict(ld_table=3), dict(heads_q=3),
                dict(heads_q=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf),
                dict(cols=1 << 25, ld_table=1 << 25)):
        a = hip.Bank8AttnArgs()
        for n, val in {**good, **bad}.items():
            setattr(a, n, val)
        assert lib.rmem_bank8_attn(C.byref(a), None) == -1, bad


@pytest.mark.parametrize("heads,group,longest,each", [(8, 1, 1, 1 + 1 / 16), (8, 8, 1, 1 + 8 / 16), (64, 1, 100, 1 + 1 / 32), (1, 1, 300, 1 + 1 / 32),
                                                      (128, 4, 1, 1 + 4 / 16)])
def test_c_abi_refuses_reads_of_too_many_workgroups(heads, group, longest, each):
    """A request of its own for every row: heads * (rows * each + parts) workgroups, which have to stay below 2^24.  The workspace's
    size and the call agree; the limit is where the header puts it, up to the parts of what is divided.  (With longest * group above
    256 a call makes a launch of tiles of 128 rows and one of 32, of which the latter has more workgroups.)"""
    from rmem_amd import hip
    lib = hip.load()

    def args(rows):
        return hip.Bank8AttnArgs(_bank(hip, heads=heads), _addr(4), _addr(5), None, 1, heads * group * 64, 64, heads * group * 64, 64, _addr(6), _addr(7),
                                 rows, rows, _addr(8), 4, 4, heads * group, longest, 1, 0.1, _addr(20), 1 << 60)

    limit = 2 ** 24 / heads / each
    parts = max(2048, heads) / heads
    fits, not_fits = args(int(limit - parts - 2)), args(int(limit + 2))
    assert lib.rmem_bank8_attn_workspace(C.byref(fits)) >= 0
    assert lib.rmem_bank8_attn_workspace(C.byref(not_fits)) == -1 and lib.rmem_bank8_attn(C.byref(not_fits), None) == -1


def test_python_refuses_host_tensors_and_bad_choices():
    from rmem_amd import bank8, hip
    z = lambda *s, dt=torch.uint8: torch.zeros(*s, dtype=dt)
    with pytest.raises(hip.RmemError):
        bank8.Pool(z(2, 1, 4, 64, 16), z(2, 1, 2, 2, 64, 16), z(2, 1, dt=torch.float32), z(2, 1, dt=torch.float32), 64)
    for kw in (dict(page=16), dict(page=100), dict(dim=80), dict(code="int4")):
        with pytest.raises(hip.RmemError):
            bank8.Pool.empty(**{**dict(pages=2, heads=1, dim=64, page=64, device="cpu"), **kw})
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    with pytest.raises(hip.RmemError):
        bank8.plan(i(2), i(2), i(2, 4), i(8), i(2), page=64, rows=2)
    with pytest.raises(hip.RmemError):
        bank8.append(None, z(1), z(1), i(1))
    with pytest.raises(hip.RmemError):
        bank8.gather("pool", i(1))
    with pytest.raises(hip.RmemError):
        bank8.attend(None, z(1), i(2), i(1), i(1, 1))


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def test_tensors_that_require_grad_are_refused(dev):
    """Codes carry no gradient, so a graph would be cut without a word; under no_grad, or detached, the same tensors are taken."""
    from types import SimpleNamespace
    from rmem_amd import bank8
    from rmem_amd.hip import RmemError
    f = lambda *s, grad=False: torch.ones(*s, dtype=torch.float16, device=dev, requires_grad=grad)
    plain, leaf = f(3, 2, 64), f(3, 2, 64, grad=True)
    if dev == "cpu":                                   # the check itself: pools live on a device
        pool = SimpleNamespace(device=plain.device, dim=64)
        for t in (leaf, leaf * 2):
            with pytest.raises(RmemError, match="grad"):
                bank8._dense(t, "k", pool, 2)
            with torch.no_grad():
                bank8._dense(t, "k", pool, 2)
            bank8._dense(t.detach(), "k", pool, 2)
        bank8._dense(plain, "k", pool, 2)
        return
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    pool = bank8.Pool.empty(2, 2, 64, 32, "int8", dev)
    slots, args = i(0, 1, 2), (i(0, 3), i(3), torch.zeros(1, 2, dtype=torch.int32, device=dev))
    before = pool.k.clone()
    for bad in ((leaf, plain), (plain, leaf)):
        with pytest.raises(RmemError, match="grad"):
            bank8.append(pool, *bad, slots)
    assert torch.equal(pool.k, before)
    with torch.no_grad():
        bank8.append(pool, leaf, leaf, slots)
        want = bank8.attend(pool, leaf, *args)
    for kw in (dict(q=leaf), dict(q=plain, out=leaf)):
        with pytest.raises(RmemError, match="grad"):
            bank8.attend(pool, kw["q"], *args, out=kw.get("out"))
    got = bank8.attend(pool, leaf.detach(), *args)
    assert torch.equal(got, want) and not got.requires_grad


def test_out_layouts_that_lie_apart():
    """Every step and size of a small range: what is taken shares no memory, and what nests is taken -- also rows that begin right
    behind the last head's end, with gaps between heads."""
    from rmem_amd import bank8
    buf, dim = torch.zeros(200), 3
    for rows in range(1, 5):
        for heads in range(1, 5):
            for row in range(0, 24):
                for head in range(0, 24):
                    t = buf.as_strided((rows, heads, dim), (row, head, 1))
                    at = (torch.arange(rows)[:, None, None] * row + torch.arange(heads)[None, :, None] * head + torch.arange(dim)).flatten()
                    apart, nested = at.unique().numel() == at.numel(), False
                    for (a, n), (b, m) in (((row, rows), (head, heads)), ((head, heads), (row, rows))):
                        nested |= (n == 1 or a >= dim) and (m == 1 or b >= a * (n - 1) + dim)
                    assert not nested or apart
                    assert bank8._apart(t) == nested, (rows, heads, row, head)


@pytest.mark.gpu
def test_python_refuses_mismatched_device_tensors(B):
    from rmem_amd.hip import RmemError
    pool = B.Pool.empty(8, 2, 64, 64, "int8", DEV)
    f = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device=DEV)
    i = lambda *s, dt=torch.int32: torch.zeros(*s, dtype=dt, device=DEV)
    k = f(4, 2, 64)
    for bad in ((f(4, 3, 64), k, i(4)), (k, f(4, 2, 32), i(4)), (k, f(4, 2, 64, dt=torch.float32), i(4)), (k, k, i(5)),
                (k, k, i(4, dt=torch.int64)), (f(4, 2, 128)[:, :, ::2], k, i(4)), (k.cpu(), k, i(4)), (k, k, i(8)[::2]),
                (k.to(torch.float64), k.to(torch.float64), i(4))):
        with pytest.raises(RmemError):
            B.append(pool, *bad)
    q, cu, lens, table = f(3, 4, 64), i(3), i(2), i(2, 16)
    B.attend(pool, q, cu, lens, table)
    for kw in (dict(q=f(3, 3, 64)), dict(q=f(3, 4, 32)), dict(cu=i(2)), dict(lens=i(2, dt=torch.int64)), dict(table=i(3, 4)),
               dict(table=i(2, 0)), dict(table=i(4, 2).t()), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
               dict(out=f(3, 4, 64, dt=torch.float32)), dict(out=f(2, 4, 64)), dict(out=f(1, 4, 64).expand(3, 4, 64)), dict(lse=f(3, 4)), dict(workspace=f(4, dt=torch.uint8))):
        a = dict(pool=pool, q=q, cu=cu, lens=lens, table=table)
        a.update(kw)
        with pytest.raises(RmemError):
            B.attend(**a)
    for kw in (dict(ctx=i(0)), dict(add=i(3)), dict(table=i(3, 4)), dict(free=i(0)), dict(state=i(3)), dict(page=20), dict(rows=-1),
               dict(had=i(3)), dict(add=i(2, dt=torch.int64))):
        a = dict(ctx=i(2), add=i(2), table=i(2, 4), free=i(8), state=i(2), page=64, rows=0)
        a.update(kw)
        with pytest.raises(RmemError):
            B.plan(**a)
    with pytest.raises(RmemError):
        B.gather(pool, i(4), torch.float64)
    with pytest.raises(RmemError):
        B.gather(pool, i(4, 1))
    # nothing to do is not an error
    B.append(pool, f(0, 2, 64), f(0, 2, 64), i(0))
    assert B.gather(pool, i(0))[0].shape == (0, 2, 64)
    assert B.attend(pool, f(0, 4, 64), i(3), lens, table).shape == (0, 4, 64)


# -------------------------------------------------------------------------------------------------------------------- plan
def plan_plain(ctx, add, table, free, state, page, rows, had=None):
    """Request by request, as the header describes it."""
    ctx, add = [max(0, int(x)) for x in ctx], [max(0, int(x)) for x in add]
    table, free = table.copy(), free.copy()
    reqs, cols, ring = len(ctx), table.shape[1], len(free)
    head, count = int(state[0]) % ring, min(max(0, int(state[1])), ring)
    up = lambda x: -(-x // page)
    back = 0
    for r in range(reqs):
        if had is not None:
            for c in range(up(ctx[r]), min(cols, up(max(0, int(had[r]))))):
                if count + back < ring:
                    free[(head + count + back) % ring] = table[r, c]
                back += 1
    cu, lens, start, slots = [0], [], [], np.full(rows, -1, np.int32)
    asked = taken = missing = 0
    for r in range(reqs):
        have, need = up(ctx[r]), up(ctx[r] + add[r]) - up(ctx[r])
        fits = have + need <= cols
        if fits:
            asked += need
        ok = fits and (need == 0 or asked <= count)
        if ok:
            for i in range(need):
                table[r, have + i] = free[(head + asked - need + i) % ring]
            taken += need
        else:
            missing += need
        for i in range(add[r]):
            if ok and cu[-1] + i < rows:
                pos = ctx[r] + i
                slots[cu[-1] + i] = table[r, pos // page] * page + pos % page
        cu.append(cu[-1] + add[r])
        lens.append(ctx[r] + (add[r] if ok else 0))
        start.append(ctx[r] if ok else -1)
    return dict(table=table, free=free, cu=cu, lens=lens, start=start, slots=slots,
                state=[(head + taken) % ring, min(ring, count - taken + back)], status=[taken, missing])


def check_plan(B, ctx, add, table, free, state, page, rows, had=None):
    want = plan_plain(ctx, add, table, free, state, page, rows, had)
    d = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
    t, f, s = d(table), d(free), d(state)
    p = B.plan(d(ctx), d(add), t, f, s, page=page, rows=rows, had=None if had is None else d(had))
    got = dict(p._asdict(), table=t, free=f)
    for n, x in want.items():
        assert np.array_equal(got[n].cpu().numpy(), np.asarray(x)), n
    assert np.array_equal(s.cpu().numpy(), np.asarray(state))


@pytest.mark.gpu
@pytest.mark.parametrize("reqs,most,ctx_most,page,spare", [
    (1, 1, 1, 32, 3), (1, 200, 500, 64, 0), (7, 1, 300, 64, 2), (64, 1, 8192, 128, 0), (65, 40, 700, 32, 5), (300, 60, 200, 64, -20),
    (1024, 3, 400, 32, 0), (1025, 2, 400, 32, -3), (2100, 9, 300, 64, -100), (40, 700, 900, 128, -30)])
def test_plan(B, reqs, most, ctx_most, page, spare):
    """Every result exactly; spare < 0: the ring is short, so some requests are not granted."""
    rs = np.random.RandomState(reqs + most)
    ctx, add = rs.randint(0, ctx_most + 1, reqs), rs.randint(0 if most > 1 else 1, most + 1, reqs)
    up = lambda x: -(-x // page)
    held = up(ctx)
    need = int((up(ctx + add) - held).sum())
    count = max(0, need + spare)
    ring = int(held.sum()) + count + 3
    ids = rs.permutation(ring)
    cols = int(up(ctx + add).max()) + 1
    table = np.full((reqs, cols), -1, np.int32)
    at = count
    for r in range(reqs):
        table[r, :held[r]] = ids[at:at + held[r]]
        at += held[r]
    head = rs.randint(ring)
    free = np.full(ring, -1, np.int32)
    free[(head + np.arange(count)) % ring] = ids[:count]
    rows = int(add.sum())
    check_plan(B, ctx, add, table, free, [head, count], page, rows)
    check_plan(B, ctx, add, table, free, [head, count], page, rows + 5)          # rows behind the last request: -1
    check_plan(B, ctx, add, table, free, [head - ring, count], page, max(0, rows - 3))
    # narrower tables: what does not fit is not granted; some requests end, some are cut
    small = max(1, cols // 2)
    had = ctx.copy()
    kept = np.where(rs.rand(reqs) < 0.3, 0, np.where(rs.rand(reqs) < 0.3, ctx // 2, ctx))
    check_plan(B, kept, np.where(kept < ctx, 0, add), table, free, [head, count], page, rows, had)
    check_plan(B, np.minimum(ctx, small * page), add, table[:, :small], free, [head, count], page, rows)
    # cut and extended in one step: its old pages go back before new entries take their place
    check_plan(B, kept, add, table, free, [head, count], page, rows, had)


@pytest.mark.gpu
def test_plan_odd_values(B):
    t = np.arange(12, dtype=np.int32).reshape(3, 4)
    f = np.arange(20, 28).astype(np.int32)
    check_plan(B, [-5, 0, 64], [3, -2, 1], t, f, [3, 8], 32, 4)                   # negative lengths count as 0
    check_plan(B, [0, 0, 0], [0, 0, 0], t, f, [0, 0], 32, 0)                      # nothing wanted
    check_plan(B, [0, 0, 0], [1, 1, 1], t, f, [5, 99], 32, 3)                     # a count beyond the ring
    check_plan(B, [0, 0, 0], [1, 1, 1], t, f, [5, -4], 32, 3)
    check_plan(B, [128, 10, 10], [1, 0, 1], t, f, [1, 4], 32, 2)                  # a full row of the table
    check_plan(B, [0, 0, 0], [0, 0, 0], t, f, [2, 6], 32, 0, [128, 128, 128])     # more pages back than the ring holds


@pytest.mark.gpu
@pytest.mark.parametrize("places", ["none", "half", "one short", "all"])
@pytest.mark.parametrize("reqs,page", [(2, 32), (40, 64), (300, 32), (1500, 32)])
def test_plan_never_gives_a_page_to_two(B, reqs, page, places):
    """Requests end, are cut and grow in one step, on rings with too few places for what goes back and with enough.  From lists,
    without the ring's arithmetic: a page is held by one request or free once, grants take the free pages in order, and what goes back
    stands behind the rest, as far as there were places that were not free."""
    rs = np.random.RandomState(reqs + len(places))
    up = lambda x: -(-x // page)
    had = rs.randint(0, 9 * page, reqs)
    had[0] = 5 * page
    ctx = np.where(rs.rand(reqs) < 0.4, 0, np.where(rs.rand(reqs) < 0.3, had // 2, had))
    ctx[0] = 0                                                   # one at least ends, one at least grows
    add = np.where(rs.rand(reqs) < 0.5, rs.randint(0, 4 * page, reqs), 0)
    add[-1] = 3 * page
    had[-1] = ctx[-1] = min(had[-1], 4 * page)
    cols = int(max(up(had).max(), up(ctx + add).max()))
    held = up(had)
    back_n, count = int(np.maximum(held - up(ctx), 0).sum()), int((up(ctx + add) - up(ctx)).sum()) + 2
    ring = count + {"none": 0, "half": back_n // 2, "one short": back_n - 1, "all": back_n}[places]
    ids = rs.permutation(int(held.sum()) + count)
    table = np.full((reqs, cols), -1, np.int32)
    at = count
    for r in range(reqs):
        table[r, :held[r]] = ids[at:at + held[r]]
        at += held[r]
    head = rs.randint(ring)
    free = np.full(ring, -1, np.int32)
    free[(head + np.arange(count)) % ring] = ids[:count]
    was_free = ids[:count].tolist()
    back = [int(table[r, c]) for r in range(reqs) for c in range(up(ctx[r]), held[r])]
    d = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
    t, f = d(table), d(free)
    p = B.plan(d(ctx), d(add), t, f, d([head, count]), page=page, rows=int(add.sum()), had=d(had))
    t, f, lens, state = t.cpu().numpy(), f.cpu().numpy(), p.lens.cpu().numpy(), p.state.cpu().tolist()
    assert np.array_equal(lens, ctx + add) and p.status.cpu().tolist() == [count - 2, 0]
    new = [int(t[r, c]) for r in range(reqs) for c in range(up(ctx[r]), up(lens[r]))]
    kept = [int(t[r, c]) for r in range(reqs) for c in range(up(ctx[r]))]
    assert kept == [int(table[r, c]) for r in range(reqs) for c in range(up(ctx[r]))]
    assert new == was_free[:count - 2]
    now_free = f[(state[0] + np.arange(state[1])) % ring].tolist()
    assert len(set(kept + new + now_free)) == len(kept + new + now_free)
    assert now_free == was_free[count - 2:] + back[:ring - count]


@pytest.mark.gpu
def test_plan_in_place_step_by_step(B):
    """The state and the lengths updated in place over many steps; every page is held once at all times."""
    page, reqs, pages = 32, 5, 40
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    table = torch.full((reqs, 12), -1, dtype=torch.int32, device=DEV)
    free, state, lens = torch.arange(pages, dtype=torch.int32, device=DEV), i([0, pages]), i([0] * reqs)
    rs = np.random.RandomState(3)
    had = None
    for step in range(60):
        add = rs.randint(0, 30, reqs)
        before = lens.cpu().numpy()
        if step % 7 == 6:
            gone = rs.rand(reqs) < 0.5
            had = lens.clone()
            lens.copy_(i(np.where(gone, 0, before)))
            add = np.where(gone, 0, add)
            before = lens.cpu().numpy()
        else:
            had = None
        rows = int(add.sum())
        out = B.Plan(torch.empty(reqs + 1, dtype=torch.int32, device=DEV), lens, torch.empty(reqs, dtype=torch.int32, device=DEV),
                     torch.empty(rows, dtype=torch.int32, device=DEV), state, torch.empty(2, dtype=torch.int32, device=DEV))
        p = B.plan(lens, i(add), table, free, state, page=page, rows=rows, had=had, out=out)
        now, tb, st = lens.cpu().numpy(), table.cpu().numpy(), state.cpu().numpy()
        start = p.start.cpu().numpy()
        assert np.array_equal(now, np.where(start >= 0, before + add, before))
        held = [tb[r, c] for r in range(reqs) for c in range(-(-now[r] // page))]
        left = free.cpu().numpy()[(st[0] + np.arange(st[1])) % pages].tolist()
        assert sorted(held + left) == list(range(pages))


# --------------------------------------------------------------------------------------------------------- append and gather
def check_pool(pool, plain, touched=None):
    k, v = load_keys(pool.k.cpu().numpy()), load_values(pool.v.cpu().numpy())
    pages = range(plain.pages) if touched is None else touched
    for pg in pages:
        assert np.array_equal(k[pg], plain.codes["k"][pg]), ("k", pg)
        assert np.array_equal(v[pg], plain.codes["v"][pg]), ("v", pg)
    assert np.array_equal(pool.k_scale.cpu().numpy(), plain.scale["k"])
    assert np.array_equal(pool.v_scale.cpu().numpy(), plain.scale["v"])


def dense(rs, rows, heads, dim, kind, spread=1.0):
    x = rs.standard_normal((rows, heads, dim)) * np.exp(rs.standard_normal((rows, 1, 1)) * spread)
    return torch.from_numpy(x.astype(np.float32)).to(TYPES[kind])


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("page,heads,dim", [(32, 1, 32), (64, 2, 64), (128, 3, 128), (128, 2, 32), (32, 2, 128)])
def test_append_exactly(B, code, kind, page, heads, dim):
    """Codes and scales bit for bit over several calls: whole pages, pieces that raise a page's scale, single tokens, skipped
    rows, pages in another order than the rows."""
    rs = np.random.RandomState(page + dim)
    pages = 9
    plain = random_pool(rs, pages, heads, dim, page, code)
    pool = plain.to_device(B)
    order = rs.permutation(pages)
    fill = np.zeros(pages, int)
    for step, lens in enumerate(([page, page // 2, 1, 5], [3, 33 % page, 1], [1], [page - 1, 7, 2], [1, 1, 1, 1, 1])):
        slots = []
        for j, n in enumerate(lens):
            pg = order[(2 * step + j) % pages]
            n = min(n, page - fill[pg])
            slots += [pg * page + fill[pg] + t for t in range(n)] + [-1] * (j % 2)
            fill[pg] += n
        slots += [pages * page, pages * page + 7, -9]
        k, v = dense(rs, len(slots), heads, dim, kind), dense(rs, len(slots), heads, dim, kind)
        skipped = np.array([not 0 <= s < pages * page for s in slots])
        k[skipped], v[skipped] = math.nan, math.inf                          # not read
        plain.append(to_np(k), to_np(v), slots)
        B.append(pool, k.to(DEV), v.to(DEV), torch.tensor(slots, dtype=torch.int32, device=DEV))
        check_pool(pool, plain)


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_append_values_that_are_not_ordinary(B, code):
    """NaN becomes 0 and an infinity the largest code without touching the scale; zero rows; the smallest and largest numbers."""
    rs = np.random.RandomState(5)
    page, heads, dim = 64, 2, 32
    plain = PlainPool(6, heads, dim, page, code)
    pool = plain.to_device(B)
    k, v = dense(rs, 40, heads, dim, "fp32"), dense(rs, 40, heads, dim, "fp32")
    k[3, 0, 5], k[4, 1, :] = math.nan, math.inf
    v[0, 0, 0], v[7, 1, 3], v[8, 1, 4] = -math.inf, math.nan, math.inf
    k[10:14], v[10:14] = 0.0, 0.0
    k[14:16] *= 1e-38
    v[14:16] *= 1e-44
    k[16:18] *= 1e37
    slots = list(range(0, 10)) + list(range(64, 68)) + [128, 129] + [192, 193] + list(range(10, 32))
    plain.append(to_np(k), to_np(v), slots)
    B.append(pool, k.to(DEV), v.to(DEV), torch.tensor(slots, dtype=torch.int32, device=DEV))
    check_pool(pool, plain)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [300, 6000])
def test_append_rows_in_any_order(B, rows):
    """Rows shuffled, slots named twice (the last row counts), gaps, pages reached by many runs; on both sides of the row count
    at which pages are marked beforehand."""
    rs = np.random.RandomState(rows)
    page, heads, dim = 32, 1, 32
    pages = rows // page + 6
    plain = random_pool(rs, pages, heads, dim, page, "int8")
    pool = plain.to_device(B)
    for step in range(3):
        slots = rs.permutation(pages * page)[:rows]
        if step == 1:                                       # runs, some pages cut in two, neighbouring pages swapped
            slots = np.sort(slots)
            slots = np.concatenate([slots[rows // 2:], slots[:rows // 2]])
        slots[rs.randint(0, rows, rows // 10)] = slots[rs.randint(0, rows, rows // 10)]
        slots[rs.randint(0, rows, 5)] = -1
        k, v = dense(rs, rows, heads, dim, "fp16"), dense(rs, rows, heads, dim, "fp16")
        plain.append(to_np(k), to_np(v), slots)
        B.append(pool, k.to(DEV), v.to(DEV), torch.tensor(slots, dtype=torch.int32, device=DEV))
        check_pool(pool, plain)


@pytest.mark.gpu
def test_append_strided_inputs_and_gather_layouts(B):
    """Keys and values as slices of one projection, heads transposed; gather in every type, with slots outside the pool."""
    rs = np.random.RandomState(6)
    page, heads, dim, rows = 64, 4, 64, 77
    for code in ("int8", "e4m3"):
        plain = PlainPool(4, heads, dim, page, code)
        pool = plain.to_device(B)
        both = torch.from_numpy(rs.standard_normal((rows, 3 * heads * dim + 5)).astype(np.float32)).to(torch.bfloat16).to(DEV)
        k = both[:, 5:5 + heads * dim].view(rows, heads, dim)
        v = torch.from_numpy(rs.standard_normal((heads, rows, dim)).astype(np.float32)).to(torch.bfloat16).to(DEV).transpose(0, 1)
        slots = np.concatenate([np.arange(128, 192), np.arange(0, 13)])
        plain.append(to_np(k), to_np(v), slots)
        B.append(pool, k, v, torch.tensor(slots, dtype=torch.int32, device=DEV))
        check_pool(pool, plain)
        ask = np.array([128, 5, -1, 191, 4 * page, 12, 12, 2 ** 31 - 1, 0, -2 ** 31])
        pages, offs = np.where((ask >= 0) & (ask < 4 * page), ask, 0) // page, np.where((ask >= 0) & (ask < 4 * page), ask, 0) % page
        on = ((ask >= 0) & (ask < 4 * page))[:, None, None]
        for kind, t in TYPES.items():
            got = B.gather(pool, torch.tensor(ask, dtype=torch.int32, device=DEV), t)
            for w, g in zip("kv", got):
                val = (decode(plain.codes[w], code).astype(np.float32) * plain.scale[w][:, None, :, None])[pages, offs] * on
                assert torch.equal(g.cpu(), torch.from_numpy(val.astype(np.float32)).to(t)), (w, kind)


# ------------------------------------------------------------------------------------------------------------------ attend
def check_attend(B, plain, q, cu, lens, table, causal, kind, pool=None, max_q=None, scale=None, **kw):
    pool = pool or plain.to_device(B)
    scale_f = 1 / math.sqrt(plain.dim) if scale is None else scale
    want, wlse, mean, most = attend64(plain, q.double().numpy(), cu, lens, table, causal, scale_f)
    i = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
    out, lse = B.attend(pool, q.to(DEV), i(cu), i(lens), i(table), causal=causal, with_lse=True, max_q=max_q, scale=scale, **kw)
    tol, tol_lse = attend_tolerance(kind, plain.dim, want, wlse, mean, most)
    got, glse = out.detach().cpu().double().numpy(), lse.cpu().double().numpy()
    assert np.array_equal(np.isfinite(wlse), np.isfinite(glse))
    if kind == "fp16":      # results from 65520 on round to infinity in fp16
        over = np.isinf(got) & (np.abs(want) + tol >= 65520) & (np.sign(got) == np.sign(want))
        got = np.where(over, want, got)
    bad = int((~(np.abs(got - want) <= tol)).sum())
    assert bad == 0, f"{bad} of {got.size} off, by {np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-300)):.3g} tolerances"
    on = np.isfinite(wlse)
    worst = (np.abs(glse[on] - wlse[on]) / tol_lse[on]).max(initial=0)
    assert worst <= 1, f"lse off by {worst:.3g} tolerances"
    return out, lse


CASES = [  # (rows of each request), (tokens of each), causal
    ([1], [1], True), ([1], [129], True), ([1, 1, 1], [31, 32, 33], True), ([2, 0, 3, 1], [5, 70, 0, 64], False),
    ([5], [3], True), ([1] * 9, [0, 1, 2, 63, 64, 65, 127, 128, 200], True), ([17, 1, 40], [17, 300, 40], True), ([33], [100], False),
    ([1], [1500], True), ([3, 1], [700, 1300], True), ([70, 2], [90, 1100], True)]


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("page,heads,group,dim", [(32, 2, 1, 32), (64, 1, 4, 64), (128, 2, 3, 128)])
def test_attend(B, code, kind, case, page, heads, group, dim):
    n, lens, causal = CASES[case]
    rs = np.random.RandomState(case * 7 + dim)
    pages = sum(-(-x // page) for x in lens) + 3
    plain = random_pool(rs, pages, heads, dim, page, code)
    cu = np.concatenate([[0], np.cumsum(n)])
    q = dense(rs, int(cu[-1]), heads * group, dim, kind, 0.5) * 2
    check_attend(B, plain, q, cu, lens, make_table(rs, lens, page, pages), causal, kind)


LONG = [  # requests of more rows than the narrow kernel takes, beside short ones; the last ones are divided over the tokens
    ([300], [300], True), ([257, 3], [400, 90], True), ([1, 385, 0, 40], [77, 385, 50, 200], True), ([270], [100], False),
    ([300, 300], [64, 0], False), ([260], [5000], True), ([400], [3], True), ([513, 2], [2500, 3100], False)]


@pytest.mark.gpu
@pytest.mark.parametrize("code,kind", [("int8", "fp32"), ("int8", "bf16"), ("e4m3", "fp16"), ("e4m3", "fp32")])
@pytest.mark.parametrize("case", range(len(LONG)))
@pytest.mark.parametrize("page,heads,group,dim", [(32, 2, 1, 32), (64, 1, 2, 64), (128, 1, 1, 128), (32, 1, 3, 128)])
def test_attend_long_requests(B, code, kind, case, page, heads, group, dim):
    n, lens, causal = LONG[case]
    rs = np.random.RandomState(case * 5 + dim + page)
    pages = sum(-(-x // page) for x in lens) + 3
    plain = random_pool(rs, pages, heads, dim, page, code)
    cu = np.concatenate([[0], np.cumsum(n)])
    q = dense(rs, int(cu[-1]), heads * group, dim, kind, 0.5) * 2
    check_attend(B, plain, q, cu, lens, make_table(rs, lens, page, pages), causal, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_attend_long_requests_absent_pages_and_nan_codes(B, code):
    """The wide kernel's masks: codes behind the last token are NaN (e4m3), pages of the table are missing, whole stages of them."""
    rs = np.random.RandomState(31)
    page, dim = 32, 64
    plain = random_pool(rs, 30, 1, dim, page, code)
    lens, n = [300, 81], [300, 280]
    table = make_table(rs, lens, page, 30, cols=11)
    cu = np.array([0, 300, 580])
    q = dense(rs, 580, 1, dim, "bf16", 0.5)
    pool = plain.to_device(B)
    if code == "e4m3":
        k, v = load_keys(pool.k.cpu().numpy()), load_values(pool.v.cpu().numpy())
        for r, ln in enumerate(lens):
            if ln % page:
                k[table[r, ln // page], ln % page:], v[table[r, ln // page], ln % page:] = 0x7f, 0xff
        pool.k.copy_(torch.from_numpy(store_keys(k)))
        pool.v.copy_(torch.from_numpy(store_values(v)))
    check_attend(B, plain, q, cu, lens, table, False, "bf16", pool=pool)
    i = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
    t2 = table.copy()
    for gone, bad in ((1, -1), (2, 30), (3, -2 ** 31), (4, 2 ** 31 - 1), (5, -1), (8, -7)):
        t2[0, gone] = bad
    left = [c for c in range(10) if t2[0, c] == table[0, c]]
    kk = table.copy()
    kk[0, :len(left)] = table[0, left]
    want, wl, mean, most = attend64(plain, q.double().numpy(), cu, [32 * (len(left) - 1) + 300 % 32, 81], kk, False, 1 / math.sqrt(dim))
    got = B.attend(pool, q.to(DEV), i(cu), i(lens), i(t2), causal=False)
    tol, _ = attend_tolerance("bf16", dim, want, wl, mean, most)
    assert (np.abs(got.cpu().double().numpy() - want) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n,lens", [([2, 1], [300, 900]), ([300, 4], [700, 1200])])
def test_attend_rows_that_are_nan_or_infinite_stay_alone(B, n, lens):
    """A query row with NaN or infinities is its own affair; the others get what they get without it."""
    rs = np.random.RandomState(32)
    plain = random_pool(rs, 50, 1, 64, 64, "int8")
    cu = np.concatenate([[0], np.cumsum(n)])
    table = make_table(rs, lens, 64, 50)
    i = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
    for kind in TYPES:
        q = dense(rs, int(cu[-1]), 2, 64, kind, 0.5).to(DEV)
        pool = plain.to_device(B)
        want = B.attend(pool, q, i(cu), i(lens), i(table), causal=False)
        q[1, 0, 3], q[-1, 1, 7], q[0, 1, 0] = math.nan, math.inf, -math.inf
        got = B.attend(pool, q, i(cu), i(lens), i(table), causal=False)
        for r, h in ((1, 0), (cu[-1] - 1, 1), (0, 1)):
            assert torch.isnan(got[r, h]).any()
            got[r, h] = want[r, h]
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_attend_overlapping_requests_stay_in_bounds(B):
    """Row offsets that go back and forth are nobody's rows twice over: what is written is unspecified, where is not."""
    rs = np.random.RandomState(33)
    plain = random_pool(rs, 80, 1, 32, 32, "int8")
    lens = [2000] * 7
    table = np.tile(rs.permutation(80)[:63].astype(np.int32), (7, 1))
    i = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
    for rows, hint in ((40, 1), (40, 40), (600, 600)):
        q = dense(rs, rows, 2, 32, "fp16", 0.5).to(DEV)
        big = torch.full((rows + 64, 2, 32), 5.0, dtype=torch.float16, device=DEV)
        B.attend(plain.to_device(B), q, i([0, rows, 0, rows, 3, rows - 2, -8, 10 ** 9]), i(lens), i(table), max_q=hint, out=big[32:32 + rows])
        assert torch.all(big[:32] == 5) and torch.all(big[32 + rows:] == 5)


@pytest.mark.gpu
def test_attend_captured_with_every_kernel_and_replayed(B):
    """More than 64 requests, short and long ones: every launch of the read in one graph, replayed with other lengths in between."""
    rs = np.random.RandomState(34)
    reqs = 70
    n = rs.randint(0, 3, reqs)
    n[10], n[20] = 300, 40
    lens = rs.randint(0, 200, reqs)
    lens[10], lens[30] = 700, 1500
    plain = random_pool(rs, 400, 1, 64, 64, "int8")
    pool = plain.to_device(B)
    cu = np.concatenate([[0], np.cumsum(n)])
    i = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
    table, q, dlens, dcu = i(rs.randint(0, 400, (reqs, 24))), dense(rs, int(cu[-1]), 2, 64, "fp16", 0.5).to(DEV), i(lens), i(cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        B.attend(pool, q, dcu, dlens, table, with_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, z = B.attend(pool, q, dcu, dlens, table, with_lse=True)
    for step in range(6):
        dlens.copy_(i(rs.permutation(lens)))
        q.copy_(dense(rs, int(cu[-1]), 2, 64, "fp16", 0.5))
        g.replay()
        torch.cuda.synchronize()
        o2, z2 = B.attend(pool, q, dcu, dlens, table, with_lse=True)
        assert torch.equal(o, o2) and torch.equal(z, z2)
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("group", [1, 2, 5, 7, 8, 16, 33])
def test_attend_groups(B, group):
    """Groups that do not divide a row tile, and one that exceeds it."""
    rs = np.random.RandomState(group)
    plain = random_pool(rs, 12, 2, 64, 64, "int8")
    n, lens = [3, 1, 9], [120, 333, 40]
    cu = np.concatenate([[0], np.cumsum(n)])
    q = dense(rs, int(cu[-1]), 2 * group, 64, "fp16", 0.5)
    check_attend(B, plain, q, cu, lens, make_table(rs, lens, 64, 12), True, "fp16")


@pytest.mark.gpu
@pytest.mark.parametrize("reqs", [63, 64, 65, 130, 1100, 4200])
def test_attend_many_requests(B, reqs):
    rs = np.random.RandomState(reqs)
    lens = rs.randint(0, 90, reqs)
    lens[reqs // 2] = 900
    n = rs.randint(0, 3, reqs)
    pages = int(sum(-(-x // 32) for x in lens)) + 1
    plain = random_pool(rs, pages, 1, 32, 32, "e4m3")
    cu = np.concatenate([[0], np.cumsum(n)])
    q = dense(rs, int(cu[-1]), 2, 32, "bf16", 0.5)
    check_attend(B, plain, q, cu, lens, make_table(rs, lens, 32, pages), True, "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
def test_attend_wide_scores_and_sizes(B, kind):
    """Scores of hundreds (one token takes all), tiny and huge queries, page scales far apart (a page of zeros among them)."""
    rs = np.random.RandomState(11)
    plain = random_pool(rs, 8, 2, 64, 32, "int8")
    plain.scale["v"][1] *= 1e6
    plain.scale["v"][2] = 1e-30
    plain.codes["v"][2] = 128
    plain.scale["k"][3] *= 30
    plain.scale["v"][4] *= 1e-7
    lens, n = [250], [7]
    cu = np.array([0, 7])
    q = dense(rs, 7, 2, 64, kind, 0.3)
    q[1] *= 200
    q[2] *= 1e-6
    q[3] = 0
    if kind != "fp16":
        q[4] *= 1e-30
        q[5] *= 1e5
    check_attend(B, plain, q, cu, lens, make_table(rs, lens, 32, 8), False, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
def test_attend_never_reads_what_is_not_there(B, causal):
    """Codes behind a request's last token and pages outside the pool: NaN codes, NaN scales, entries -1 and beyond the pool."""
    rs = np.random.RandomState(12)
    page, dim = 64, 64
    plain = random_pool(rs, 9, 2, dim, page, "e4m3")
    lens, n = [70, 33, 129], [2, 1, 3]
    table = make_table(rs, lens, page, 9, cols=5)
    used = {int(x) for x in table.ravel() if x >= 0}
    cu = np.array([0, 2, 3, 6])
    q = dense(rs, 6, 4, dim, "bf16", 0.5)
    pool = plain.to_device(B)
    k, v = load_keys(pool.k.cpu().numpy()), load_values(pool.v.cpu().numpy())
    for r, ln in enumerate(lens):
        pg = table[r, ln // page]
        k[pg, ln % page:], v[pg, ln % page:] = 0x7f, 0xff
    for pg in range(9):
        if pg not in used:
            k[pg], v[pg] = 0x7f, 0x7f
            pool.k_scale[pg] = math.nan
            pool.v_scale[pg] = math.nan
    pool.k.copy_(torch.from_numpy(store_keys(k)))
    pool.v.copy_(torch.from_numpy(store_values(v)))
    check_attend(B, plain, q, cu, lens, table, causal, "bf16", pool=pool)
    # a page outside the pool stands for one that nobody sees: as if its tokens were left out (non-causal: order does not matter)
    if not causal:
        for bad in (-1, 9, 2 ** 31 - 1, -2 ** 31):
            t2 = table.copy()
            gone = t2[2, 0]
            t2[2, 0] = bad
            i = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
            got = B.attend(pool, q.to(DEV), i(cu), i(lens), i(t2), causal=False)
            kk = table.copy()
            kk[2, :2] = kk[2, 1:3]
            want, wl, mean, most = attend64(plain, q.double().numpy(), cu, [70, 33, 65], kk, False, 1 / math.sqrt(dim))
            tol, _ = attend_tolerance("bf16", dim, want, wl, mean, most)
            assert (np.abs(got.cpu().double().numpy() - want) <= tol).all() and gone >= 0


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,group", [(1, 1), (9, 2), (300, 1), (130, 4)])
def test_attend_beside_pages_of_nan_codes(B, n, group, causal):
    """Every page that no request names holds NaN codes and scales, the first one among them: absent pages, the last tile of a part and
    the token behind the last one read nothing of them, in every kernel."""
    rs = np.random.RandomState(n)
    page, dim, pages = 32, 32, 40
    plain = random_pool(rs, pages, 1, dim, page, "e4m3")
    lens = [n + 289, n + 257]
    held = [-(-x // page) for x in lens]
    ids = 1 + rs.permutation(pages - 1)[:sum(held)]
    table = np.full((2, max(held) + 2), -1, np.int64)
    table[0, :held[0]], table[1, :held[1]] = ids[:held[0]], ids[held[0]:]
    cu = np.array([0, n, 2 * n])
    q = dense(rs, 2 * n, group, dim, "bf16", 0.5)
    pool = plain.to_device(B)
    k, v = load_keys(pool.k.cpu().numpy()), load_values(pool.v.cpu().numpy())
    for r, ln in enumerate(lens):
        if ln % page:
            k[table[r, ln // page], ln % page:], v[table[r, ln // page], ln % page:] = 0x7f, 0xff
    for pg in set(range(pages)) - set(ids.tolist()):
        k[pg], v[pg] = 0x7f, 0x7f
        pool.k_scale[pg] = math.nan
        pool.v_scale[pg] = math.nan
    pool.k.copy_(torch.from_numpy(store_keys(k)))
    pool.v.copy_(torch.from_numpy(store_values(v)))
    check_attend(B, plain, q, cu, lens, table, causal, "bf16", pool=pool)
    i = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
    t2 = table.copy()
    t2[0, 1], t2[1, 4] = -1, pages
    if not causal:                                     # as if the tokens of the absent pages were left out
        kk = np.full_like(table, -1)
        kk[0, :held[0] - 1], kk[1, :held[1] - 1] = np.delete(table[0, :held[0]], 1), np.delete(table[1, :held[1]], 4)
        want, wl, mean, most = attend64(plain, q.double().numpy(), cu, [x - page for x in lens], kk, False, 1 / math.sqrt(dim))
        tol, _ = attend_tolerance("bf16", dim, want, wl, mean, most)
        got = B.attend(pool, q.to(DEV), i(cu), i(lens), i(t2), causal=False)
        assert (np.abs(got.cpu().double().numpy() - want) <= tol).all()
    else:
        assert torch.isfinite(B.attend(pool, q.to(DEV), i(cu), i(lens), i(t2), causal=True)).all()


@pytest.mark.gpu
def test_attend_lengths_beyond_the_table_and_odd_offsets(B):
    """Lengths are limited to the table's row, row offsets to the rows; rows that belong to nobody are left as they were."""
    rs = np.random.RandomState(13)
    plain = random_pool(rs, 6, 1, 32, 32, "int8")
    table = make_table(rs, [64, 64], 32, 6, cols=2)
    i = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
    q = dense(rs, 6, 2, 32, "fp32", 0.5)
    pool = plain.to_device(B)
    out = torch.full((6, 2, 32), 7.0, device=DEV)
    lse = torch.full((6, 2), 7.0, device=DEV)
    B.attend(pool, q.to(DEV), i([0, 2, 4]), i([64, 64]), i(table), causal=False, out=out, lse=lse)
    assert torch.all(out[4:] == 7) and torch.all(lse[4:] == 7) and torch.all(out[:4] != 7)
    again = torch.full((6, 2, 32), 7.0, device=DEV)
    B.attend(pool, q.to(DEV), i([0, 2, 4]), i([10 ** 9, 65]), i(table), causal=False, out=again)
    assert torch.equal(out, again)
    again.fill_(7.0)
    B.attend(pool, q.to(DEV), i([0, 2, 100]), i([-3, 64]), i(table), causal=False, out=again)     # rows 2 .. 5 of request 1
    assert torch.all(again[:2] == 0) and torch.equal(again[2:4], out[2:4]) and torch.all(again[4:] != 7)
    again.fill_(7.0)
    B.attend(pool, q.to(DEV), i([4, 2, -1]), i([64, 64]), i(table), causal=False, out=again)      # no rows
    assert torch.all(again == 7)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
def test_attend_strides_and_given_results(B, kind):
    """Queries as a slice of one projection at an odd offset (not 16-byte aligned), results into a wider tensor, heads first."""
    rs = np.random.RandomState(14)
    heads, group, dim, rows = 2, 2, 64, 5
    plain = random_pool(rs, 12, heads, dim, 64, "int8")
    lens, cu = [300, 200], np.array([0, 3, 5])
    table = make_table(rs, lens, 64, 12)
    hq = heads * group
    wide = torch.zeros(rows, hq * dim + 3, dtype=TYPES[kind], device=DEV)
    q = dense(rs, rows, hq, dim, kind, 0.5)
    wide[:, 3:] = q.reshape(rows, -1).to(DEV)
    i = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
    pool = plain.to_device(B)
    base, lse0 = check_attend(B, plain, q, cu, lens, table, True, kind, pool=pool)
    out = torch.full((rows, hq * dim + 1), 9.0, dtype=TYPES[kind], device=DEV)
    B.attend(pool, wide[:, 3:].view(rows, hq, dim), i(cu), i(lens), i(table), out=out[:, 1:].view(rows, hq, dim))
    assert torch.equal(out[:, 1:].reshape(rows, hq, dim), base) and torch.all(out[:, 0] == 9)
    turned = torch.empty(hq, rows, dim, dtype=TYPES[kind], device=DEV)
    qt = q.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    B.attend(pool, qt, i(cu), i(lens), i(table), out=turned.transpose(0, 1))
    assert torch.equal(turned.transpose(0, 1), base)
    wt = torch.full((2, 9), -1, dtype=torch.int32, device=DEV)
    wt[:, :table.shape[1]] = i(table)
    assert torch.equal(B.attend(pool, q.to(DEV), i(cu), i(lens), wt[:, :table.shape[1]]), base)


@pytest.mark.gpu
def test_attend_results_do_not_depend_on_hints_or_neighbours(B):
    """The same rows alone and in a batch: the batch decides the split, so up to fp32 roundings; twice the same call: bit for bit;
    with other max_q hints: within tolerance."""
    rs = np.random.RandomState(15)
    plain = random_pool(rs, 40, 2, 64, 64, "int8")
    lens, n = [1100, 40, 600], [40, 1, 2]
    cu = np.concatenate([[0], np.cumsum(n)])
    table = make_table(rs, lens, 64, 40)
    q = dense(rs, int(cu[-1]), 4, 64, "fp16", 0.5)
    pool = plain.to_device(B)
    a, la = check_attend(B, plain, q, cu, lens, table, True, "fp16", pool=pool)
    b, lb = check_attend(B, plain, q, cu, lens, table, True, "fp16", pool=pool)
    assert torch.equal(a, b) and torch.equal(la, lb)
    for hint in (0, 1, 40, 10 ** 6):
        check_attend(B, plain, q, cu, lens, table, True, "fp16", pool=pool, max_q=hint)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "fp32"])
def test_attend_each_request_alone(B, kind):
    """A batch whose requests go to the narrow and the wide kernel, and each of its requests in a call of its own: the division differs,
    both are within tolerance of the 64-bit result."""
    rs = np.random.RandomState(17)
    plain = random_pool(rs, 60, 2, 64, 64, "e4m3")
    lens, n = [1100, 40, 600, 450, 7], [40, 1, 2, 300, 0]
    cu = np.concatenate([[0], np.cumsum(n)])
    table = make_table(rs, lens, 64, 60)
    q = dense(rs, int(cu[-1]), 4, 64, kind, 0.5)
    pool = plain.to_device(B)
    check_attend(B, plain, q, cu, lens, table, True, kind, pool=pool)
    for r, rows in enumerate(n):
        if rows:
            check_attend(B, plain, q[cu[r]:cu[r + 1]], [0, rows], lens[r:r + 1], table[r:r + 1], True, kind, pool=pool)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hint", [(40, 1), (40, 40), (600, 600)])
def test_attend_many_overlapping_requests_stay_in_bounds(B, rows, hint):
    """More than 64 requests (the division is looked up) whose row offsets go back and forth: what is written is unspecified, where is
    not."""
    rs = np.random.RandomState(rows + hint)
    reqs = 70
    pool = random_pool(rs, 80, 1, 32, 32, "int8").to_device(B)
    i = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
    table = i(np.tile(rs.permutation(80)[:63], (reqs, 1)))
    cu = rs.randint(-20, rows + 20, reqs + 1)
    cu[::2] = 0
    cu[5], cu[-1] = 10 ** 9, rows
    q = dense(rs, rows, 2, 32, "fp16", 0.5).to(DEV)
    big = torch.full((rows + 64, 2, 32), 5.0, dtype=torch.float16, device=DEV)
    sums = torch.full((rows + 64, 2), 5.0, device=DEV)
    B.attend(pool, q, i(cu), i(rs.randint(0, 2017, reqs)), table, max_q=hint, causal=False, out=big[32:32 + rows], lse=sums[32:32 + rows])
    for t in (big, sums):
        assert torch.all(t[:32] == 5) and torch.all(t[32 + rows:] == 5)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(B):
    """A pool of more than 4 GiB of codes: pages at its end written, read back and attended to."""
    heads, dim, page = 8, 128, 128
    pages = (1 << 32) // (heads * dim * page) + 40
    pool = B.Pool.empty(pages, heads, dim, page, "int8", DEV)
    assert pool.k.numel() > 1 << 32
    rs = np.random.RandomState(16)
    ids = [pages - 1, 3, pages - 7]
    small = PlainPool(3, heads, dim, page, "int8")
    rows = 300
    k, v = dense(rs, rows, heads, dim, "fp16", 0.3), dense(rs, rows, heads, dim, "fp16", 0.3)
    slots = np.array([ids[t // page] * page + t % page for t in range(rows)])
    small.append(to_np(k), to_np(v), np.arange(rows))
    i = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
    B.append(pool, k.to(DEV), v.to(DEV), i(slots))
    assert np.array_equal(load_keys(pool.k[ids].cpu().numpy()), small.codes["k"])
    assert np.array_equal(load_values(pool.v[ids].cpu().numpy()), small.codes["v"])
    got = B.gather(pool, i(slots), torch.float32)
    for w, g in zip("kv", got):
        val = decode(small.codes[w], "int8").astype(np.float32) * small.scale[w][:, None, :, None]
        assert np.array_equal(g.cpu().numpy(), val.reshape(-1, heads, dim)[:rows])
    q = dense(rs, 2, heads, dim, "fp16", 0.3)
    want, wl, mean, most = attend64(small, q.double().numpy(), [0, 2], [rows], [[0, 1, 2]], True, 1 / math.sqrt(dim))
    tol, _ = attend_tolerance("fp16", dim, want, wl, mean, most)
    out = B.attend(pool, q.to(DEV), i([0, 2]), i([rows]), i([ids]))
    assert (np.abs(out.cpu().double().numpy() - want) <= tol).all()


# ------------------------------------------------------------------------------------------------------------ used together
def _generate(B, code, kind, capture):
    """Prompts, then single tokens, one request ending on the way and another taking its pages: the steps a serving loop makes.
    Every step's output against 64-bit attention over what the plain pool holds; with `capture`, the single-token step is
    recorded once and replayed, every replay equal to the eager step on a copy."""
    rs = np.random.RandomState(21)
    page, heads, group, dim, reqs, pages, cols = 32, 2, 2, 32, 3, 14, 6
    pool = B.Pool.empty(pages, heads, dim, page, code, DEV)
    plain = PlainPool(pages, heads, dim, page, code)
    i = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
    table = torch.full((reqs, cols), -1, dtype=torch.int32, device=DEV)
    free, state, lens = torch.arange(pages, dtype=torch.int32, device=DEV), i([0, pages]), torch.zeros(reqs, dtype=torch.int32, device=DEV)

    def step(add, k, v, q, had=None, out=None):
        p = B.plan(lens, add, table, free, state, page=page, rows=k.shape[0], had=had, out=out)
        B.append(pool, k, v, p.slots)
        return p, B.attend(pool, q, p.cu, p.lens, table, max_q=k.shape[0], out=None)

    def check(p, o, k, v, q):
        cu, ln, tb = p.cu.cpu().numpy(), p.lens.cpu().numpy(), table.cpu().numpy()
        plain.append(to_np(k), to_np(v), p.slots.cpu().numpy())
        want, wl, mean, most = attend64(plain, q.double().cpu().numpy(), cu, ln, tb, True, 1 / math.sqrt(dim))
        tol, _ = attend_tolerance(kind, dim, want, wl, mean, most)
        assert (np.abs(o.cpu().double().numpy() - want) <= tol).all()
        check_pool(pool, plain)

    def inputs(n):
        return [dense(rs, n, h, dim, kind, 0.4).to(DEV) for h in (heads, heads, heads * group)]

    for add, keep in (([40, 1, 70], None), ([5, 33, 2], None), ([0, 20, 1], [False, True, True]), ([64, 1, 1], None)):
        had = None
        if keep is not None:
            had = lens.clone()
            lens.mul_(i([int(x) for x in keep]))
        k, v, q = inputs(sum(add))
        p, o = step(i(add), k, v, q, had)
        check(p, o, k, v, q)
        assert p.status.cpu().tolist()[1] == 0
        lens.copy_(p.lens)
        state.copy_(p.state)
    if not capture:
        for _ in range(4):
            k, v, q = inputs(reqs)
            p, o = step(i([1] * reqs), k, v, q)
            check(p, o, k, v, q)
            lens.copy_(p.lens)
            state.copy_(p.state)
        return
    k, v, q = inputs(reqs)
    one = i([1] * reqs)
    e = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)
    plan_out = B.Plan(e(reqs + 1), lens, e(reqs), e(reqs), state, e(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    saved = [t.clone() for t in (lens, state, table, free, pool.k, pool.v, pool.k_scale, pool.v_scale)]
    with torch.cuda.stream(side):
        step(one, k, v, q, out=plan_out)                      # warm-up
    torch.cuda.current_stream().wait_stream(side)
    for t, s in zip((lens, state, table, free, pool.k, pool.v, pool.k_scale, pool.v_scale), saved):
        t.copy_(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p, o = step(one, k, v, q, out=plan_out)
    for _ in range(12):
        for t, x in zip((k, v, q), inputs(reqs)):
            t.copy_(x)
        g.replay()
        torch.cuda.synchronize()
        check(p, o, k, v, q)
        o2 = B.attend(pool, q, p.cu, p.lens, table)           # eager work between replays
        assert torch.equal(o, o2)


@pytest.mark.gpu
@pytest.mark.parametrize("code,kind", [("int8", "fp32"), ("int8", "bf16"), ("e4m3", "fp16")])
def test_steps_of_a_serving_loop(B, code, kind):
    _generate(B, code, kind, False)


@pytest.mark.gpu
@pytest.mark.parametrize("code,kind", [("int8", "fp16"), ("e4m3", "fp32")])
def test_a_captured_step_replayed(B, code, kind):
    _generate(B, code, kind, True)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("most", [4, 300])
def test_rows_of_requests_that_were_not_granted_see_nothing(B, most, causal):
    """A step on a short ring, eager and captured: with plan's `start` the rows of a request that found no page get 0 and -inf, all
    others what the 64-bit attention gives; the same graph replayed once the ring has pages grants them."""
    rs = np.random.RandomState(most)
    page, heads, group, dim, pages, reqs = 32, 1, 2, 64, 60, 4
    plain = random_pool(rs, pages, heads, dim, page, "int8")
    ctx, add = np.array([64, 40, 64, 96]), np.array([2, most, 3, 1])
    table = make_table(rs, ctx, page, 12, cols=20)
    spare = [p for p in range(pages) if p not in table]
    rows = int(add.sum())
    i = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
    e = lambda n: torch.zeros(n, dtype=torch.int32, device=DEV)
    pool, dt, dlens, state = plain.to_device(B), i(table), i(ctx), i([0, 0])
    free = i(spare + [-1] * (pages - len(spare)))
    k, v, q = (dense(rs, rows, h, dim, "fp16", 0.4) for h in (heads, heads, heads * group))
    dk, dv, dq, dadd = k.to(DEV), v.to(DEV), q.to(DEV), i(add)

    def step(out):
        p = B.plan(dlens, dadd, dt, free, state, page=page, rows=rows, out=out)
        B.append(pool, dk, dv, p.slots)
        return p, *B.attend(pool, dq, p.cu, p.lens, dt, start=p.start, causal=causal, max_q=most, with_lse=True)

    mine = B.Plan(e(reqs + 1), e(reqs), e(reqs), e(rows), e(2), e(2))
    start = [t.clone() for t in (pool.k, pool.v, pool.k_scale, pool.v_scale)]

    def check(p, o, lse, few):
        st, ln, cu = p.start.cpu().numpy(), p.lens.cpu().numpy(), p.cu.cpu().numpy()
        # four tokens fit into request 1's page; the others ask for one page, and of two free ones 0 takes the first
        want_on = (np.array([True, most == 4, most == 4, False]) if few else np.ones(4, bool))
        assert np.array_equal(st >= 0, want_on)
        now = PlainPool(pages, heads, dim, page, "int8")
        for w in "kv":
            now.codes[w], now.scale[w] = plain.codes[w].copy(), plain.scale[w].copy()
        now.append(to_np(k), to_np(v), p.slots.cpu().numpy())
        want, wl, mean, tops = attend64(now, q.double().numpy(), cu, np.where(want_on, ln, 0), dt.cpu().numpy(), causal, 1 / math.sqrt(dim))
        tol, tol_lse = attend_tolerance("fp16", dim, want, wl, mean, tops)
        o, lse = o.cpu().double().numpy(), lse.cpu().double().numpy()
        assert (np.abs(o - want) <= tol).all()
        for r in range(reqs):
            part = slice(cu[r], cu[r + 1])
            assert want_on[r] or ((o[part] == 0).all() and (lse[part] == -np.inf).all())
            assert not want_on[r] or (np.abs(lse[part] - wl[part]) <= tol_lse[part]).all()

    def reset(count):
        for t, x in zip((pool.k, pool.v, pool.k_scale, pool.v_scale), start):
            t.copy_(x)
        dt.copy_(i(table))
        state.copy_(i([0, count]))

    for bad in (mine.start[:2], mine.start.long(), mine.start.cpu(), [0] * reqs):
        with pytest.raises(B.RmemError):
            B.attend(pool, dq, mine.cu, mine.lens, dt, start=bad)
    reset(2)
    check(*step(mine), True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(mine)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(mine)
    for count in (2, len(spare), 2, len(spare)):
        reset(count)
        g.replay()
        torch.cuda.synchronize()
        check(*got, count == 2)


@pytest.mark.gpu
def test_two_streams_at_once(B):
    """Two pools on two streams, calls interleaved on the host: no buffer is shared behind the caller's back."""
    rs = np.random.RandomState(23)
    jobs = []
    i = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
    for s in range(2):
        plain = random_pool(rs, 30, 2, 64, 64, "int8")
        lens, cu = [900, 700], np.array([0, 1, 3])
        table = make_table(rs, lens, 64, 30)
        q = dense(rs, 3, 4, 64, "fp16", 0.4)
        pool = plain.to_device(B)
        jobs.append((pool, q.to(DEV), i(cu), i(lens), i(table)))
    want = [B.attend(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]
    for _ in range(10):
        for s, (st, j) in enumerate(zip(streams, jobs)):
            with torch.cuda.stream(st):
                got[s].append(B.attend(*j))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)


@pytest.mark.gpu
def test_two_streams_of_long_calls_at_once(B):
    """The calls that need scratch -- an append of more than 4096 rows in any order, a read of more than 64 requests, short and long
    and divided over their tokens -- and a gather, on two streams at once: every result as on one stream, bit for bit."""
    rs = np.random.RandomState(24)
    i = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)
    page, pages, heads, dim, reqs = 32, 160, 2, 64, 70

    def job():
        n, lens = rs.randint(0, 3, reqs), rs.randint(0, 200, reqs)
        n[10], n[20], lens[10], lens[30] = 300, 40, 700, 1500
        cu = np.concatenate([[0], np.cumsum(n)])
        k, v = (dense(rs, pages * page, heads, dim, "bf16", 0.5).to(DEV) for _ in range(2))
        q = dense(rs, int(cu[-1]), 2 * heads, dim, "bf16", 0.5).to(DEV)
        return B.Pool.empty(pages, heads, dim, page, "int8", DEV), k, v, i(rs.permutation(pages * page)), q, i(cu), i(lens), i(rs.randint(0, pages, (reqs, 48)))

    def work(pool, k, v, slots, q, cu, lens, table):
        B.append(pool, k, v, slots)                    # (every page whole: it begins anew, the same each time)
        return [*B.attend(pool, q, cu, lens, table, with_lse=True), *B.gather(pool, slots, torch.bfloat16)]

    jobs = [job(), job()]
    want = [[t.clone() for t in work(*j) + [j[0].k, j[0].v, j[0].k_scale, j[0].v_scale]] for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]
    for _ in range(6):
        for s, (st, j) in enumerate(zip(streams, jobs)):
            with torch.cuda.stream(st):
                got[s].append(work(*j))
    torch.cuda.synchronize()
    for w, g, j in zip(want, got, jobs):
        for x in g:
            assert all(torch.equal(a, b) for a, b in zip(w, x))
        assert all(torch.equal(a, b) for a, b in zip(w[4:], (j[0].k, j[0].v, j[0].k_scale, j[0].v_scale)))


@pytest.mark.gpu
def test_attend_out_layouts(B):
    """Rows and heads of `out` in either order, with gaps, of one row or head; refused where they overlap."""
    from rmem_amd.hip import RmemError
    f = lambda *s: torch.zeros(*s, dtype=torch.float16, device=DEV)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    rs = np.random.RandomState(5)
    plain = random_pool(rs, 4, 1, 64, 32, "int8")
    pool, table = plain.to_device(B), i([[0, 1], [2, 3]])
    q = dense(rs, 5, 3, 64, "fp16", 0.5).to(DEV)
    args = (i([0, 2, 5]), i([40, 64]), table)
    want = B.attend(pool, q, *args)
    for out in (f(3, 5, 64).transpose(0, 1), f(5, 2, 3, 64)[:, 1], f(5, 3, 80)[:, :, 8:72], f(5, 200).as_strided((5, 3, 64), (200, 65, 1))):
        assert B.attend(pool, q, *args, out=out) is out and torch.equal(out, want)
    for out in (f(2000).as_strided((5, 3, 64), (64, 64, 1)), f(2000).as_strided((5, 3, 64), (191, 64, 1)), f(2000).as_strided((5, 3, 64), (192, 63, 1)),
                f(2000).as_strided((5, 3, 64), (64, 319, 1))):
        with pytest.raises(RmemError):
            B.attend(pool, q, *args, out=out)
    one = f(500).as_strided((1, 3, 64), (1, 64, 1))
    assert torch.equal(B.attend(pool, q[:1], i([0, 1]), i([40]), table[:1], out=one), B.attend(pool, q[:1], i([0, 1]), i([40]), table[:1]))


@pytest.mark.gpu
def test_attend_out_rows_right_behind_the_last_head(B):
    """Heads with gaps between them, rows without (the next row begins where the last head ends): shares no memory, so it is taken."""
    f = lambda *s: torch.zeros(*s, dtype=torch.float16, device=DEV)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    rs = np.random.RandomState(6)
    pool = random_pool(rs, 4, 1, 64, 32, "int8").to_device(B)
    q = dense(rs, 5, 3, 64, "fp16", 0.5).to(DEV)
    args = (i([0, 2, 5]), i([40, 64]), i([[0, 1], [2, 3]]))
    want = B.attend(pool, q, *args)
    for row, head in ((224, 80), (80, 5 * 80 - 16), (193, 64)):
        buf = f(2000).fill_(9)
        out = buf.as_strided((5, 3, 64), (row, head, 1))
        assert B.attend(pool, q, *args, out=out) is out and torch.equal(out, want)
        out.fill_(9)
        assert torch.all(buf == 9)                      # nothing beside it


@pytest.mark.gpu
def test_append_of_millions_of_rows(B):
    """More windows than the grid's y holds: every row is written once and comes back within half a step of its page's scale."""
    rows, page = 2_200_003, 128
    pages = -(-rows // page) + 2
    gen = torch.Generator(device=DEV).manual_seed(11)
    x = torch.randn((rows, 2, 32), generator=gen, device=DEV, dtype=torch.float32).to(torch.bfloat16)
    k, v = x[:, :1], x[:, 1:]
    pool = B.Pool.empty(pages, 1, 32, page, "int8", DEV)
    ids = torch.randperm(pages, generator=gen, device=DEV)
    slots = (ids[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)[:rows].to(torch.int32)
    B.append(pool, k, v, slots)
    got_k, got_v = B.gather(pool, slots, torch.float32)
    for got, want, scale in ((got_k, k, pool.k_scale), (got_v, v, pool.v_scale)):
        s = scale[(slots // page).long()][:, :, None]
        pad = torch.zeros((pages * page - rows, 1, 32), device=DEV)
        top = torch.cat([want.float().abs(), pad]).reshape(pages, -1).amax(1)[:-(-rows // page)]
        at = ids[:-(-rows // page)]
        # divided on the host: a device tensor over a number is a product with the number's inverse
        assert np.array_equal(scale[at, 0].cpu().numpy(), top.cpu().numpy() / np.float32(127))
        # half a step, and the roundings of 1 / s, the product and code * s: at most 127 codes times 3 * 2^-24, below 2^-15 of a step
        assert ((got - want.float()).abs() <= s * (0.5 + 2.0 ** -14)).all()
