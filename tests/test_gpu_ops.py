"""The device operators on the GPU against their definitions in 64 bits.

Tolerances (each derived where it is used): u(t) = finfo(t).eps / 2 is the
largest relative error of one rounding to t.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import opsabi
import qxlib
import qxops

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U32 = 2.0 ** -24


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def make_cache(g, slots, layers, ctx, kvh, hd, layer_major=False):
    lead = (layers, slots) if layer_major else (slots, layers)
    t = lambda x: x.transpose(0, 1) if layer_major else x  # noqa: E731
    code = lambda: t(torch.randint(-127, 128, lead + (ctx, kvh, hd), generator=g, device=DEV, dtype=torch.int8))  # noqa: E731
    scale = lambda: t(0.005 + 0.02 * torch.rand(*lead, ctx, generator=g, device=DEV))  # noqa: E731
    return qxops.KvCache(code(), code(), scale(), scale())


def copies(c):
    return [x.clone() for x in (c.k, c.v, c.k_scales, c.v_scales)]


# ---- rotary append -----------------------------------------------------------------------------------------------

def turned(x, pos, inv, factor, rd, interleaved):
    """The rotation in 64 bits: [..., head_dim] by pos [seqs][nodes]."""
    x = x.double()
    a = pos.double()[..., None, None] * inv
    c, s = torch.cos(a) * factor, torch.sin(a) * factor
    y = x.clone()
    i = torch.arange(rd // 2, device=x.device)
    p0, p1 = (2 * i, 2 * i + 1) if interleaved else (i, i + rd // 2)
    y[..., p0] = x[..., p0] * c - x[..., p1] * s
    y[..., p1] = x[..., p0] * s + x[..., p1] * c
    return y


def codes_of(x):
    """The cache's row rule on F32 values [..., row], in numpy."""
    x = x.cpu().numpy()
    fin = np.where(np.isfinite(x), x, np.float32(0))
    scale = (np.abs(fin).max(-1) / np.float32(127)).astype(np.float32)
    scale = np.where(scale > 0, scale, np.float32(1))
    q = np.clip(np.rint(fin / scale[..., None]), -127, 127).astype(np.int8)
    return torch.from_numpy(q).to(DEV), torch.from_numpy(scale).to(DEV)


def check_rope(c, before, layer, slots, lens, nodes, q, k, v, inv, pos, factor, rd, interleaved, q_out, q_before):
    seqs, n, qh, hd = q.shape
    kvh = c.kv_heads
    valid = torch.arange(n, device=DEV)[None] < nodes[:, None]
    want = turned(q, pos, inv, factor, rd, interleaved)
    # c, s: half a step each; two products, one sum: three roundings of terms of at most |x0| + |x1|; then the type's
    i = torch.arange(hd, device=DEV)
    mate = i.clone()
    p = torch.arange(rd // 2, device=DEV)
    a, b = (2 * p, 2 * p + 1) if interleaved else (p, p + rd // 2)
    mate[a], mate[b] = b, a
    size = abs(factor) * (q.double().abs() + q.double()[..., mate].abs())
    # (half types also round near their smallest normal number: half a step there)
    tol = 5 * U32 * size + torch.finfo(q.dtype).eps / 2 * (want.abs() + 5 * U32 * size) + torch.finfo(q.dtype).tiny * torch.finfo(q.dtype).eps / 2
    off = (q_out.double() - want).abs()
    assert bool((off <= tol)[valid].all()), float((off - tol)[valid].max())
    assert torch.equal(q_out[~valid], q_before[~valid])
    kr = turned(k, pos, inv, factor, rd, interleaved).float().reshape(seqs, n, kvh * hd)
    kc, ks = codes_of(kr)
    vc, vs = codes_of(v.float().reshape(seqs, n, kvh * hd))
    expect = [x.clone() for x in before]
    for s in range(seqs):
        for j in range(int(nodes[s])):
            sl, r = int(slots[s]), int(lens[s]) + j
            expect[0][sl, layer, r] = kc[s, j].view(kvh, hd)
            expect[1][sl, layer, r] = vc[s, j].view(kvh, hd)
            expect[2][sl, layer, r] = ks[s, j]
            expect[3][sl, layer, r] = vs[s, j]
    for got, e, what in zip((c.k, c.v, c.k_scales, c.v_scales), expect, ("k", "v", "k scales", "v scales")):
        assert torch.equal(got, e), what


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,hd,rd", [((8, 2), 128, 128), ((4, 4), 64, 32), ((5, 1), 128, 2), ((6, 3), 64, 50), ((3, 1), 48, 48)])
def test_rope_append(kind, interleaved, heads, hd, rd):
    g = gen(rd + hd)
    t, (qh, kvh) = TYPES[kind], heads
    seqs, n, ctx = 5, 4, 23
    c = make_cache(g, 7, 2, ctx, kvh, hd)
    before = copies(c)
    r = lambda h: torch.randn(seqs, n, h, hd, generator=g, device=DEV).to(t)  # noqa: E731
    q, k, v = r(qh), r(kvh), r(kvh)
    slots, lens, nodes = ints([6, 0, 3, 2, 5]), ints([0, 7, 19, 5, 22]), ints([4, 0, 4, 3, 1])
    pos = torch.randint(0, 1000000, (seqs, n), generator=g, device=DEV, dtype=torch.int32)
    inv, factor = qxops.rope_frequencies(rd, 1e4, "yarn" if rd > 2 else "none", 4.0, 2048)
    inv = torch.from_numpy(inv).to(DEV)
    q_out = torch.full_like(q, 7)
    status = ints([0])
    got = qxops.rope_append(c, 1, slots, lens, q, k, v, inv, positions=pos, nodes=nodes, interleaved=interleaved,
                            factor=factor, q_out=q_out, status=status)
    assert got is q_out and int(status) == 0
    check_rope(c, before, 1, slots, lens, nodes, q, k, v, inv, pos, factor, rd, interleaved, q_out, torch.full_like(q, 7))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("shift", [0, 1])
def test_rope_append_takes_views_of_one_projection_in_place(kind, shift):
    """q, k, v as views of one projection's rows (shift 1: off every 16-byte boundary), q rotated in place, positions from lens."""
    g = gen(5)
    t, seqs, n, qh, kvh, hd = TYPES[kind], 3, 2, 4, 2, 64
    c = make_cache(g, 3, 1, 9, kvh, hd, layer_major=True)
    before = copies(c)
    flat = torch.randn(seqs * n * (qh + 2 * kvh) * hd + 8, generator=g, device=DEV).to(t)
    qkv = flat[shift:shift + seqs * n * (qh + 2 * kvh) * hd].view(seqs, n, qh + 2 * kvh, hd)
    q, k, v = qkv[:, :, :qh], qkv[:, :, qh:qh + kvh], qkv[:, :, qh + kvh:]
    q0, rest = q.clone(), qkv[:, :, qh:].clone()
    slots, lens, nodes = ints([2, 0, 1]), ints([0, 7, 3]), ints([2, 2, 2])
    inv = torch.from_numpy(qxops.rope_frequencies(hd)[0]).to(DEV)
    qxops.rope_append(c, 0, slots, lens, q, k, v, inv, q_out=q)
    pos = lens[:, None] + torch.arange(n, device=DEV, dtype=torch.int32)
    check_rope(c, before, 0, slots, lens, nodes, q0, k, v, inv, pos, 1.0, hd, False, q, q0)
    assert torch.equal(qkv[:, :, qh:], rest)


def test_rope_queries_or_keys_alone():
    g = gen(6)
    c = make_cache(g, 2, 1, 8, 2, 64)
    inv = torch.from_numpy(qxops.rope_frequencies(64)[0]).to(DEV)
    q, k, v = (torch.randn(2, 3, h, 64, generator=g, device=DEV) for h in (4, 2, 2))
    slots, lens = ints([0, 1]), ints([1, 5])
    before = copies(c)
    both = qxops.rope_append(c, 0, slots, lens, q, k, v, inv)
    after = copies(c)
    for x, b in zip((c.k, c.v, c.k_scales, c.v_scales), before):
        x.copy_(b)
    only = qxops.rope_append(c, 0, slots, lens, q, None, None, inv)
    assert torch.equal(only, both) and all(torch.equal(x, b) for x, b in zip(copies(c), before))
    assert qxops.rope_append(c, 0, slots, lens, None, k, v, inv) is None
    assert all(torch.equal(x, b) for x, b in zip(copies(c), after))


def test_rope_append_of_non_finite_and_zero_rows():
    c = make_cache(gen(7), 1, 1, 4, 1, 64)
    inv = torch.from_numpy(qxops.rope_frequencies(64)[0]).to(DEV)
    k, v = torch.zeros(1, 3, 1, 64, device=DEV), torch.zeros(1, 3, 1, 64, device=DEV)
    v[0, 0, 0, 3], v[0, 0, 0, 4], v[0, 0, 0, 5], v[0, 0, 0, 6] = math.nan, math.inf, -2.0, 1.0
    v[0, 1, 0, 7] = 1e-44                                       # a denormal row
    qxops.rope_append(c, 0, ints([0]), ints([0]), None, k, v, inv, positions=ints([[0, 0, 0]]))
    codes, scales = codes_of(v.reshape(3, 64))
    assert torch.equal(c.v[0, 0, :3].reshape(3, 64), codes) and torch.equal(c.v_scales[0, 0, :3], scales)
    assert c.v[0, 0, 0, 0, 3:7].tolist() == [0, 0, -127, 64] and c.v_scales[0, 0, 2] == 1 and not c.k[0, 0, :3].any()


@pytest.mark.parametrize("scale", [2.0 ** -6, 0.013, 1e-30, 3e-38, 7e-41, 3e30])
def test_codes_of_values_next_to_a_half(scale):
    """Quotients that are a half, or a few units of the last place from it, round like the definition's; whole rows of tiny,
    denormal and huge scales too."""
    halves = np.arange(-126, 127, dtype=np.float64) + 0.5
    rows = [np.float32(127 * scale) * np.ones(256, np.float32) for _ in range(5)]
    step = rows[0][0] / np.float32(127)
    for i, row in enumerate(rows):
        x = (halves * float(step)).astype(np.float32)
        for _ in range(abs(i - 2)):
            x = np.nextafter(x, np.float32(math.copysign(math.inf, i - 2)))
        row[1:1 + len(x)] = x
        assert np.abs(row).max() == row[0]
    v = torch.from_numpy(np.stack(rows)).to(DEV).view(1, 5, 2, 128)
    c = make_cache(gen(3), 1, 1, 8, 2, 128)
    inv = torch.from_numpy(qxops.rope_frequencies(128)[0]).to(DEV)
    # at position 0 keys turn by nothing, so both halves of the cache hold the same
    qxops.rope_append(c, 0, ints([0]), ints([1]), None, v.clone(), v, inv, positions=ints([[0] * 5]))
    codes, scales = codes_of(v.reshape(5, 256))
    for got, s in ((c.k, c.k_scales), (c.v, c.v_scales)):
        assert torch.equal(got[0, 0, 1:6].reshape(5, 256), codes) and torch.equal(s[0, 0, 1:6], scales)


def test_rope_append_of_many_wide_heads():
    """More items of each kind than threads, in heads that turn in part: 40 query and 24 KV heads of 136 values, 48 of them turned."""
    g = gen(31)
    c = make_cache(g, 2, 1, 9, 24, 136)
    before = copies(c)
    q, k, v = (torch.randn(2, 3, h, 136, generator=g, device=DEV).bfloat16() for h in (40, 24, 24))
    inv = torch.from_numpy(qxops.rope_frequencies(48)[0]).to(DEV)
    slots, lens, nodes = ints([1, 0]), ints([2, 6]), ints([3, 3])
    for il in (False, True):
        out = torch.zeros_like(q)
        pos = ints([[5, 6, 900], [70000, 1, 0]])
        for x, b in zip((c.k, c.v, c.k_scales, c.v_scales), before):
            x.copy_(b)
        qxops.rope_append(c, 0, slots, lens, q, k, v, inv, positions=pos, interleaved=il, q_out=out)
        check_rope(c, before, 0, slots, lens, nodes, q, k, v, inv, pos, 1.0, 48, il, out, torch.zeros_like(q))


@pytest.mark.parametrize("kind,interleaved", [("f32", True), ("bf16", False), ("f16", True)])
def test_rope_append_of_long_prompts(kind, interleaved):
    """More tokens than run at once: chunks of up to 700 of three sequences, one ragged, one with nothing to append."""
    g = gen(41)
    c = make_cache(g, 3, 1, 720, 2, 64)
    before = copies(c)
    q, k, v = (torch.randn(3, 700, h, 64, generator=g, device=DEV).to(TYPES[kind]) for h in (6, 2, 2))
    inv = torch.from_numpy(qxops.rope_frequencies(40)[0]).to(DEV)
    slots, lens, nodes = ints([2, 0, 1]), ints([20, 3, 700]), ints([700, 411, 0])
    pos = (lens[:, None] + torch.arange(700, device=DEV, dtype=torch.int32)).contiguous()
    out = torch.full_like(q, 5)
    qxops.rope_append(c, 0, slots, lens, q, k, v, inv, nodes=nodes, interleaved=interleaved, q_out=out)
    check_rope(c, before, 0, slots, lens, nodes, q, k, v, inv, pos, 1.0, 40, interleaved, out, torch.full_like(q, 5))


def test_rope_append_from_threads_with_caches_of_different_width():
    """Rows of 16384 and of 12288 bytes, each from a thread of its own through the C ABI: neither call sets what the other goes by."""
    import threading
    lib = opsabi.lib()
    inv = torch.from_numpy(qxops.rope_frequencies(128)[0]).to(DEV)
    said, out, keep = {}, {}, []

    def calls(kvh, start):
        c = make_cache(gen(kvh), 1, 1, 4, kvh, 128)
        k = torch.randn(1, 2, kvh, 128, generator=gen(kvh), device=DEV)
        slots, lens = ints([0]), ints([1])
        keep.append((c, k, slots, lens))
        h = opsabi.Heads(k.data_ptr(), 2 * kvh * 128, kvh * 128, 128)
        d, r, none = opsabi.Drafts(1, 2, slots.data_ptr(), lens.data_ptr(), None), opsabi.Rotary(inv.data_ptr(), 1.0, 128, 0), opsabi.Heads()
        stream = torch.cuda.Stream()
        err = qxlib.err_buf()
        torch.cuda.synchronize()
        start.wait()
        for i in range(4000):
            if i % 64 == 0:
                stream.synchronize()                             # a full queue would have the threads take turns
            if not lib.qx_cuda_rope_append(C.byref(c.c), 0, C.byref(d), C.byref(r), 0, 0, C.byref(none), C.byref(none), C.byref(h),
                                           C.byref(h), None, None, stream.cuda_stream, err, len(err)):
                said[kvh] = err.value
                break
        stream.synchronize()
        out[kvh] = (c.v[0, 0, 1:3].reshape(2, -1), codes_of(k.reshape(2, -1))[0])

    start = threading.Barrier(6)
    threads = [threading.Thread(target=calls, args=(kvh, start)) for kvh in (128, 96) * 3]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not said
    assert all(torch.equal(*out[kvh]) for kvh in (128, 96))


def test_rope_append_leaves_out_what_does_not_fit():
    g = gen(8)
    c = make_cache(g, 3, 1, 6, 1, 64)
    before = copies(c)
    inv = torch.from_numpy(qxops.rope_frequencies(64)[0]).to(DEV)
    slots = ints([3, -1, 0, 1, 1, 2, 2, 0])
    lens = ints([0, 0, 5, 0, 2, 2, 0, -1])
    nodes = ints([1, 1, 2, 1, 1, 2, 0, 1])                      # only sequence 5 is sound (6 is empty)
    q, k, v = (torch.randn(8, 2, 1, 64, generator=g, device=DEV) for _ in range(3))
    status = ints([0])
    out = torch.full_like(q, 9)
    qxops.rope_append(c, 0, slots, lens, q, k, v, inv, nodes=nodes, q_out=out, status=status)
    assert int(status) == qxops.STATUS_RANGE | qxops.STATUS_SHARED
    assert bool((out[[0, 1, 2, 3, 4, 6, 7]] == 9).all()) and bool((out[5] != 9).any())
    now = copies(c)
    for x, b in zip(now, before):
        assert torch.equal(x[:2], b[:2]) and torch.equal(x[2, :, [0, 1, 4, 5]], b[2, :, [0, 1, 4, 5]])
        assert not torch.equal(x[2, 0, 2:4], b[2, 0, 2:4])


# ---- tree attention ----------------------------------------------------------------------------------------------

def attention(c, layer, slots, lens, nodes, q, mask, scale):
    """The definition in 64 bits: (out, lse, mass, tol, tol_lse, tol_mass), rows past a sequence's nodes NaN.

    Tolerances.  A score in base 2, x = log2e scale ks (q . k) + log2 vs, is a sum of head_dim products (one F16 term of q
    is exact for half types up to 2^-38 of the row's largest value, two leave at most 2^-22 of a value), held in F32: with
    S = log2e scale sum |q k| ks at most (terms + head_dim / 16 + 4) roundings of 2^-23 S, and 2^-22 (1 + |log2 vs| + |x|)
    for the last sum, the logarithm and the exponent's argument.  An error d of x is a factor 2^d of its weight and at most
    as much again through the sum of weights, so each weight is off by at most w = 2 ln 2 d relatively.  A weight meets the
    value codes as one F16 number (2^-11) or two (2^-22); sums of T weights in F32 add (T / 16 + 8) 2^-23 at most.
    The output rounds to its type."""
    seqs, n, qh, hd = q.shape
    grp, f32 = qh // c.kv_heads, q.dtype is torch.float32
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=DEV)
    lse = torch.full(q.shape[:3], math.nan, dtype=torch.float64, device=DEV)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    mass = torch.zeros(c.k_scales.shape, dtype=torch.float64, device=DEV)
    tol_mass = torch.zeros_like(mass)
    for s in range(seqs):
        sl, a, m = int(slots[s]), int(lens[s]), int(nodes[s])
        if not m:
            continue                                            # no row to compare
        t = a + m
        ks, vs = c.k_scales[sl, layer, :t].double(), c.v_scales[sl, layer, :t].double().clamp(min=2.0 ** -90)
        k, v = c.k[sl, layer, :t].double(), c.v[sl, layer, :t].double()
        sees = torch.ones(m, t, dtype=torch.bool, device=DEV)
        for i in range(m):
            for j in range(m):
                sees[i, a + j] = j <= i if mask is None else bool(int(mask[s, i, j // 64]) >> (j % 64) & 1)
        for h in range(qh):
            g = h // grp
            kk = k[:, g] * ks[:, None]
            x = scale * (q[s, :m, h].double() @ kk.T)
            big = abs(scale) * (q[s, :m, h].double().abs() @ kk.abs().T) * math.log2(math.e)
            x = x.masked_fill(~sees, -math.inf)
            lse[s, :m, h] = torch.logsumexp(x, -1)
            top = lse[s, :m, h, None]
            w = torch.where(sees, torch.exp(x - torch.where(torch.isfinite(top), top, torch.zeros_like(top))), torch.zeros((), dtype=torch.float64, device=DEV))
            w = torch.nan_to_num(w) if not torch.isfinite(x[sees]).all() else w
            out[s, :m, h] = w @ torch.where(sees.any(0)[:, None], v[:, g] * vs[:, None], torch.zeros((), dtype=torch.float64, device=DEV))
            size = w @ torch.where(sees.any(0)[:, None], (v[:, g] * vs[:, None]).abs(), torch.zeros((), dtype=torch.float64, device=DEV))
            seen = lambda y: torch.where(sees, y, torch.zeros((), dtype=torch.float64, device=DEV)).nan_to_num(0, 0, 0).amax(-1)  # noqa: E731
            terms = hd / 16 * (2 if f32 else 1) + 8
            d = terms * 2.0 ** -23 * seen(big) + 2.0 ** -22 * (1 + seen(torch.log2(vs).abs().expand_as(x)) + seen(x.abs() * 1.5) + 17)
            d = d + seen(big) * (2.0 ** -22 if f32 else 2.0 ** -37)
            rel = 2 * math.log(2) * d + (t / 16 + 8) * 2.0 ** -23
            o = (rel + (2.0 ** -22 if f32 else 2.0 ** -11))[:, None] * size
            tol[s, :m, h] = o + torch.finfo(q.dtype).eps / 2 * (out[s, :m, h].abs() + o) + 1e-30
            if q.dtype is torch.float16:
                tol[s, :m, h] += 2.0 ** -25                      # half a step of its subnormals
            tol_lse[s, :m, h] = rel + 2.0 ** -22 * lse[s, :m, h].abs().nan_to_num(0, 0, 0)
            mass[sl, layer, :t] += w.sum(0)
            tol_mass[sl, layer, :t] += ((rel + 2.0 ** -22 * (2 + seen(x.abs())))[:, None] * w).sum(0) + 1e-37
    return out, lse, mass, tol, tol_lse, tol_mass * (1 + n * qh * 2.0 ** -23)


def near(got, want, tol, what):
    most = torch.finfo(got.dtype).max
    got = got.double()
    # at least half a step past the type's largest number, whatever the error: infinity in that type
    want = torch.where(want.abs() - tol > most * (1 + torch.finfo(torch.float16).eps), want.sign() * math.inf, want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    off = (got - want).abs()
    ok = ~torch.isnan(want) & ~inf
    bad = (off > tol) & ok
    assert not bool(bad.any()), "%s: off by up to %g where %g is allowed" % (what, float(off[ok].max()), float(tol[bad].min()))


def check_tree(c, layer, slots, lens, nodes, q, mask, scale, want_mass=True):
    seqs, n, qh, _ = q.shape
    out = torch.full_like(q, 5)
    lse = torch.full((seqs, n, qh), 5.0, device=DEV)
    mass = torch.full_like(c.k_scales, 0.25) if want_mass else None
    status = ints([0])
    got = qxops.tree_attention(c, layer, slots, lens, q, nodes=nodes, mask=mask, scale=scale, out=out, lse=lse, mass=mass,
                               status=status)
    assert got is out and int(status) == 0
    nn = nodes if nodes is not None else ints([n] * seqs)
    w_out, w_lse, w_mass, tol, tol_lse, tol_mass = attention(c, layer, slots, lens, nn, q, mask, scale)
    pad = torch.arange(n, device=DEV)[None] >= nn[:, None]
    assert bool((out[pad] == 5).all()) and bool((lse[pad] == 5).all())
    near(out[~pad], w_out[~pad], tol[~pad], "out")
    near(lse[~pad], w_lse[~pad], tol_lse[~pad], "lse")
    if want_mass:
        near(mass, w_mass + 0.25, tol_mass + U32 * (w_mass + 1), "mass")
        assert bool((mass[w_mass == 0] == 0.25).all())
    return out, lse, mass


def random_tree(seqs, n, seed, roots=0.2):
    r = np.random.RandomState(seed)
    parents = [[-1 if i == 0 or r.rand() < roots else r.randint(0, i) for i in range(n)] for _ in range(seqs)]
    return qxops.tree_mask(parents).to(DEV)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,hd", [((8, 2), 128), ((8, 2), 64), ((5, 1), 128), ((3, 3), 64), ((16, 1), 128)])
@pytest.mark.parametrize("n,chain", [(1, True), (3, False), (7, True), (17, False)])
def test_tree_attention(kind, heads, hd, n, chain):
    g = gen(n + hd)
    qh, kvh = heads
    c = make_cache(g, 6, 2, 333, kvh, hd)
    lens = ints([0, 1, 63, 64, 200, 333 - n])
    nodes = ints([n, max(0, n - 1), n, max(1, n // 2), n, n])
    q = (1.5 * torch.randn(6, n, qh, hd, generator=g, device=DEV)).to(TYPES[kind])
    mask = None if chain else random_tree(6, n, n)
    check_tree(c, 1, ints([5, 0, 4, 1, 2, 3]), lens, nodes, q, mask, hd ** -0.5)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("seqs,n,ctx", [(1, 1, 5000), (1, 13, 3001), (2, 70, 500), (1, 130, 40), (37, 2, 257)])
def test_tree_attention_splits(kind, seqs, n, ctx):
    """Long rows shared over many CTAs, trees of more than one mask word and row block, many short sequences."""
    g = gen(ctx)
    c = make_cache(g, seqs, 1, ctx + n, 2, 128)
    q = torch.randn(seqs, n, 8, 128, generator=g, device=DEV).to(TYPES[kind])
    lens = ints([ctx - (i * 7) % min(ctx, 250) for i in range(seqs)])
    check_tree(c, 0, ints(list(range(seqs))), lens, None, q, random_tree(seqs, n, 3), 0.1)


@pytest.mark.parametrize("kind,n", [("bf16", 1), ("f32", 3), ("f16", 9)])
def test_tree_attention_of_hundreds_of_sequences(kind, n):
    """More sequences than threads that look them up, some without nodes, in each of the kernels."""
    g = gen(n)
    seqs = 300
    c = make_cache(g, seqs, 1, 90 + n, 1, 64)
    q = torch.randn(seqs, n, 8, 64, generator=g, device=DEV).to(TYPES[kind])
    lens = torch.randint(0, 91, (seqs,), generator=g, device=DEV, dtype=torch.int32)
    nodes = torch.randint(0, n + 1, (seqs,), generator=g, device=DEV, dtype=torch.int32)
    slots = torch.randperm(seqs, generator=g, device=DEV).to(torch.int32)
    check_tree(c, 0, slots, lens, nodes, q, random_tree(seqs, n, 8), 0.125)


def test_tree_attention_of_a_chain_of_many_rows():
    g = gen(77)
    c = make_cache(g, 1, 1, 700, 1, 64)
    q = torch.randn(1, 300, 2, 64, generator=g, device=DEV).half()
    check_tree(c, 0, ints([0]), ints([400]), None, q, None, 0.2)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [2, 24])
def test_rows_that_see_nothing_and_poison_in_masked_places(kind, n):
    """A node with an empty mask on an empty cache is zeros; scales that are NaN or infinite where no node looks, and codes and scales behind the
    sequence, change nothing; a poisoned tree row reaches only the nodes that see it."""
    g = gen(9)
    c = make_cache(g, 2, 1, 96, 2, 64)
    q = torch.randn(2, n, 16, 64, generator=g, device=DEV).to(TYPES[kind])
    mask = torch.zeros(2, n, 1, dtype=torch.int64, device=DEV)
    mask[0, 0, 0] = 1                                           # sequence 0, empty cache: node 0 sees itself, the others nothing
    mask[1, :, 0] = 1                                           # sequence 1: all see its node 0 only
    c.k_scales[0, 0, 1:] = math.nan
    c.v_scales[0, 0, 1:] = math.inf
    c.k_scales[1, 0, 41:] = math.inf
    c.v_scales[1, 0, 41:] = math.nan
    out, lse, _ = check_tree(c, 0, ints([0, 1]), ints([0, 40]), None, q, mask, 0.2)
    assert bool((out[0, 1:] == 0).all()) and bool((lse[0, 1:] == -math.inf).all())
    mask[1, 1, 0] = 3                                           # now node 1 sees the poisoned row 41
    again = qxops.tree_attention(c, 0, ints([0, 1]), ints([0, 40]), q, mask=mask, scale=0.2)
    assert bool(torch.isnan(again[1, 1]).all())
    keep = [i for i in range(n) if i != 1]
    assert torch.equal(again[1, keep], out[1, keep]) and torch.equal(again[0], out[0])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_scales_and_queries_of_far_apart_sizes(kind):
    """Value scales over 40 powers of ten, one key that takes all weight, queries near the ends of their type."""
    g = gen(10)
    c = make_cache(g, 4, 1, 300, 1, 128)
    c.v_scales[0, 0] = 10.0 ** (torch.rand(300, generator=g, device=DEV) * 40 - 20)
    c.v_scales[1, 0] = 0
    c.k_scales[2, 0, 100] = 5.0
    q = torch.randn(4, 5, 4, 128, generator=g, device=DEV)
    q[2] *= 3
    q[3, 0] *= 1e-6
    q[3, 1] *= 1e4
    q[3, 2] = 0
    q[3, 3, 0] *= 1e-3 ** torch.arange(128, device=DEV).remainder(3)
    check_tree(c, 0, ints([0, 1, 2, 3]), ints([290, 290, 290, 290]), None, q.to(TYPES[kind]), None, 0.05)


@pytest.mark.parametrize("kind,n", [("bf16", 1), ("f16", 4), ("f32", 20), ("bf16", 20)])
def test_value_scales_as_far_apart_as_they_may_lie(kind, n):
    """One row's value scale 2^100 times the others', with scores that are equal, and a little apart: none loses its share."""
    g = gen(18)
    c = make_cache(g, 2, 1, 300, 2, 64)
    c.v_scales[:] = 2.0 ** -84
    c.v_scales[:, 0, 77] = 2.0 ** 16
    c.k_scales[0] = 0
    q = torch.randn(2, n, 16, 64, generator=g, device=DEV).to(TYPES[kind])
    slots, lens, status = ints([0, 1]), ints([270, 270]), ints([0])
    lse, mass = torch.zeros(2, n, 16, device=DEV), torch.zeros_like(c.k_scales)
    out = qxops.tree_attention(c, 0, slots, lens, q, scale=0.05, lse=lse, mass=mass, status=status)
    assert int(status) == 0
    w_out, w_lse, w_mass, tol, tol_lse, tol_mass = attention(c, 0, slots, lens, ints([n, n]), q, None, 0.05)
    # On top of attention()'s tolerances: a row meets the codes (127 at most) with P_t = 2^(x_t - m + 8) as F16 numbers, which are
    # off by up to 2^-25 below 2^-14 (half a subnormal step; two terms too: the rest of such a number is 0).  The reference m is at
    # most 1 above the largest x, that of the row of scale 2^16, so the sum that divides is at least 2^7 / 2^16:
    # T rows are off by T 127 2^-25 2^9 together, in dims where that row's code is 0 all there is to see.
    near(out, w_out, tol + (270 + n) * 127 * 2.0 ** -16, "out")
    near(lse, w_lse, tol_lse, "lse")
    near(mass, w_mass, tol_mass + U32 * w_mass, "mass")


def test_the_smaller_term_of_f32_queries_reaches_the_scores():
    """128 values of 8192 + 7 2^-10 against codes of 64: the first F16 terms give 2^26, whose last bit is 8, the rest 7 in each of
    the eight steps of 16 products.  Added to 2^26 one by one, by a unit that cuts sums off, they would all be lost.

    lse of one row is its score, here 2^26 2^-20 and 92 in base 2.  Queries with and without the rest go through the same steps:
    the product with the row's factor, the reference less 8 and its sum with the logarithm, the product with ln 2, a rounding
    of 2^-24 each; the sum itself is exact where the rests come first (56 is a multiple of every partial sum's last bit)."""
    c = qxops.KvCache(*(torch.full((1, 1, 8, 1, 128), 64, dtype=torch.int8, device=DEV) for _ in range(2)),
                      *(torch.ones(1, 1, 8, device=DEV) for _ in range(2)))
    q = torch.full((1, 5, 8, 128), 8192.0, device=DEV)
    q[:, :, ::2] += 7 * 2.0 ** -10
    lse = torch.zeros(1, 5, 8, device=DEV)
    qxops.tree_attention(c, 0, ints([0]), ints([1]), q, mask=torch.zeros(1, 5, 1, dtype=torch.int64, device=DEV), scale=2.0 ** -20, lse=lse)
    more = (lse[:, :, ::2].double() - lse[:, :, 1::2].double()) / 64
    assert bool(((more - 56 * 2.0 ** -26).abs() <= 8 * 2.0 ** -24).all()), more


def test_shared_slots_broadcast_queries_and_strides():
    g = gen(11)
    c = make_cache(g, 2, 3, 120, 2, 128, layer_major=True)
    wide = torch.randn(4, 3, 12, 128, generator=g, device=DEV).bfloat16()
    q = wide[:, :, 2:10]                                         # heads inside a projection
    check_tree(c, 2, ints([1, 1, 0, 1]), ints([100, 50, 7, 100]), None, q, None, 0.09, want_mass=False)
    q1 = torch.randn(1, 3, 8, 128, generator=g, device=DEV).expand(4, 3, 8, 128)
    out = qxops.tree_attention(c, 2, ints([1, 1, 0, 1]), ints([100, 50, 7, 100]), q1)
    assert torch.equal(out[0], out[3]) and torch.equal(out, qxops.tree_attention(c, 2, ints([1, 1, 0, 1]), ints([100, 50, 7, 100]), q1.contiguous()))
    # off every 16-byte boundary
    flat = torch.zeros(4 * 3 * 8 * 128 + 8, dtype=torch.bfloat16, device=DEV)
    odd, to = flat[1:-7].view(4, 3, 8, 128), torch.zeros_like(flat)[3:-5].view(4, 3, 8, 128)
    odd.copy_(q)
    qxops.tree_attention(c, 2, ints([1, 1, 0, 1]), ints([100, 50, 7, 100]), odd, out=to)
    assert torch.equal(to, qxops.tree_attention(c, 2, ints([1, 1, 0, 1]), ints([100, 50, 7, 100]), q))


@pytest.mark.parametrize("n", [1, 20])
def test_tree_attention_leaves_out_what_does_not_fit(n):
    g = gen(12)
    c = make_cache(g, 2, 1, 50, 2, 64)
    q = torch.randn(6, n, 16, 64, generator=g, device=DEV)
    slots, lens = ints([2, 0, 1, -1, 0, 1]), ints([0, 50, -1, 3, 20, 20])
    out, status = torch.full_like(q, 3), ints([0])
    qxops.tree_attention(c, 0, slots, lens, q, out=out, status=status)
    assert int(status) == qxops.STATUS_RANGE
    assert bool((out[:4] == 3).all())
    want, _, _, tol, _, _ = attention(c, 0, slots[4:], lens[4:], ints([n, n]), q[4:], None, 64 ** -0.5)
    near(out[4:], want, tol, "out")
    # mass of two sequences of one slot: neither is added
    status.zero_()
    mass = torch.zeros_like(c.k_scales)
    qxops.tree_attention(c, 0, ints([0, 0, 1]), ints([20, 10, 20]), q[:3], mass=mass, status=status)
    assert int(status) == qxops.STATUS_SHARED and not mass[0].any() and bool((mass[1, 0, :20] > 0).all())


@pytest.mark.parametrize("n", [1, 4, 20])
def test_sequences_that_share_a_slot_attend_but_add_no_mass(n):
    """In each kernel: out and lse are those of the call without mass, mass grows where a slot has one sequence."""
    g = gen(14)
    c = make_cache(g, 3, 1, 60, 2, 64)
    q = torch.randn(4, n, 16, 64, generator=g, device=DEV)
    args = (c, 0, ints([0, 2, 0, 1]), ints([20, 7, 33, 40]), q)
    lse, lse_m, mass, status = (torch.zeros(4, n, 16, device=DEV), torch.zeros(4, n, 16, device=DEV), torch.zeros_like(c.k_scales), ints([0]))
    out = qxops.tree_attention(*args, lse=lse, status=status)
    assert int(status) == 0
    got = qxops.tree_attention(*args, lse=lse_m, mass=mass, status=status)
    assert int(status) == qxops.STATUS_SHARED
    assert torch.equal(got, out) and torch.equal(lse_m, lse)
    assert not mass[0].any() and bool((mass[1, 0, :40 + n] > 0).all()) and bool((mass[2, 0, :7 + n] > 0).all())


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,hd", [(3, 64), (4, 128)])
def test_poison_in_trees_of_seventeen_to_thirty_two_rows(kind, n, hd):
    g = gen(19)
    c = make_cache(g, 2, 1, 96, 2, hd)
    q = torch.randn(2, n, 16, hd, generator=g, device=DEV).to(TYPES[kind])
    mask = torch.zeros(2, n, 1, dtype=torch.int64, device=DEV)
    mask[0, 0, 0] = 1                                           # sequence 0, empty cache: node 0 sees itself, the others nothing
    mask[1, :, 0] = 1
    c.k_scales[0, 0, 1:], c.v_scales[0, 0, 1:] = math.nan, math.inf
    c.k_scales[1, 0, 41:], c.v_scales[1, 0, 41:] = math.inf, math.nan
    out, lse, _ = check_tree(c, 0, ints([0, 1]), ints([0, 40]), None, q, mask, 0.2)
    assert bool((out[0, 1:] == 0).all()) and bool((lse[0, 1:] == -math.inf).all())
    mask[1, 1, 0] = 3                                           # now node 1 sees the poisoned row 41
    again = qxops.tree_attention(c, 0, ints([0, 1]), ints([0, 40]), q, mask=mask, scale=0.2)
    assert bool(torch.isnan(again[1, 1]).all())
    keep = [i for i in range(n) if i != 1]
    assert torch.equal(again[1, keep], out[1, keep]) and torch.equal(again[0], out[0])


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("heads,hd,n", [((12, 3), 128, 97), ((12, 3), 64, 150), ((24, 8), 128, 5)])
def test_mass_of_more_queries_than_one_pass_holds(kind, heads, hd, n):
    """Query blocks that are held in several passes, cut inside a KV head and between heads; lengths that end inside a step."""
    g = gen(n)
    qh, kvh = heads
    c = make_cache(g, 4, 1, 400, kvh, hd)
    q = torch.randn(4, n, qh, hd, generator=g, device=DEV).to(TYPES[kind])
    check_tree(c, 0, ints([2, 0, 3, 1]), ints([200, 0, 17, 400 - n]), ints([n, n, 0, n - 1]), q, random_tree(4, n, 5), hd ** -0.5)


@pytest.mark.parametrize("kind,n", [("bf16", 1), ("f16", 4), ("f32", 20)])
def test_output_in_place_of_the_queries(kind, n):
    """Without mass out may be q itself; with mass, whose weights are taken from q after out is written, it is refused."""
    g = gen(17)
    c = make_cache(g, 3, 1, 700, 2, 64)
    q = torch.randn(3, n, 16, 64, generator=g, device=DEV).to(TYPES[kind])
    args = (c, 0, ints([0, 2, 1]), ints([640, 7, 300]))
    want = qxops.tree_attention(*args, q)
    here = q.clone()
    mass = torch.zeros_like(c.k_scales)
    with pytest.raises(RuntimeError, match="out may not be q itself where mass is collected"):
        qxops.tree_attention(*args, here, out=here, mass=mass)
    assert torch.equal(here, q) and not mass.any()
    assert qxops.tree_attention(*args, here, out=here) is here and torch.equal(here, want)


def test_calls_on_two_streams_at_once():
    """Each call has scratch of its own: the bits are those of the calls alone."""
    g = gen(23)
    c = make_cache(g, 6, 1, 3000, 2, 128)
    slots, lens = ints([0, 1, 2, 3, 4, 5]), ints([2900, 1500, 7, 0, 2000, 100])
    qs = [torch.randn(6, n, 16, 128, generator=g, device=DEV).bfloat16() for n in (1, 3, 12)]
    want = [(qxops.tree_attention(c, 0, slots, lens, q, mass=m), m) for q in qs for m in [torch.zeros_like(c.k_scales)]]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                m = torch.zeros_like(c.k_scales)
                got.append((qxops.tree_attention(c, 0, slots, lens, q, mass=m), m))
    torch.cuda.synchronize()
    for i, (out, m) in enumerate(got):
        assert torch.equal(out, want[i % 3][0]) and torch.equal(m, want[i % 3][1]), i


def test_the_same_call_gives_the_same_bits():
    g = gen(13)
    c = make_cache(g, 8, 1, 1000, 4, 128)
    q = torch.randn(8, 16, 32, 128, generator=g, device=DEV).bfloat16()
    args = (c, 0, ints([3, 1, 2, 0, 7, 6, 5, 4]), ints([984, 3, 500, 0, 77, 640, 641, 900]), q)
    mass = [torch.zeros_like(c.k_scales) for _ in range(2)]
    first, second = (qxops.tree_attention(*args, mass=m) for m in mass)
    assert torch.equal(first, second) and torch.equal(*mass)


# ---- eviction ----------------------------------------------------------------------------------------------------

def evicted(before, mass, slots, dst, lens, budget, sink, recent):
    """(cache tensors, mass, kept, new lengths) by the definition, on the host."""
    arr = [x.cpu().clone() for x in before]
    m = mass.cpu().clone()
    src_arr, src_m = [x.clone() for x in arr], m.clone()
    layers, seqs = m.shape[1], len(slots)
    kept = np.full((layers, seqs, budget), -1, np.int32)
    new = [min(n, budget) for n in lens]
    for i in range(seqs):
        n = lens[i]
        for l in range(layers):
            w = src_m[slots[i], l, :n].numpy().astype(np.float64)
            rows = list(range(n))
            if n > budget:
                mid = rows[sink:n - recent]
                need = budget - sink - recent
                rank = sorted(mid, key=lambda r: (math.isnan(w[r]), -w[r] if not math.isnan(w[r]) else 0, r))[:need]
                rows = rows[:sink] + sorted(rank) + rows[n - recent:]
            kept[l, i, :len(rows)] = rows
            for to, fr in zip(arr, src_arr):
                to[dst[i], l, :len(rows)] = fr[slots[i], l, rows]
            m[dst[i], l, :n] = 0
            m[dst[i], l, :len(rows)] = src_m[slots[i], l, rows]
    return arr, m, torch.from_numpy(kept), torch.tensor(new, dtype=torch.int32)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("kvh,hd", [(4, 128), (1, 64), (3, 16), (2, 136)])
@pytest.mark.parametrize("budget,sink,recent", [(1, 0, 0), (37, 4, 9), (40, 0, 40), (64, 64, 0), (300, 3, 5), (700, 1, 1)])
def test_evict(in_place, kvh, hd, budget, sink, recent):
    g = gen(budget)
    layers, ctx = 3, 613
    c = make_cache(g, 10, layers, ctx, kvh, hd, layer_major=budget == 37)
    mass = torch.rand(c.k_scales.shape, generator=g, device=DEV).pow(6)
    mass[torch.rand(mass.shape, generator=g, device=DEV) < 0.4] = 0
    mass[1] = torch.randint(0, 3, mass[1].shape, generator=g, device=DEV).float()          # ties everywhere
    mass[2] = 0
    keep = torch.empty_strided(mass.shape, c.k_scales.stride(), device=DEV)
    mass = keep.copy_(mass)
    slots, lens = [1, 0, 2, 4, 3], [613, 500, 612, 0, 41]
    dst = slots if in_place else [5, 6, 7, 8, 9]
    before = copies(c)
    want = evicted(before, mass, slots, dst, lens, budget, sink, recent)
    status = ints([0])
    kept, new = qxops.evict(c, ints(slots), ints(lens), mass, budget, sink, recent, dst_slots=None if in_place else ints(dst), status=status)
    assert int(status) == 0
    assert torch.equal(kept.cpu(), want[2]) and torch.equal(new.cpu(), want[3])
    assert torch.equal(mass.cpu(), want[1])
    for got, e, what in zip((c.k, c.v, c.k_scales, c.v_scales), want[0], ("k", "v", "k scales", "v scales")):
        assert torch.equal(got.cpu(), e), what


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("kvh,hd", [(4, 128), (2, 136), (1, 16)])
def test_evict_of_many_layers(in_place, kvh, hd):
    """Enough sequences and layers for the wide slices, and rows that end inside one."""
    g = gen(kvh)
    layers, ctx, seqs = 48, 150, 4
    c = make_cache(g, 2 * seqs, layers, ctx, kvh, hd)
    mass = torch.rand(c.k_scales.shape, generator=g, device=DEV)
    slots, lens = [0, 3, 1, 2], [150, 140, 90, 31]
    dst = slots if in_place else [4, 5, 6, 7]
    want = evicted(copies(c), mass, slots, dst, lens, 70, 2, 8)
    kept, new = qxops.evict(c, ints(slots), ints(lens), mass, 70, 2, 8, dst_slots=None if in_place else ints(dst))
    assert torch.equal(kept.cpu(), want[2]) and torch.equal(new.cpu(), want[3]) and torch.equal(mass.cpu(), want[1])
    for got, e, what in zip((c.k, c.v, c.k_scales, c.v_scales), want[0], ("k", "v", "k scales", "v scales")):
        assert torch.equal(got.cpu(), e), what


def test_evict_orders_any_weight():
    """Negative weights, infinities, both zeros, denormals, NaN (less than any number)."""
    c = make_cache(gen(1), 1, 1, 12, 1, 16)
    w = [math.nan, -math.inf, -1.0, -1e-44, -0.0, 0.0, 1e-44, 1e-38, 1.0, math.inf, math.nan, 0.0]
    mass = torch.tensor(w, device=DEV).view(1, 1, 12)
    for budget in range(1, 12):
        m = mass.clone()
        cc = qxops.KvCache(*copies(c))
        want = evicted(copies(c), m, [0], [0], [12], budget, 0, 0)
        kept, _ = qxops.evict(cc, ints([0]), ints([12]), m, budget)
        assert torch.equal(kept.cpu(), want[2]), budget
        assert torch.equal(m.cpu().view(torch.int32), want[1].view(torch.int32)), budget


def test_evict_of_a_long_cache():
    g = gen(3)
    n = 40000
    c = make_cache(g, 2, 1, n, 1, 64)
    mass = torch.rand(c.k_scales.shape, generator=g, device=DEV).mul_(2000).floor_()       # about 20 rows share each weight
    want = evicted(copies(c), mass, [0, 1], [0, 1], [n, n - 1], 20011, 7, 1000)
    kept, new = qxops.evict(c, ints([0, 1]), ints([n, n - 1]), mass, 20011, 7, 1000)
    assert torch.equal(kept.cpu(), want[2]) and torch.equal(new.cpu(), want[3]) and torch.equal(mass.cpu(), want[1])
    assert torch.equal(c.k.cpu(), want[0][0]) and torch.equal(c.v_scales.cpu(), want[0][3])


def test_evict_leaves_out_what_does_not_fit():
    g = gen(4)
    c = make_cache(g, 6, 2, 20, 1, 64)
    mass = torch.rand(c.k_scales.shape, generator=g, device=DEV)
    before, m0 = copies(c), mass.clone()
    #         0: slot out, 1: length out, 2 and 3: one destination, 4: destination is 5's source, 5: sound, 6: empty
    slots, dst, lens = ints([6, 0, 0, 1, 1, 3, 2]), ints([0, 1, 2, 2, 3, 4, 4]), ints([5, 21, 9, 9, 9, 20, 0])
    status = ints([0])
    kept, new = qxops.evict(c, slots, lens, mass, 8, 1, 1, dst_slots=dst, status=status)
    assert int(status) == qxops.STATUS_RANGE | qxops.STATUS_SHARED
    assert new.tolist() == [5, 21, 9, 9, 9, 8, 0]
    assert bool((kept[:, [0, 1, 2, 3, 4, 6]] == -1).all()) and bool((kept[:, 5] >= 0).all())
    for x, b in zip(copies(c) + [mass], before + [m0]):
        assert torch.equal(x[[0, 1, 2, 3, 5]], b[[0, 1, 2, 3, 5]]) and not torch.equal(x[4], b[4])


# ---- picking -----------------------------------------------------------------------------------------------------

def picked(logits, hist, hlens, rep, freq, pres, bids, bvals, blens, allowed):
    """The definition in F32, one rounding a step, on the host: (x in F32, token)."""
    x = logits.float().cpu().numpy().copy()
    rows, vocab = x.shape
    tok = np.zeros(rows, np.int64)
    f = np.float32
    for r in range(rows):
        if hist is not None:
            h = hist[r, :max(0, min(hist.shape[1], hlens[r] if hlens is not None else hist.shape[1]))]
            h = h[(h >= 0) & (h < vocab)]
            ids, cnt = np.unique(h, return_counts=True)
            for i, n in zip(ids, cnt):
                with np.errstate(all="ignore"):
                    a = f(rep[r]) if rep is not None else f(1)
                    y = x[r, i] / a if x[r, i] > 0 else x[r, i] * a
                    y = f(y - f(f(freq[r] if freq is not None else 0) * f(n)))
                    x[r, i] = f(y - f(pres[r] if pres is not None else 0))
        if bids is not None:
            last = {}
            for j in range(max(0, min(bids.shape[1], blens[r] if blens is not None else bids.shape[1]))):
                last[int(bids[r, j])] = bvals[r, j]
            for i, b in last.items():
                if 0 <= i < vocab:
                    x[r, i] = f(x[r, i] + f(b))
        if allowed is not None:
            t = np.arange(vocab)
            x[r, (allowed[r, t >> 5].astype(np.int64) >> (t & 31)) & 1 == 0] = -np.inf
        bad = np.isnan(x[r]).any() or (x[r] == np.inf).any() or x[r].max() == -np.inf
        tok[r] = -1 if bad else int(np.argmax(x[r]))
    return torch.from_numpy(x), torch.from_numpy(tok).to(torch.int32)


def run_pick(seed, rows, vocab, kind, hist, bias, grammar, stride=None, in_place=False, extremes=False, lens=True):
    g = gen(seed)
    t = TYPES[kind]
    store = torch.zeros(rows, stride or vocab, dtype=t, device=DEV)
    logits = store[:, :vocab]
    logits.copy_((4 * torch.randn(rows, vocab, generator=g, device=DEV)).to(t))
    if extremes:
        logits[0, ::3] = torch.finfo(t).min
        logits[1 % rows, :] = -math.inf
        logits[2 % rows, 5] = math.nan
        logits[3 % rows, 7] = math.inf
        logits[4 % rows, :] = 0.0
        logits[4 % rows, 1::2] = -0.0
    r = np.random.RandomState(seed)
    h = r.randint(-3, min(vocab + 3, 400), (rows, hist)).astype(np.int32) if hist else None
    hl = r.randint(-1, hist + 3, rows).astype(np.int32) if hist and lens else None
    rep, fr, pr = (r.uniform(a, b, rows).astype(np.float32) for a, b in ((0.8, 1.5), (-0.2, 0.7), (0, 0.6)))
    bi = r.randint(-2, vocab + 2, (rows, bias)).astype(np.int32) if bias else None
    bv = (r.randn(rows, bias) * 6).astype(np.float32) if bias else None
    bl = r.randint(-1, bias + 2, rows).astype(np.int32) if bias and lens else None
    if bias > 2:
        bi[:, 1] = bi[:, 0]                                       # the same id twice
    al = r.randint(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32)).astype(np.int32) if grammar else None
    if grammar:
        al[-1] = 0                                                # nothing is allowed
        if extremes:
            al[2 % rows, 0] &= ~(1 << 5)                          # NaN and infinity in masked places
            al[3 % rows, 0] &= ~(1 << 7)
    want_x, want_t = picked(logits, h, hl, rep, fr, pr, bi, bv, bl, al)
    d = lambda a: None if a is None else torch.from_numpy(a).to(DEV)  # noqa: E731
    rest = store[:, vocab:].clone()
    out, tok = qxops.pick_tokens(logits, d(h), d(hl), d(rep), d(fr), d(pr), d(bi), d(bv), d(bl), d(al), out=logits if in_place else None)
    want = want_x.to(t)
    assert torch.equal(tok.cpu(), want_t)
    assert torch.equal(torch.isnan(out).cpu(), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(out.cpu().float(), 0, 3e38, -3e38), torch.nan_to_num(want.float(), 0, 3e38, -3e38))
    assert torch.equal(store[:, vocab:], rest)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 31), (6, 1000), (5, 4099), (7, 20001), (2, 151936)])
@pytest.mark.parametrize("hist,bias,grammar", [(0, 0, False), (57, 0, True), (0, 9, False), (300, 33, True)])
def test_pick_tokens(kind, rows, vocab, hist, bias, grammar):
    run_pick(vocab + hist, rows, vocab, kind, hist, bias, grammar)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("grammar", [False, True])
def test_pick_tokens_with_extremes(kind, grammar):
    """Lowest values, rows of -infinity, NaN and +infinity seen or masked, ties of both zeros."""
    run_pick(5, 7, 517, kind, 0, 0, grammar, extremes=True)
    run_pick(6, 7, 517, kind, 40, 5, grammar, extremes=True)


@pytest.mark.parametrize("stride,in_place", [(5003, False), (5008, True), (5001, True)])
def test_pick_tokens_of_strided_rows(stride, in_place):
    run_pick(stride, 5, 5000, "f32", 64, 12, True, stride=stride, in_place=in_place)
    run_pick(stride, 5, 5000, "bf16", 64, 12, True, stride=stride, in_place=in_place, lens=False)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(25, 30011), (45, 151936), (60, 60001), (90, 4099), (170, 33), (170, 30011)])
def test_pick_tokens_of_more_rows_than_fit_at_once(kind, rows, vocab):
    """Each way of sharing rows and vocabulary out, with rows that follow one another in the same CTAs."""
    run_pick(rows + vocab, rows, vocab, kind, 200, 17, True)
    run_pick(rows, rows, vocab, kind, 0, 0, False)


def test_pick_tokens_of_a_large_vocabulary_and_history():
    run_pick(8, 2, 393216, "bf16", 70000, 4095, True)


@pytest.mark.parametrize("rows,vocab", [(1, 300), (18, 5000), (30, 40001), (100, 9000)])
def test_pick_tokens_call_after_call(rows, vocab):
    """Hundreds of short calls on two streams at once, each way of sharing rows out: CTAs of a cluster start one after the other
    while others still run, and the first of each joins what the others leave with it."""
    x = torch.randn(64, rows, vocab, generator=gen(rows), device=DEV)
    want = x.argmax(-1).to(torch.int32)
    tok = torch.zeros(2, 64, rows, dtype=torch.int32, device=DEV)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        tok.fill_(-2)
        torch.cuda.synchronize()
        for i in range(64):
            for s, t in zip(streams, tok):
                with torch.cuda.stream(s):
                    qxops.pick_tokens(x[i], picked=t[i])
        torch.cuda.synchronize()
        assert torch.equal(tok[0], want) and torch.equal(tok[1], want)


def test_pick_without_output():
    x = torch.randn(3, 777, device=DEV)
    args = opsabi.Pick(x.data_ptr(), None, 777, 0, 3, 777, 0, 0, 0, 0, *([None] * 9), 0, 0, 0, 0)
    tok = torch.zeros(3, dtype=torch.int32, device=DEV)
    args.picked = tok.data_ptr()
    err = qxlib.err_buf()
    assert opsabi.lib().qx_cuda_pick_tokens(C.byref(args), torch.cuda.current_stream().cuda_stream, err, len(err)), err.value
    assert torch.equal(tok.long(), x.argmax(-1))


# ---- together ----------------------------------------------------------------------------------------------------

class Loop:
    """A verify step over one layer: rotate and append a tree, attend, project to logits, pick, evict."""

    def __init__(self, seed, seqs=3, n=6, ctx=160, vocab=999):
        g = gen(seed)
        self.c = make_cache(g, seqs, 1, ctx, 2, 128)
        r = lambda h: torch.randn(seqs, n, h, 128, generator=g, device=DEV).bfloat16()  # noqa: E731
        self.q, self.k, self.v = r(8), r(2), r(2)
        self.slots, self.lens = ints([2, 0, 1]), ints([100, 3, 150])
        self.mask = random_tree(seqs, n, seed)
        self.pos = (self.lens[:, None] + ints([[0, 1, 1, 2, 2, 3]])).contiguous()
        self.inv = torch.from_numpy(qxops.rope_frequencies(128)[0]).to(DEV)
        self.head = torch.randn(8 * 128, vocab, generator=g, device=DEV)
        self.hist = torch.randint(0, vocab, (seqs * n, 50), generator=g, device=DEV, dtype=torch.int32)
        self.rep = torch.full((seqs * n,), 1.2, device=DEV)
        self.mass = torch.zeros_like(self.c.k_scales)
        self.q_out, self.out = torch.zeros_like(self.q), torch.zeros_like(self.q)

    def step(self):
        qxops.rope_append(self.c, 0, self.slots, self.lens, self.q, self.k, self.v, self.inv, positions=self.pos, q_out=self.q_out)
        qxops.tree_attention(self.c, 0, self.slots, self.lens, self.q_out, mask=self.mask, out=self.out, mass=self.mass)
        logits = (self.out.float().flatten(2).flatten(0, 1)[:, :, None] * self.head).sum(1)      # one order of sums everywhere
        self.logits, self.tokens = qxops.pick_tokens(logits, history=self.hist, repetition=self.rep)
        self.total = self.lens + self.q.shape[1]
        self.kept, self.new = qxops.evict(self.c, self.slots, self.total, self.mass, 64, 4, 16)

    def results(self):
        return copies(self.c) + [self.mass, self.q_out, self.out, self.logits, self.tokens, self.kept, self.new]


def test_a_verify_step_and_its_captured_replay():
    """The operators in order; the same step captured into a graph, replayed on fresh contents and changed lengths; and on
    another stream: the same bits."""
    a = Loop(21)
    a.step()
    first = a.results()
    b = Loop(21)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b.step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, y) for x, y in zip(first, b.results()))
    graph = torch.cuda.CUDAGraph()
    d = Loop(21)
    d.step()
    d0 = Loop(21)
    with torch.cuda.graph(graph):
        d.step()
    for lens in ([100, 3, 150], [0, 130, 60]):
        for x, y in zip((d.c.k, d.c.v, d.c.k_scales, d.c.v_scales), copies(d0.c)):
            x.copy_(y)
        d.mass.zero_()
        d.out.zero_()
        d.lens.copy_(ints(lens))
        graph.replay()
        torch.cuda.synchronize()
        e = Loop(21)
        e.lens.copy_(ints(lens))
        e.step()
        assert all(torch.equal(x, y) for x, y in zip(d.results(), e.results())), lens


def test_weights_of_rejected_nodes_do_not_reach_the_tokens_that_take_their_rows():
    """Two verify steps, the first of which accepts none of its nodes (or one), on a cache whose mass behind the committed rows
    is left over from something else: eviction goes by what each row's own token was given."""
    g = gen(51)
    n, ctx = 6, 120
    c = make_cache(g, 3, 2, ctx, 2, 128)
    slots, lens, mask = ints([2, 0, 1]), ints([100, 30, 57]), random_tree(3, n, 4)
    inv = torch.from_numpy(qxops.rope_frequencies(128)[0]).to(DEV)
    mass = 0.5 * torch.rand(c.k_scales.shape, generator=g, device=DEV)
    other = mass[:, 0].clone()
    want = mass.double()
    tol = torch.zeros_like(want)
    for accepted in ([0, 0, 1], None):
        q, k, v = (torch.randn(3, n, h, 128, generator=g, device=DEV).bfloat16() for h in (8, 2, 2))
        qo = qxops.rope_append(c, 1, slots, lens, q, k, v, inv, mass=mass)
        for i in range(3):
            rows = slice(int(lens[i]), int(lens[i]) + n)
            want[int(slots[i]), 1, rows] = tol[int(slots[i]), 1, rows] = 0
        qxops.tree_attention(c, 1, slots, lens, qo, mask=mask, mass=mass)
        _, _, w, _, _, t = attention(c, 1, slots, lens, ints([n] * 3), qo, mask, 128 ** -0.5)
        want, tol = want + w, tol + t + U32 * (want + w)
        near(mass, want, tol, "mass")
        lens = lens + ints(accepted) if accepted else lens + n
    assert torch.equal(mass[:, 0], other)                        # the other layer's rows were not written
    before, m0 = copies(c), mass.clone()
    kept, new = qxops.evict(c, slots, lens, mass, 24, 2, 4)
    e = evicted(before, m0, slots.tolist(), slots.tolist(), lens.tolist(), 24, 2, 4)
    assert torch.equal(kept.cpu(), e[2]) and torch.equal(mass.cpu(), e[1])


def test_rope_append_clears_the_mass_of_rows_it_writes_only():
    g = gen(52)
    c = make_cache(g, 4, 1, 12, 1, 64, layer_major=True)
    inv = torch.from_numpy(qxops.rope_frequencies(64)[0]).to(DEV)
    k, v = torch.randn(4, 3, 1, 64, generator=g, device=DEV), torch.randn(4, 3, 1, 64, generator=g, device=DEV)
    mass = torch.ones_like(c.k_scales)
    # sequence 0: two of three nodes; 1 and 2: one slot; 3: past the end
    qxops.rope_append(c, 0, ints([3, 1, 1, 0]), ints([5, 0, 4, 11]), None, k, v, inv, nodes=ints([2, 3, 3, 3]), mass=mass)
    want = torch.ones_like(mass)
    want[3, 0, 5:7] = 0
    assert torch.equal(mass, want)


def test_verify_step_against_the_definitions():
    a = Loop(22)
    n = a.q.shape[1]
    before = copies(a.c)
    qxops.rope_append(a.c, 0, a.slots, a.lens, a.q, a.k, a.v, a.inv, positions=a.pos, q_out=a.q_out)
    check_rope(a.c, before, 0, a.slots, a.lens, ints([n] * 3), a.q, a.k, a.v, a.inv, a.pos, 1.0, 128, False, a.q_out, a.q_out)
    _, _, mass = check_tree(a.c, 0, a.slots, a.lens, None, a.q_out, a.mask, 128 ** -0.5)
    total = (a.lens + n).tolist()
    want = evicted(copies(a.c), mass, a.slots.tolist(), a.slots.tolist(), total, 64, 4, 16)
    kept, new = qxops.evict(a.c, a.slots, a.lens + n, mass, 64, 4, 16)
    assert torch.equal(kept.cpu(), want[2]) and torch.equal(new.cpu(), want[3])
    assert all(torch.equal(x.cpu(), y) for x, y in zip(copies(a.c), want[0]))
    # and attention goes on over the shortened cache
    check_tree(a.c, 0, a.slots, new, None, a.q_out, a.mask, 128 ** -0.5)


def test_operators_over_an_engines_cache(mini_image):
    """A prompt that the engine prefilled, and a drafted tree run over the engine's cache by the operators."""
    eng = qxlib.Engine(mini_image, ctx=64, device=0)
    try:
        eng.prefill(np.arange(20, dtype=np.uint32) + 5)
        view = qxops.EngineCache(eng)
        assert (view.slots, view.layers, view.ctx, view.kv_heads, view.head_dim) == (1, eng.layers, 64, 2, 128)
        with pytest.raises(RuntimeError, match="sequence slots exist"):
            qxops.EngineCache(eng, batch=True)
        g = gen(31)
        n, layer = 5, eng.layers - 1
        q, k, v = (torch.randn(1, n, h, 128, generator=g, device=DEV) for h in (8, 2, 2))
        slots, lens, mask = ints([0]), ints([20]), random_tree(1, n, 4)
        inv = torch.from_numpy(qxops.rope_frequencies(128)[0]).to(DEV)
        pos = ints([[20, 21, 21, 22, 22]])
        q_out = qxops.rope_append(view, layer, slots, lens, q, k, v, inv, positions=pos)
        out = qxops.tree_attention(view, layer, slots, lens, q_out, mask=mask)
        torch.cuda.synchronize()
        host = [torch.from_numpy(x).to(DEV) for x in eng.kv_read(layer, 0, 25)]
        c = qxops.KvCache(host[0].view(1, 1, 25, 2, 128), host[1].view(1, 1, 25, 2, 128), host[2].view(1, 1, 25), host[3].view(1, 1, 25))
        kc, ks = codes_of(turned(k, pos, inv, 1.0, 128, False).float().reshape(1, n, 256))
        assert torch.equal(c.k[0, 0, 20:].reshape(n, 256), kc[0]) and torch.equal(c.k_scales[0, 0, 20:], ks[0])
        w_out, _, _, tol, _, _ = attention(c, 0, slots, lens, ints([n]), q_out, mask, 128 ** -0.5)
        near(out, w_out, tol, "out")
        eng.decode_batch([0], [7], [0])
        assert qxops.EngineCache(eng, batch=True).slots == 64
    finally:
        eng.close()


def test_a_view_ends_with_its_engine_and_knows_its_device(mini_image):
    """The engine's memory is gone once it is closed: calls with a view of it are refused, before anything is queued."""
    eng = qxlib.Engine(mini_image, ctx=64, device=0)
    try:
        with pytest.raises(ValueError, match="the engine's cache is on cuda:0"):
            qxops.EngineCache(eng, device=1)
        view = qxops.EngineCache(eng, device=0)
        assert view.device == torch.device("cuda", 0) == qxops.EngineCache(eng).device
    finally:
        eng.close()
    q = torch.randn(1, 1, 8, 128, device=DEV)
    for call in (lambda: qxops.tree_attention(view, 0, ints([0]), ints([0]), q), lambda: qxops.EngineCache(eng)):
        with pytest.raises(ValueError, match="closed"):
            call()


def test_offsets_past_32_bits():
    """A cache whose last slot starts more than 2^32 bytes in."""
    kvh, hd, ctx, slots = 4, 128, 4096, 2200
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    big = [torch.empty(slots, 1, ctx, kvh, hd, dtype=torch.int8, device=DEV) for _ in range(2)]
    sc = [torch.empty(slots, 1, ctx, device=DEV) for _ in range(2)]
    c = qxops.KvCache(big[0], big[1], sc[0], sc[1])
    g = gen(41)
    small = make_cache(g, 2, 1, ctx, kvh, hd)
    at = [slots - 1, slots - 2]
    for x, y in zip((c.k, c.v, c.k_scales, c.v_scales), (small.k, small.v, small.k_scales, small.v_scales)):
        x[at] = y
    q, k, v = (torch.randn(2, 3, h, hd, generator=g, device=DEV).bfloat16() for h in (8, kvh, kvh))
    inv = torch.from_numpy(qxops.rope_frequencies(hd)[0]).to(DEV)
    lens = ints([4000, 4093])
    mass_b, mass_s = torch.zeros_like(c.k_scales), torch.zeros_like(small.k_scales)
    got = []
    for cache, sl, mass in ((c, at, mass_b), (small, [0, 1], mass_s)):
        qo = qxops.rope_append(cache, 0, ints(sl), lens, q, k, v, inv)
        out = qxops.tree_attention(cache, 0, ints(sl), lens, qo, mass=mass)
        kept, new = qxops.evict(cache, ints(sl), lens, mass, 1000, 4, 100)
        got.append([qo, out, kept, new, mass[sl], cache.k[sl], cache.v[sl], cache.k_scales[sl], cache.v_scales[sl]])
    assert all(torch.equal(x, y) for x, y in zip(*got))
