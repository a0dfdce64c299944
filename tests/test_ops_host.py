"""The device operators' host side: refusals before anything is queued (no GPU
needed: the pointers here are never followed), rotary frequencies, tree masks
and workspace sizes."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import opsabi
import qxops

BASE = 1 << 20            # a 16-byte aligned address that nobody reads


def cache(**over):
    c = dict(k=BASE, v=BASE, k_scales=BASE, v_scales=BASE, slot_rows=200, layer_rows=100, slots=3, layers=2, ctx_tokens=100,
             kv_heads=2, head_dim=64, reserved=0)
    c.update(over)
    return opsabi.Cache(*(c[f] for f, _ in opsabi.Cache._fields_))


def drafts(**over):
    d = dict(seqs=2, max_nodes=3, slots=BASE, lens=BASE, nodes=None)
    d.update(over)
    return opsabi.Drafts(*(d[f] for f, _ in opsabi.Drafts._fields_))


def heads(data=BASE, seq=3 * 4 * 64, node=4 * 64, head=64):
    return opsabi.Heads(data, seq, node, head)


def said(fn, *args):
    err = C.create_string_buffer(256)
    ok = fn(*args, err, 256)
    return ok, err.value.decode()


def rope(c=None, layer=0, d=None, freq=BASE, amplitude=1.0, rd=64, dtype=0, qh=4, q=None, qo=None, k=None, v=None,
         positions=None, status=None, no_q=False, no_kv=False):
    r = opsabi.Rotary(freq, amplitude, rd, 0)
    ref = lambda x: None if x is None else C.byref(x)  # noqa: E731
    q, qo = (None, None) if no_q else (q or heads(), qo or heads())
    k, v = (None, None) if no_kv else (k or heads(), v or heads())
    return said(opsabi.lib().qx_cuda_rope_append, C.byref(c or cache()), layer, C.byref(d or drafts()), C.byref(r), dtype, qh,
                ref(q), ref(qo), ref(k), ref(v), positions, status, None)


@pytest.mark.parametrize("args,message", [
    (dict(c=cache(k=None)), "invalid cache argument"),
    (dict(c=cache(k=BASE + 8)), "cache codes must be 16-byte aligned"),
    (dict(c=cache(v_scales=BASE + 2)), "cache scales must be 4-byte aligned"),
    (dict(c=cache(ctx_tokens=0)), "the cache has no rows"),
    (dict(c=cache(layer_rows=99)), "the layers of the cache overlap"),
    (dict(c=cache(slot_rows=199)), "the slots of the cache overlap"),
    (dict(c=cache(kv_heads=1, head_dim=40)), "a cache row must be a multiple of 16 bytes and at most 16384"),
    (dict(c=cache(kv_heads=512)), "a cache row must be a multiple of 16 bytes and at most 16384"),
    (dict(layer=2), "layer outside the cache"),
    (dict(d=drafts(slots=None)), "invalid drafts argument"),
    (dict(d=drafts(seqs=0)), "a call needs at least one sequence and one node"),
    (dict(d=drafts(max_nodes=4097)), "at most 4096 sequences and 4096 nodes"),
    (dict(d=drafts(lens=BASE + 1)), "slots, lengths and nodes must be 4-byte aligned"),
    (dict(freq=None), "invalid rotary argument"),
    (dict(freq=BASE + 4), "frequencies must be 8-byte, positions and status 4-byte aligned"),
    (dict(rd=63), "rotary_dim must be even, 2 to 512, and at most head_dim"),
    (dict(rd=66), "rotary_dim must be even, 2 to 512, and at most head_dim"),
    (dict(amplitude=math.inf), "the rotary amplitude must be finite"),
    (dict(dtype=3), "unsupported element type"),
    (dict(qh=0), "1 to 1024 query heads"),
    (dict(q=heads(BASE + 2)), "tensors must be aligned to their element"),
    (dict(qo=heads(head=63)), "an output tensor overlaps itself"),
    (dict(qo=heads(seq=0)), "an output tensor overlaps itself"),
    (dict(q=heads(), qo=heads(seq=8 * 4 * 64)), "q_out in place of q must have its strides"),
    (dict(k=heads(data=None)), "q goes with q_out, k with v"),
    (dict(no_q=True, no_kv=True), "nothing to rotate"),
])
def test_rope_append_refusals(args, message):
    assert rope(**args) == (0, message)


def tree(c=None, layer=0, d=None, dtype=0, qh=4, q=None, out=None, mask=None, scale=0.1, lse=None, mass=None, work=BASE,
         size=1 << 40, status=None):
    return said(opsabi.lib().qx_cuda_tree_attention, C.byref(c or cache()), layer, C.byref(d or drafts()), dtype, qh,
                C.byref(q or heads()), C.byref(out or heads()), mask, scale, lse, mass, work, size, status, None)


@pytest.mark.parametrize("args,message", [
    (dict(c=cache(head_dim=32)), "tree attention needs head_dim 64 or 128"),
    (dict(qh=3), "q_heads must be a multiple of kv_heads, at most 1024"),
    (dict(qh=0), "q_heads must be a multiple of kv_heads, at most 1024"),
    (dict(dtype=7), "unsupported element type"),
    (dict(q=heads(data=None)), "invalid tensor argument"),
    (dict(out=heads(node=128)), "an output tensor overlaps itself"),
    (dict(out=heads(data=BASE + 2)), "tensors must be aligned to their element"),
    (dict(layer=2), "layer outside the cache"),
    (dict(scale=math.nan), "the score scale must be finite"),
    (dict(mask=BASE + 4), "the mask must be 8-byte aligned"),
    (dict(lse=BASE + 2), "lse, mass and status must be 4-byte aligned"),
    (dict(work=None), "the workspace is missing, misaligned or too small"),
    (dict(work=BASE + 8), "the workspace is missing, misaligned or too small"),
    (dict(size=1024), "the workspace is missing, misaligned or too small"),
    (dict(c=cache(v=None)), "invalid cache argument"),
])
def test_tree_attention_refusals(args, message):
    assert tree(**args) == (0, message)


def test_tree_attention_refuses_more_steps_than_it_counts():
    """4096 sequences of 2^24 rows: 2^30 tiles of 64 rows, but 2^32 steps of 16 for the mass."""
    wide = cache(slots=1, layers=1, ctx_tokens=1 << 24, kv_heads=1, slot_rows=1 << 24, layer_rows=1 << 24)
    d, q = drafts(seqs=4096, max_nodes=1), heads(seq=64, node=64)
    args = dict(c=wide, d=d, qh=1, q=q, out=q)
    assert tree(mass=BASE, **args) == (0, "more rows and cache than one call can take")
    assert tree(**args)[1] != "more rows and cache than one call can take"      # refused later, for its made-up addresses


def evict(c=None, seqs=2, slots=BASE, dst=None, lens=BASE, mass=BASE, budget=8, sink=2, recent=2, kept=BASE, new=BASE + 64,
          status=None):
    return said(opsabi.lib().qx_cuda_kv_evict, C.byref(c or cache()), seqs, slots, dst, lens, mass, budget, sink, recent, kept,
                new, status, None)


@pytest.mark.parametrize("args,message", [
    (dict(c=cache(slots=0)), "the cache has no rows"),
    (dict(slots=None), "invalid eviction argument"),
    (dict(kept=None), "invalid eviction argument"),
    (dict(seqs=0), "1 to 4096 sequences"),
    (dict(budget=0, sink=0, recent=0), "sink + recent must fit the budget, which is at least 1"),
    (dict(sink=7), "sink + recent must fit the budget, which is at least 1"),
    (dict(sink=0xFFFFFFFF, recent=2), "sink + recent must fit the budget, which is at least 1"),
    (dict(budget=(1 << 24) + 1), "the budget is larger than any cache"),
    (dict(new=BASE), "new_lens may not be lens itself"),
    (dict(mass=BASE + 1), "eviction buffers must be 4-byte aligned"),
])
def test_evict_refusals(args, message):
    assert evict(**args) == (0, message)


def pick(**over):
    p = dict(logits=BASE, out=None, logits_stride=1000, out_stride=1000, rows=2, vocab=1000, dtype=0, max_history=4, max_bias=4,
             reserved=0, history=BASE, history_lens=None, repetition=None, frequency=None, presence=None, bias_ids=None,
             bias_lens=None, bias_values=None, allowed=None, history_stride=4, bias_stride=4, allowed_stride=32, picked=BASE)
    p.update(over)
    a = opsabi.Pick(*(p[f] for f, _ in opsabi.Pick._fields_))
    return said(opsabi.lib().qx_cuda_pick_tokens, C.byref(a), None)


@pytest.mark.parametrize("args,message", [
    (dict(logits=None), "invalid pick argument"),
    (dict(picked=None), "invalid pick argument"),
    (dict(rows=0), "a call needs at least one row and one token"),
    (dict(vocab=393217), "vocab is at most 393216"),
    (dict(dtype=9), "unsupported element type"),
    (dict(max_history=1 << 20), "max_history must be below 2^20"),
    (dict(bias_ids=BASE, bias_values=BASE, max_bias=4096), "max_bias is at most 4095"),
    (dict(bias_ids=BASE), "bias ids go with bias values"),
    (dict(out=BASE + 4096, out_stride=999), "an output tensor overlaps itself"),
    (dict(out=BASE, out_stride=1008), "out in place of logits must have their stride"),
    (dict(logits=BASE + 2), "tensors must be aligned to their element"),
    (dict(allowed=BASE + 2), "penalty, bias, mask and pick buffers must be 4-byte aligned"),
    (dict(logits_stride=1 << 41), "strides are too large"),
])
def test_pick_refusals(args, message):
    assert pick(**args) == (0, message)


def test_workspace_sizes_and_refusals():
    f = opsabi.lib().qx_cuda_tree_attention_workspace
    b = C.c_uint64()
    assert said(f, 1, 1, 32, 4, 128, 0, C.byref(b))[0] == 1 and b.value > 0 and b.value % 16 == 0
    small = b.value
    assert said(f, 64, 64, 32, 4, 128, 0, C.byref(b))[0] == 1 and b.value >= small
    assert said(f, 0, 1, 32, 4, 128, 0, C.byref(b)) == (0, "at least one and at most 4096 sequences and nodes")
    assert said(f, 1, 1, 32, 5, 128, 0, C.byref(b)) == (0, "q_heads must be a multiple of kv_heads, at most 1024")
    assert said(f, 1, 1, 32, 4, 128, 0, None) == (0, "invalid workspace argument")


def test_frequencies_against_their_formulas():
    rd, base, f, ctx = 128, 1e6, 8.0, 4096.0
    i = np.arange(rd // 2)
    plain = base ** (-2.0 * i / rd)
    near = dict(rtol=1e-13)
    unscaled, amp = qxops.rope_frequencies(rd, base)
    np.testing.assert_allclose(unscaled, plain, **near)
    assert amp == 1.0
    np.testing.assert_allclose(qxops.rope_frequencies(rd, base, "linear", f)[0], plain / f, **near)
    ntk = (base * f ** (rd / (rd - 2.0))) ** (-2.0 * i / rd)
    np.testing.assert_allclose(qxops.rope_frequencies(rd, base, "ntk", f)[0], ntk, **near)
    # by parts: untouched where a pair turns 32 times within ctx, slowed where it does not turn once
    got, amp = qxops.rope_frequencies(rd, base, "yarn", f, ctx)
    turns = ctx * plain / (2 * math.pi)
    assert amp == pytest.approx(0.1 * math.log(f) + 1, rel=1e-15)
    first = max(math.floor(rd * math.log(ctx / (32 * 2 * math.pi)) / (2 * math.log(base))), 0)
    last = min(math.ceil(rd * math.log(ctx / (2 * math.pi)) / (2 * math.log(base))), rd - 1)
    w = np.clip((i - first) / (last - first), 0, 1)
    np.testing.assert_allclose(got, plain * (1 - w) + plain / f * w, **near)
    assert np.array_equal(got[turns > 40], unscaled[turns > 40])       # left as they are, bit for bit
    np.testing.assert_allclose(got[turns < 0.7], plain[turns < 0.7] / f, **near)
    got, amp = qxops.rope_frequencies(rd, base, "bands", f, ctx, low=1.0, high=4.0)
    share = np.clip((turns - 1) / 3, 0, 1)
    np.testing.assert_allclose(got, plain * share + plain / f * (1 - share), **near)


@pytest.mark.parametrize("args", [
    dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=1.0), dict(rotary_dim=8, base=math.nan),
    dict(rotary_dim=8, scheme="linear", factor=0.5), dict(rotary_dim=2, scheme="ntk", factor=2.0),
    dict(rotary_dim=8, scheme="yarn", factor=2.0, original_ctx=0), dict(rotary_dim=8, scheme="bands", factor=2.0, low=4.0, high=1.0),
])
def test_frequencies_refusals(args):
    with pytest.raises(RuntimeError):
        qxops.rope_frequencies(**args)


def test_tree_mask_holds_ancestors():
    m = qxops.tree_mask([[-1, 0, 0, 2, -1, 3]])
    sees = [{0}, {0, 1}, {0, 2}, {0, 2, 3}, {4}, {0, 2, 3, 5}]
    assert m.shape == (1, 6, 1) and [int(x) for x in m[0, :, 0]] == [sum(1 << b for b in s) for s in sees]
    chain = qxops.tree_mask([list(range(-1, 129))])
    assert chain.shape == (1, 130, 3)
    bits = chain.numpy().view(np.uint64)
    assert [int(x) for x in bits[0, 129]] == [2 ** 64 - 1, 2 ** 64 - 1, 3]
    with pytest.raises(ValueError):
        qxops.tree_mask([[0]])


def test_python_handles_check_tensors():
    k = torch.zeros(2, 3, 8, 2, 64, dtype=torch.int8)
    s = torch.zeros(2, 3, 8)
    c = qxops.KvCache(k, k.clone(), s, s.clone())
    assert (c.c.slot_rows, c.c.layer_rows, c.c.ctx_tokens, c.c.slots) == (24, 8, 8, 2)
    # layer-major caches: [layer][slot] in memory
    kt, st = k.view(3, 2, 8, 2, 64).transpose(0, 1), s.view(3, 2, 8).transpose(0, 1)
    c = qxops.KvCache(kt, kt, st, st)
    assert (c.c.slot_rows, c.c.layer_rows) == (8, 16)
    for bad in (lambda: qxops.KvCache(k.float(), k, s, s), lambda: qxops.KvCache(k, k, s[..., :4], s),
                lambda: qxops.KvCache(k[..., :32], k[..., :32], s, s), lambda: qxops.KvCache(k, k, st.transpose(0, 1)[:, :, ::2], s)):
        with pytest.raises(ValueError):
            bad()


def test_host_memory_is_refused():
    """Without a GPU the call fails with CUDA's message; with one, host pointers are not device pointers."""
    k = torch.zeros(1, 1, 8, 1, 64, dtype=torch.int8)
    s = torch.zeros(1, 1, 8)
    one = torch.zeros(1, dtype=torch.int32)
    c = qxops.KvCache(k, k.clone(), s, s.clone())
    kept, new = torch.zeros(4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    ok, msg = said(opsabi.lib().qx_cuda_kv_evict, C.byref(c.c), 1, one.data_ptr(), None, one.data_ptr(), s.data_ptr(), 4, 0, 0,
                   kept.data_ptr(), new.data_ptr(), None, None)
    assert ok == 0 and msg


def test_view_refusals():
    ok, msg = said(opsabi.lib().qx_cuda_kv_view, None, 0, None)
    assert (ok, msg) == (0, "invalid cache view argument")


def test_rope_append_mass_refusals():
    fn = opsabi.lib().qx_cuda_rope_append_mass
    P, U32 = C.c_void_p, C.c_uint32
    fn.argtypes, fn.restype = [P, U32, P, P, U32, U32, P, P, P, P, P, P, P, P, C.c_char_p, C.c_uint64], C.c_int
    c, d, r, h = cache(), drafts(), opsabi.Rotary(BASE, 1.0, 64, 0), heads()
    call = lambda k, mass: said(fn, C.byref(c), 0, C.byref(d), C.byref(r), 0, 4, C.byref(h), C.byref(h), k, k, None, mass, None, None)  # noqa: E731
    assert call(None, BASE) == (0, "mass goes with k and v")
    assert call(C.byref(h), BASE + 2) == (0, "mass must be 4-byte aligned")


def test_tree_attention_in_place_refusals():
    assert tree(mass=BASE) == (0, "out may not be q itself where mass is collected")
    assert tree(q=heads(), out=heads(seq=8 * 4 * 64)) == (0, "out in place of q must have its strides")
    for apart in (dict(mass=BASE, out=heads(data=1 << 21)), dict()):
        assert tree(**apart)[1] not in ("", "out may not be q itself where mass is collected")       # refused later, for its made-up addresses


def test_a_closed_engine_gives_no_view():
    class Closed:
        h = None
    with pytest.raises(ValueError, match="the engine is closed"):
        qxops.EngineCache(Closed())
    view = object.__new__(qxops.EngineCache)
    view.engine = Closed()
    with pytest.raises(ValueError, match="the engine of this cache is closed"):
        view.handle
