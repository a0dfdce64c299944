"""What the torch module of the device operators (csrc/qx_torch.cpp) refuses before the library is called: shapes, types,
strides, devices, tensors that want a gradient.  On the host, where a sound call ends at "the operators take CUDA tensors", and
on a GPU, where it runs."""
import pytest
import torch

import qxops

SEQS, NODES, QH, KVH, HD, SLOTS, LAYERS, CTX = 2, 3, 4, 2, 64, 3, 2, 10
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def ints(dev, *shape):
    return torch.zeros(shape, dtype=torch.int32, device=dev)


def cache(dev):
    k = torch.zeros(SLOTS, LAYERS, CTX, KVH, HD, dtype=torch.int8, device=dev)
    s = torch.ones(SLOTS, LAYERS, CTX, device=dev)
    return qxops.KvCache(k, k.clone(), s, s.clone())


def arguments(op, dev):
    """A sound call's arguments by name."""
    x = lambda h: torch.randn(SEQS, NODES, h, HD, device=dev)  # noqa: E731
    slots, lens = torch.arange(SEQS, dtype=torch.int32, device=dev), ints(dev, SEQS)
    if op == "rope_append":
        return dict(cache=cache(dev), layer=1, slots=slots, lens=lens, q=x(QH), k=x(KVH), v=x(KVH),
                    inv_freq=torch.ones(HD // 2, dtype=torch.float64, device=dev), positions=ints(dev, SEQS, NODES),
                    nodes=torch.full((SEQS,), NODES, dtype=torch.int32, device=dev), q_out=x(QH), status=ints(dev, 1),
                    mass=torch.zeros(SLOTS, LAYERS, CTX, device=dev))
    if op == "tree_attention":
        return dict(cache=cache(dev), layer=1, slots=slots, lens=lens, q=x(QH), nodes=ints(dev, SEQS), out=x(QH),
                    mask=torch.ones(SEQS, NODES, 1, dtype=torch.int64, device=dev), lse=torch.zeros(SEQS, NODES, QH, device=dev),
                    mass=torch.zeros(SLOTS, LAYERS, CTX, device=dev), status=ints(dev, 1))
    if op == "evict":
        return dict(cache=cache(dev), slots=slots, lens=lens, mass=torch.zeros(SLOTS, LAYERS, CTX, device=dev), budget=4, sink=1,
                    recent=1, dst_slots=slots.clone(), kept=ints(dev, LAYERS, SEQS, 4), new_lens=ints(dev, SEQS), status=ints(dev, 1))
    f = lambda *s: torch.ones(s, device=dev)  # noqa: E731
    return dict(logits=torch.randn(5, 70, device=dev), history=ints(dev, 5, 6), history_lens=ints(dev, 5), repetition=f(5),
                frequency=f(5), presence=f(5), bias_ids=ints(dev, 5, 2), bias_values=f(5, 2), bias_lens=ints(dev, 5),
                allowed=ints(dev, 5, 3), out=f(5, 70), picked=ints(dev, 5))


def call(op, args):
    return getattr(qxops, op)(**args)


OPS = ["rope_append", "tree_attention", "evict", "pick_tokens"]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("op", OPS)
def test_sound_arguments(op, dev):
    if dev == "cuda":
        call(op, arguments(op, dev))
        torch.cuda.synchronize()
    else:
        with pytest.raises(ValueError, match="the operators take CUDA tensors"):
            call(op, arguments(op, dev))


WRONG = []
for _op in OPS:
    for _name, _x in arguments(_op, "cpu").items():
        if isinstance(_x, torch.Tensor):
            WRONG += [(_op, _name, how) for how in ("type", "shape", "dims", "stride", "grad", "list")]


def spoiled(x, how):
    """x with another type, one row more, a dimension more, every second value of twice as many; or as a list."""
    if how == "type":
        return x.to(torch.int16 if not x.is_floating_point() else torch.float8_e5m2)
    if how == "shape":
        return torch.cat((x, x[:1]))
    if how == "dims":
        return x[None]
    if how == "stride":
        return torch.stack((x, x), -1)[..., 0]
    if how == "grad":
        return x.clone().requires_grad_() if x.is_floating_point() else None
    return x.tolist()


@pytest.mark.parametrize("op,name,how", WRONG)
def test_each_tensor_is_checked(op, name, how):
    check_refused(op, name, how, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
def test_each_tensor_is_checked_on_a_gpu(op):
    for o, name, how in WRONG:
        if o == op:
            check_refused(op, name, how, "cuda")


def check_refused(op, name, how, dev):
    args = arguments(op, dev)
    bad = spoiled(args[name], how)
    if bad is None or (how == "stride" and bad.is_contiguous()) or (name, how) == ("inv_freq", "shape"):
        return                                                   # no such form of this tensor (inv_freq: another rotary_dim)
    args[name] = bad
    match = {"grad": "no backward pass", "list": "must be a tensor"}.get(how)
    with pytest.raises(ValueError, match=match) as e:
        call(op, args)
    assert "take CUDA tensors" not in str(e.value)
    if how == "grad":
        with torch.no_grad():                                    # the same tensors where no gradient is wanted
            if dev == "cuda":
                call(op, args)
                torch.cuda.synchronize()
            else:
                with pytest.raises(ValueError, match="take CUDA tensors"):
                    call(op, args)


@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
def test_tensors_of_another_device_are_refused(op):
    for name, x in arguments(op, "cuda").items():
        if isinstance(x, torch.Tensor):
            args = arguments(op, "cuda")
            args[name] = x.cpu()
            with pytest.raises(ValueError):
                call(op, args)


@pytest.mark.parametrize("dev", DEVICES)
def test_shapes_that_belong_together(dev):
    for op, change, match in [
            ("rope_append", lambda a: a.update(q=a["q"][..., :32].contiguous(), q_out=None), "head_dim differs"),
            ("rope_append", lambda a: a.update(q=None), "q_out without q"),
            ("rope_append", lambda a: a.update(q=None, q_out=None, k=None), "nothing to rotate"),
            ("rope_append", lambda a: a.update(k=a["k"].half()), "k must be a contiguous Float"),
            ("rope_append", lambda a: a.update(k=a["k"][:, :, :1]), "k must be a contiguous Float tensor of shape"),
            ("rope_append", lambda a: a.update(layer=-1), "layer must fit 32 bits"),
            ("tree_attention", lambda a: a.update(q=a["q"].double()), "unsupported element type Double"),
            ("tree_attention", lambda a: a.update(out=a["out"].bfloat16()), "out must be a contiguous Float"),
            ("tree_attention", lambda a: a.update(mass=a["mass"].transpose(0, 1).contiguous().transpose(0, 1)), "mass must be a float32 tensor like the scales"),
            ("evict", lambda a: a.update(budget=5), "kept must be a contiguous Int tensor of shape"),
            ("evict", lambda a: a.update(sink=1 << 32), "sink must fit 32 bits"),
            ("pick_tokens", lambda a: a.update(allowed=a["allowed"][:, :2]), "out, bias_values and allowed must match"),
            ("pick_tokens", lambda a: a.update(bias_values=a["bias_values"][:, :1]), "out, bias_values and allowed must match"),
            ("pick_tokens", lambda a: a.update(out=a["out"][:, :69]), "out, bias_values and allowed must match")]:
        args = arguments(op, dev)
        change(args)
        with pytest.raises(ValueError, match=match):
            call(op, args)


@pytest.mark.parametrize("dev", DEVICES)
def test_errors_of_arguments_that_are_no_tensors_come_through(dev):
    class Undecided:
        def __bool__(self):
            raise KeyError("undecided")
    with pytest.raises(KeyError):
        call("rope_append", dict(arguments("rope_append", dev), interleaved=Undecided()))
    with pytest.raises(TypeError):
        call("tree_attention", dict(arguments("tree_attention", dev), scale="half"))
    with pytest.raises(TypeError):
        call("evict", dict(arguments("evict", dev), budget=None))
