"""The norm of many gradients together, and clipping by it (hetuctr_amd.nn, hctr_gradient_norm, hctr_clip_gradients), against 64 bits.

The squares and their sums are held in 64 bits, so that the norm is rounded once, to float: half a unit of 2^-23, and a unit more for
what 64 bits leave; below 2^-126 a float is a multiple of 2^-149, and half a step is 2^-150 however small the norm is (of 1001 values of
1.0e-42 it is 3.1655e-41, 2^-134: a 2^-23th of that is 2^-157, less than the step).  A gradient is multiplied by a factor that is one float, max_norm / norm (half a unit of 2^-23), the product is one
rounding more, and that to its type another: two units of 2^-24 and UNIT, of the product."""
import math

import pytest
import torch

from hetuctr_amd import capi, nn
from tests import products_reference as ref

gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def values(shape, kind, seed, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * std).to(TYPES[kind]).cuda()


def norm64(gradients):
    return math.sqrt(math.fsum(g.double().square().sum().item() for g in gradients))


def check(gradients, max_norm, norm, results):
    want = norm64(gradients)
    assert norm.shape == () and norm.dtype == torch.float32 and abs(norm.item() - want) <= max(2 ** -23 * want, 2 ** -150)
    factor = min(1.0, max_norm / want) if want else 1.0
    for g, r in zip(gradients, results):
        assert r.shape == g.shape and r.dtype == g.dtype
        if factor == 1.0:
            assert torch.equal(r, g)
        else:
            ref.check(r, g.double() * factor, 2 * ref.U * (g.double() * factor).abs(), "clipped")


def lists():
    # one value; one and a bit more than a vector, a block's pieces, a chunk (32 KiB); several; many; of all types; none
    for kind in TYPES:
        size = 4 if kind == "f32" else 2
        chunk = 32768 // size
        for n in (1, 3, 7, 8, 9, 255, chunk - 1, chunk, chunk + 1, 5 * chunk + 13):
            yield [values(n, kind, n)]
        yield [values((i % 50 + 1, i % 7 + 1), kind, i) for i in range(300)]
    yield [values((13, 17), kind, i, 10.0 ** -i) for i, kind in enumerate(("f32", "bf16", "f16", "f32"))]
    yield [values(0, "f32", 1), values(5, "f32", 1), values((0, 4), "bf16", 1)]
    yield [values(0, "f32", 1)]
    yield [values((1000, 1001), "bf16", 1), values((3001, 128), "f32", 2), values(11, "f16", 3)]


@gpu
def test_norm_and_clipping():
    for gradients in lists():
        kept = [g.clone() for g in gradients]
        norm = nn.gradient_norm(gradients)
        assert all(torch.equal(g, k) for g, k in zip(gradients, kept))
        for max_norm in (0.5, 1e9, 0.0):
            into = [torch.full_like(g, 7.0) for g in gradients]
            got = nn.clip_gradients(gradients, max_norm, into=into)
            assert torch.equal(got, norm) and all(torch.equal(g, k) for g, k in zip(gradients, kept))
            check(kept, max_norm, got, into)
            here = [g.clone() for g in gradients]
            assert torch.equal(nn.clip_gradients(here, max_norm), norm)
            assert all(torch.equal(a, b) for a, b in zip(here, into))
            # a norm that is known, as where other GPUs hold a part
            other = norm * 3 + 1
            here, want = [g.clone() for g in gradients], min(1.0, max_norm / other.item())
            assert nn.clip_gradients(here, max_norm, norm=other) is other
            for g, k in zip(here, kept):
                ref.check(g, k.double() * want, 2 * ref.U * (k.double() * want).abs(), "given")


@gpu
@pytest.mark.parametrize("kind", TYPES)
def test_gradients_anywhere_in_memory(kind):
    # at any address, in any order of memory; what lies beside them stays
    base = values((40, 70), kind, 1)
    turned = base.t()
    space = torch.full((3000,), 5.0, dtype=TYPES[kind], device="cuda")
    for at in (0, 1, 2, 3, 7):
        space.fill_(5.0)
        part = space[at:at + 2800].view(40, 70)
        part.copy_(base)
        norm = nn.clip_gradients([part], 1.0)
        check([base], 1.0, norm, [part])
        assert (space[:at] == 5).all() and (space[at + 2800:] == 5).all()
    part = base.clone().t()
    check([turned], 1.0, nn.clip_gradients([part], 1.0), [part])
    # rows apart: read as they are, but not written in place
    wide = values((40, 140), kind, 2)
    cut = wide[:, :70]
    into = torch.empty((40, 70), dtype=TYPES[kind], device="cuda")
    check([cut], 1.0, nn.clip_gradients([cut], 1.0, into=[into]), [into])
    other = torch.empty((70, 40), dtype=TYPES[kind], device="cuda").t()
    check([cut], 1.0, nn.clip_gradients([cut], 1.0, into=[other]), [other])
    assert abs(nn.gradient_norm([cut, base[:1].expand(9, 70)]).item() - norm64([cut, base[:1].expand(9, 70)])) < 1e-4
    negative = torch._neg_view(base.clone())
    assert torch.equal(nn.gradient_norm([negative]), nn.gradient_norm([base]))
    out = torch.empty_like(base)
    nn.clip_gradients([negative], 1.0, into=[out])
    assert torch.equal(out, nn_clipped(-base))
    two = [base.clone(), base.clone()]
    nn.clip_gradients([two[0], base], 1.0, into=[two[0], two[1]])     # one read twice, and written elsewhere
    check([base, base], 1.0, nn.gradient_norm([base, base]), two)


def nn_clipped(g):
    g = g.clone()
    nn.clip_gradients([g], 1.0)
    return g


@gpu
def test_norms_that_leave_the_range_of_squares():
    for kind, size in (("f32", 1e30), ("f32", 1e-30), ("bf16", 1e30), ("bf16", 1e-30), ("f32", 1e-42), ("f16", 6e-8), ("f16", 6e4)):
        g = torch.full((1001,), size, dtype=TYPES[kind], device="cuda")
        check([g], 1e-3, nn.gradient_norm([g]), [nn_scaled(g, 1e-3)])
    # larger than any float: infinity, and the gradients vanish
    g = torch.full((16,), 3e38, device="cuda")
    assert nn.clip_gradients([g], 1.0).item() == float("inf")


def nn_scaled(g, max_norm):
    out = torch.empty_like(g)
    nn.clip_gradients([g], max_norm, into=[out])
    return out


@gpu
def test_norms_that_are_not_finite():
    for odd, rest in ((float("nan"), float("nan")), (float("inf"), 0.0), (-float("inf"), 0.0)):
        for at in (0, 999, 70000):
            g, h = values(70001, "f32", 1), values(33, "bf16", 2)
            g[at] = odd
            norm = nn.clip_gradients([g, h], 1.0)
            assert norm.isnan() if odd != odd else norm.item() == float("inf")
            assert g[at].isnan() and (h.isnan().all() if rest != rest else (h == 0).all())
    for odd in (float("nan"), float("inf")):
        g = values(10, "f32", 1)
        nn.clip_gradients([g], 1.0, norm=torch.tensor(odd, device="cuda"))
        assert g.isnan().all() if odd != odd else (g == 0).all()
    g = values(10, "f32", 1)
    kept = g.clone()
    nn.clip_gradients([g], float("inf"))
    assert torch.equal(g, kept)
    zero = torch.zeros(10, device="cuda")
    assert nn.clip_gradients([zero], 0.0).item() == 0 and (zero == 0).all()


@gpu
def test_what_is_written_in_place_is_known_to_autograd():
    x = values(8, "f32", 1).requires_grad_()
    g = values(8, "f32", 2)
    y = (x * g).sum()
    nn.clip_gradients([g], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with pytest.raises(RuntimeError, match="wants a gradient"):
        nn.clip_gradients([g], 1.0, into=[x])
    with torch.no_grad():
        nn.clip_gradients([g], 1.0, into=[x])
    with pytest.raises(RuntimeError, match="not differentiable"):
        nn.gradient_norm([x])
    with torch.no_grad():
        assert nn.gradient_norm([x]) > 0


@gpu
def test_clipping_in_graphs_and_on_streams():
    gradients = [values((300, 70), "bf16", 1), values((1000, 128), "f32", 2), values(5, "f32", 3)] + [values(i + 1, "f16", i) for i in range(200)]
    kept = [g.clone() for g in gradients]
    into = [torch.empty_like(g) for g in gradients]
    nn.clip_gradients(gradients, 0.1, into=into)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = nn.clip_gradients(gradients, 0.1, into=into)
        again = nn.gradient_norm(into)
        nn.clip_gradients(gradients, 50.0)
    side = torch.cuda.Stream()
    for i in range(4):
        for g, k in zip(gradients, kept):
            g.copy_(k * (i + 1))
        want = [g.clone() for g in gradients]
        graph.replay()
        torch.cuda.synchronize()
        check(want, 0.1, norm, into)
        assert torch.equal(again, nn.gradient_norm(into))
        check(want, 50.0, norm, gradients)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = [torch.empty_like(g) for g in gradients]
            assert torch.equal(nn.clip_gradients(want, 0.1, into=other), norm)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(other, into))


@gpu
def test_more_gradients_than_arguments_hold():
    # thousands of small ones, and one of more values than 32 bits count
    gradients = [values(i % 13 + 1, "f32", i) for i in range(3000)]
    into = [torch.empty_like(g) for g in gradients]
    check(gradients, 1.0, nn.clip_gradients(gradients, 1.0, into=into), into)
    big = torch.zeros(2 ** 32 + 11, dtype=torch.bfloat16, device="cuda")
    big[-1], big[5], big[2 ** 31 + 3] = 3.0, 4.0, 12.0
    assert nn.gradient_norm([big, torch.zeros(3, device="cuda")]).item() == 13.0
    assert nn.clip_gradients([big], 6.5).item() == 13.0
    assert big[-1] == 1.5 and big[5] == 2.0 and big[2 ** 31 + 3] == 6.0 and big.count_nonzero() == 3
    del big
    torch.cuda.empty_cache()


# ---- refusals -----------------------------------------------------------------------------------------------------------------
def test_the_c_entry_points_refuse_what_they_cannot_do():
    # refused before anything is launched: no GPU is needed
    f32, space = capi.F32, (4096, 1 << 30)
    good = [(65536, 65536, 100, f32), (1 << 20, 1 << 21, 50, capi.BF16)]
    for gradients, max_norm, norm, workspace, match in [
            (good, -1.0, 64, space, "max_norm"), (good, float("nan"), 64, space, "max_norm"), (good, 1.0, 64, (0, 0), "workspace"),
            (good, 1.0, 64, (4100, 1 << 30), "workspace"), ([(0, 65536, 9, f32)], 1.0, 64, space, "null"), ([(65536, 0, 9, f32)], 1.0, 64, space, "null"),
            ([(65536, 65536, 9, 7)], 1.0, 64, space, "type"), ([(65536, 65536, 1 << 45, f32)], 1.0, 64, space, "2.44"),
            ([(65536, 65536, 9, f32), (65536, 65536, 9, f32)], 1.0, 64, space, "lies where"),               # the same one twice
            ([(65536, 65536, 9, f32), (65536 + 32, 65536 + 32, 9, f32)], 1.0, 64, space, "lies where"),
            ([(65536, 65536 + 16, 9, f32)], 1.0, 64, space, "lies where"),                                  # onto itself, moved
            ([(65536, 1 << 20, 9, f32), (1 << 21, (1 << 20) + 20, 9, f32)], 1.0, 64, space, "lies where"),
            ([(65536, 1 << 20, 9, f32), (1 << 20, 1 << 21, 9, f32)], 1.0, 64, space, "lies where")]:        # onto another that is read
        with pytest.raises(RuntimeError, match=match):
            capi.clip_gradients(gradients, max_norm, norm, 0, workspace)
    need = capi.clip_gradients(good, 1.0, 64, 0, (0, 0), space=True)
    with pytest.raises(RuntimeError, match="workspace"):
        capi.clip_gradients(good, 1.0, 64, 0, (4096, need - 1))
    with pytest.raises(RuntimeError, match="null"):
        capi.clip_gradients(good, 1.0, 0, 0, space, norm_only=True)
    with pytest.raises(RuntimeError, match="null"):
        capi.clip_gradients([(0, 0, 4, f32)], 1.0, 64, 0, space, norm_only=True)
    with pytest.raises(RuntimeError, match="type"):
        capi.clip_gradients([(65536, 0, 4, 9)], 1.0, 64, 0, space, space=True)
    for name in ("hctr_gradient_norm", "hctr_clip_gradients"):
        with pytest.raises(RuntimeError, match="null argument"):
            capi._check(getattr(capi.lib(), name)(None))
    assert capi.lib().hctr_gradient_workspace(None) == 2 ** 64 - 1


def test_lists_that_are_refused_without_a_gpu():
    for f in (nn.gradient_norm, lambda g: nn.clip_gradients(g, 1.0)):
        with pytest.raises(RuntimeError, match="no gradients"):
            f([])
        with pytest.raises(RuntimeError, match="on the GPU"):
            f([torch.zeros(3)])


@gpu
def test_the_functions_refuse_what_does_not_fit():
    g, h = torch.zeros((4, 6), device="cuda"), torch.zeros((4, 6), device="cuda")
    for f, match in [
            (lambda: nn.gradient_norm([g, g.cpu()]), "GPU"), (lambda: nn.gradient_norm([g.double()]), "float32, bfloat16 or float16"),
            (lambda: nn.gradient_norm([g, None]), "tensors"), (lambda: nn.clip_gradients([g], 1.0, into=[]), "as many"),
            (lambda: nn.clip_gradients([g], 1.0, into=[h.half()]), "type and shape"), (lambda: nn.clip_gradients([g], 1.0, into=[h[:2]]), "type and shape"),
            (lambda: nn.clip_gradients([g[:, :3]], 1.0), "one behind the other"), (lambda: nn.clip_gradients([g[:1].expand(4, 6)], 1.0), "one behind the other"),
            (lambda: nn.clip_gradients([torch._neg_view(g)], 1.0), "one behind the other"), (lambda: nn.clip_gradients([g, g], 1.0), "lies where"),
            (lambda: nn.clip_gradients([g, g.view(-1)[3:]], 1.0), "lies where"), (lambda: nn.clip_gradients([g], 1.0, into=[h.cpu()]), "GPU"),
            (lambda: nn.clip_gradients([g], -1.0), "max_norm"), (lambda: nn.clip_gradients([g], 1.0, norm=torch.zeros(2, device="cuda")), "norm"),
            (lambda: nn.clip_gradients([g], 1.0, norm=torch.zeros(())), "norm"), (lambda: nn.clip_gradients([g], 1.0, norm=torch.zeros((), device="cuda").double()), "norm")]:
        with pytest.raises(RuntimeError, match=match):
            f()
    with pytest.raises(TypeError):
        nn.clip_gradients([g], "one")
