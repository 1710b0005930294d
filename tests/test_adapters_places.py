"""Where ``adapters.add`` may store its rows: apart from ``base`` and ``x``, over ``base`` itself, or in columns of their own of the
buffer that holds them; the rule is checked here against a byte-by-byte count, without a GPU."""

import pytest
import torch

BF, F32 = torch.bfloat16, torch.float32


def touched(t, m):
    """Every byte of the first m rows."""

    size = t.element_size()
    return {t.data_ptr() + r * t.stride(0) * size + i for r in range(m) for i in range(t.shape[1] * size)}


@pytest.mark.parametrize("m", [1, 2, 5])
def test_the_rule_says_yes_wherever_a_byte_is_shared(m):
    """Every pair of column ranges of one buffer, of equal and of unequal types and steps; where no byte is shared and the steps
    are equal the rule says no."""

    from tensorfold_b200 import adapters

    buf = torch.zeros((m * 24 + 48,), dtype=F32)
    views = []
    for dtype, scale in ((F32, 1), (BF, 2)):
        flat = buf.view(dtype)
        for step in (12 * scale, 24 * scale):
            for first in range(0, 28 * scale, 3):
                for width in (1, 5, 11):
                    if first + (m - 1) * step + width <= flat.numel():
                        views.append(flat.as_strided((m, width), (step, 1), first))
    for a in views[::3]:
        for b in views:
            shared = bool(touched(a, m) & touched(b, m))
            says = adapters._overlap(a, b, m)
            assert says or not shared
            if m > 1 and a.stride(0) * a.element_size() == b.stride(0) * b.element_size() and not shared and says:
                # the only doubt left: ranges that pass one another before or behind the last row
                at = (b.data_ptr() - a.data_ptr()) % (a.stride(0) * a.element_size())
                assert at < a.shape[1] * a.element_size() or at + b.shape[1] * b.element_size() > a.stride(0) * a.element_size()


def test_columns_of_their_own_do_not_overlap():
    from tensorfold_b200 import adapters

    buf = torch.zeros((6, 100))
    for lo, hi, overlap in ((0, 40, True), (40, 80, False), (39, 79, True), (60, 100, False), (20, 30, True)):
        assert adapters._overlap(buf[:, :40], buf[:, lo:hi], 6) is overlap
        assert adapters._overlap(buf[:, lo:hi], buf[:, :40], 6) is overlap
    assert adapters._overlap(buf[:, :40], buf.view(BF)[:, 20:40], 6) and not adapters._overlap(buf[:, :40], buf.view(BF)[:, 80:120], 6)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 7, 150])
@pytest.mark.parametrize("first", [72, 75, 80])
def test_base_out_and_x_in_one_buffer(rows, first):
    """Columns of a fused projection: base, out and x side by side in the same rows, at aligned and unaligned columns; what lies
    between stays."""

    from tensorfold_b200 import adapters

    g = torch.Generator(device="cuda").manual_seed(2)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(BF)

    ad = adapters.make(normal(3, 16, 64) * 0.1, normal(3, 70, 16) * 0.3, 1.5)
    ids = (torch.arange(rows, device="cuda") % 4).to(torch.int32)
    plan = adapters.Plan(rows, 3, "cuda")
    adapters.route(ids, plan)
    buf = normal(rows, 256)
    x, base, out = buf[:, 160:224], buf[:, :70], buf[:, first:first + 70]
    want = adapters.add(x.clone(), ad, plan, base.clone())
    kept = buf.clone()
    assert adapters.add(x, ad, plan, base, out) is out and torch.equal(out, want)
    kept[:, first:first + 70] = want
    assert torch.equal(buf, kept)
    for lo in (1, 100, 155):
        with pytest.raises(ValueError, match="must not overlap"):
            adapters.add(x, ad, plan, base, buf[:, lo:lo + 70])
