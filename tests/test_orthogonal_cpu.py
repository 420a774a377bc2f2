"""The number format of csrc/orthogonal.hip, without a GPU: three bf16 limbs hold an f32 value, six of their products make one product."""
import torch


def limbs(v):
    out = []
    for _ in range(3):
        out.append(v.bfloat16().float())
        v = v - out[-1]
    return out


def values(seed):
    gen = torch.Generator().manual_seed(seed)
    v = torch.randn(200000, generator=gen) * torch.exp2(torch.randint(-90, 90, (200000,), generator=gen).float())
    edge = torch.tensor([0.0, 1.0, -1.0, 1.0 - 2.0 ** -24, 1.0 + 2.0 ** -23, 257.0 / 256, 65535.0 / 65536, 2.0 ** -100, 1.5 * 2.0 ** 100])
    return torch.cat([v, edge])


def test_three_limbs_hold_an_f32_value():
    v = values(0)
    a, b, c = limbs(v)
    assert torch.equal(a + (b + c), v) and torch.equal(a.double() + b.double() + c.double(), v.double())
    # one rounding to 8 bits each
    assert bool((b.abs() <= 2.0 ** -8 * v.abs()).all()) and bool((c.abs() <= 2.0 ** -16 * v.abs()).all())


def test_six_products_make_one():
    v, w = values(1), values(1).flip(0)
    keep = (v.double() * w.double()).abs() < 2.0 ** 120
    x, y = [t[keep].double() for t in limbs(v)], [t[keep].double() for t in limbs(w)]
    got = x[0] * y[0] + x[0] * y[1] + x[1] * y[0] + x[1] * y[1] + x[0] * y[2] + x[2] * y[0]
    want = v[keep].double() * w[keep].double()
    # v = m 2^e, 1 <= m < 2: the first limb leaves half a step of 8 bits, |limb 1| <= 2^(e - 8); limb 1 is below that power of two or is
    # exactly it, so it leaves |limb 2| <= 2^(e - 17).  Dropped are 1 2, 2 1 and 2 2: at most 2 * 2^-25 + 2^-34 of the product
    assert bool(((got - want).abs() <= (2.0 ** -24 + 2.0 ** -34) * want.abs()).all())
