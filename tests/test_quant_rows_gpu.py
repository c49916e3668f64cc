"""Rows in 8 bits: quantised and read back by rule, bit for bit, in order, by number and through the hash map."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
FORMATS = ["e4m3", "int8"]
TYPES = [torch.float32, torch.bfloat16, torch.float16]
WIDTHS = [1, 2, 3, 4, 5, 16, 31, 64, 100, 128, 129, 256, 512, 513, 1000]


def plain(x, fmt):
    """Codes as float32 and scales, by the documented rule in float32."""
    x = x.float()
    share = torch.tensor(1.0, device=DEV) / torch.tensor(448.0 if fmt == "e4m3" else 127.0, device=DEV)
    scale = (x.abs().amax(-1) * share).clamp_min(2.0**-126)
    v = x * (1.0 / scale)[..., None]
    codes = v.to(torch.float8_e4m3fn).float() if fmt == "e4m3" else torch.round(v)
    return codes, scale


def values(n, width, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(n, width, generator=g, device=DEV) * torch.exp(3 * torch.randn(n, 1, generator=g, device=DEV))
    if n > 4:
        x[1] = 0
        x[2] *= 1e-41
        x[3, 0] = 3e4                 # one value far above the others
    return x.to(dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_rows_in_order_and_by_number(width, dtype, fmt):
    import ash

    for n in (1, 255, 256, 700):
        x = values(n, width, dtype, n + width)
        q = ash.quantize_rows(x, fmt)
        codes, scale = plain(x, fmt)
        fine = torch.isfinite(x).all(1)          # float16 rows whose values were beyond its range hold infinities
        assert torch.equal(q.scales[fine], scale[fine]) and torch.equal(q.codes.float()[fine], codes[fine])
        assert bool(q.scales[~fine].isnan().all())
        back = torch.where(fine[:, None], codes * scale[:, None], torch.nan)
        same = lambda a, b: torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0), b.nan_to_num(0))
        for out in TYPES:
            assert same(ash.dequantize_rows(q, dtype=out), back.to(out))
        which = torch.randint(0, n, (333,), device=DEV)
        which[5], which[6], which[7] = -1, n, 2**40
        want = back[which.clamp(0, n - 1)]
        want[5:8] = 0
        assert same(ash.dequantize_rows(q, which), want)
        assert same(ash.dequantize_rows(q, which.reshape(3, 111)), want.reshape(3, 111, width))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("width", [3, 8, 64, 600])
def test_infinities_and_nans_stay_in_their_rows(width, fmt):
    import ash

    x = values(40, width, torch.float32, 1)
    x[7, width // 2], x[9, 0], x[11, width - 1] = float("inf"), float("-inf"), float("nan")
    back = ash.dequantize_rows(ash.quantize_rows(x, fmt))
    odd = torch.zeros(40, dtype=torch.bool, device=DEV)
    odd[[7, 9, 11]] = True
    assert bool(back[odd].isnan().all()) and bool(torch.isfinite(back[~odd]).all())


def test_views_and_shapes():
    import ash

    x = torch.randn(6, 7, 33, device=DEV)
    for v in (x, x[:, 1:, 1:], x.transpose(0, 1), x[..., ::2], x[0, 0]):
        q = ash.quantize_rows(v)
        codes, scale = plain(v, "e4m3")
        assert q.codes.shape == v.shape and q.scales.shape == v.shape[:-1]
        assert torch.equal(q.codes.float(), codes) and torch.equal(q.scales, scale)
    assert ash.dequantize_rows(ash.quantize_rows(x[:0])).shape == (0, 7, 33)


def keys_of(n, dim, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    i = torch.randperm(4 * n, generator=g, device=DEV)[:n]
    cols = [(i // 37**d) % 37 if d < dim - 1 else i // 37**d for d in range(dim)]
    return torch.stack(cols, 1).int() - 18


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [1, 2, 3, 4])
@pytest.mark.parametrize("width", [1, 3, 16, 100, 300])
def test_map(dim, width, fmt):
    import ash

    n = 3001
    keys, x = keys_of(2 * n, dim, 5), values(2 * n, width, torch.float32, 2)
    m = ash.HashMap(dim, width, 2 * n, DEV, value_formats=fmt)
    m.insert(keys[:n], x[:n])
    m.insert(keys[n // 2:n + 100], x[n // 2:n + 100].to(torch.bfloat16))     # the first half of it is there already
    codes, scale = plain(x, fmt)
    want = codes * scale[:, None]
    c2, s2 = plain(x.to(torch.bfloat16), fmt)
    want[n:n + 100] = (c2 * s2[:, None])[n:n + 100]
    want[n + 100:] = 0
    order = torch.randperm(2 * n, device=DEV)
    masks, indices, rows = m.find(keys[order], return_values=True)
    assert torch.equal(masks, order < n + 100) and torch.equal(rows, want[order])
    assert torch.unique(indices[masks]).numel() == n + 100 == m.size()
    masks2, half = m.find(keys[order], return_indices=False, return_values=True, value_dtype=torch.float16)
    assert torch.equal(masks2, masks) and torch.equal(half, want[order].half())
    k, i, v = m.items(return_values=True)
    assert torch.equal(m.find(k, return_indices=False, return_values=True)[1], v)
    # a state of its own, another capacity, erased keys and an emptied map
    other = ash.HashMap(dim, width, 2 * n, DEV, value_formats=fmt)
    other.load_state_dict(m.state_dict())
    assert torch.equal(other.find(keys[order], return_values=True)[2], want[order])
    for capacity in (4 * n, n + 200):
        other.resize(capacity)
        assert torch.equal(other.find(keys[order], return_values=True)[2], want[order])
    m.erase(keys[:n // 2])
    masks, _, rows = m.find(keys[:n], return_values=True)
    assert not bool(masks[:n // 2].any()) and bool(masks[n // 2:].all())
    assert not bool(rows[:n // 2].any()) and torch.equal(rows[n // 2:], want[n // 2:n])
    m.insert(keys[:10], x[10:20])
    assert torch.equal(m.find(keys[:10], return_values=True)[2], want[10:20])
    m.clear()
    masks, _, rows = m.find(keys, return_values=True)
    assert m.size() == 0 and not bool(masks.any()) and not bool(rows.any())


def test_map_of_mixed_values():
    import ash

    n = 1000
    m = ash.HashMap(3, {"sdf": 1, "feature": 24, "color": 3}, n, DEV, value_formats={"feature": "e4m3", "color": "int8"})
    keys = keys_of(n, 3, 1)
    v = {"sdf": torch.randn(n, 1, device=DEV), "feature": torch.randn(n, 24, device=DEV), "color": torch.rand(n, 3, device=DEV)}
    m.insert(keys, v)
    masks, got = m.find(keys, return_indices=False, return_values=True)
    assert bool(masks.all()) and torch.equal(got["sdf"], v["sdf"])
    for name, fmt in (("feature", "e4m3"), ("color", "int8")):
        codes, scale = plain(v[name], fmt)
        assert torch.equal(got[name], codes * scale[:, None])
    _, got = m.items(return_indices=False, return_values=True)
    assert got["sdf"].shape == (n, 1) and got["feature"].shape == (n, 24)
    listed = ash.HashMap(3, [2, 8], n, DEV, value_formats=[None, "int8"])
    listed.insert(keys, [v["sdf"].expand(n, 2).contiguous(), v["feature"][:, :8]])
    assert torch.equal(listed.find(keys, return_values=True)[2][0], v["sdf"].expand(n, 2))


def test_duplicates_and_overflow():
    import ash

    n = 5000
    keys = keys_of(n, 3, 3)
    x = values(n, 20, torch.float32, 3)
    m = ash.HashMap(3, 20, n, DEV, value_formats="e4m3")
    twice = torch.cat([keys, keys, keys])
    m.insert(twice, torch.cat([x, x, x]))
    codes, scale = plain(x, "e4m3")
    assert m.size() == n and torch.equal(m.find(keys, return_values=True)[2], codes * scale[:, None])
    for many in (1500, n):
        small = ash.HashMap(3, 20, 1000, DEV, value_formats="e4m3")
        with pytest.warns(UserWarning, match="capacity"):
            if many < 2048:
                small.insert(keys[:many], x[:many])
            else:      # more keys than the table has slots: an error besides, as of any map
                with pytest.raises(RuntimeError, match="status"):
                    small.insert(keys, x)
        masks, _, rows = small.find(keys, return_values=True)
        assert int(masks.sum()) == small.size() <= 1000 and (many > 2048 or small.size() == 1000)
        assert torch.equal(rows[masks], (codes * scale[:, None])[masks]) and not bool(rows[~masks].any())


def test_empty_batches():
    import ash

    m = ash.HashMap(3, 8, 100, DEV, value_formats="int8")
    with pytest.warns(UserWarning, match="empty"):
        m.insert(torch.zeros(0, 3, dtype=torch.int32, device=DEV), torch.zeros(0, 8, device=DEV))
    with pytest.warns(UserWarning, match="empty"):
        masks, indices, rows = m.find(torch.zeros(0, 3, dtype=torch.int32, device=DEV), return_values=True)
    assert masks.shape == (0,) and indices.shape == (0,) and rows.shape == (0, 8)


def test_filtered_table():
    """A table beyond L2's share asks its occupancy bits first."""
    import ash

    n = 3_000_000
    m = ash.HashMap(3, 4, n, DEV, value_formats="int8")
    i = torch.arange(n, device=DEV)
    keys = torch.stack([i % 150, i // 150 % 150, i // 22500], 1).int()
    x = torch.randn(n, 4, device=DEV)
    m.insert(keys[::2].contiguous(), x[::2].contiguous())
    masks, _, rows = m.find(keys, return_values=True)
    codes, scale = plain(x, "int8")
    want = codes * scale[:, None]
    assert bool(masks[::2].all()) and not bool(masks[1::2].any())
    assert torch.equal(rows[::2], want[::2]) and not bool(rows[1::2].any())


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_cleared_map_reads_zeros(fmt):
    """Rows that keys without values are given after clear(), and the buffers themselves, a state's among them."""
    import ash

    n, width = 500, 20
    keys, x = keys_of(n, 3, 7), values(n, width, torch.float32, 7)
    x[::3, 1], x[1::3, 2] = float("inf"), float("nan")
    m = ash.HashMap(3, width, n, DEV, value_formats=fmt)
    m.insert(keys, x)
    m.clear()
    m.engine.insert_keys(keys)
    masks, _, rows = m.find(keys, return_values=True)
    assert bool(masks.all()) and not bool((rows != 0).any())
    assert not bool((m.items(return_values=True)[2] != 0).any())
    state = m.state_dict()
    assert not bool(state["default"].view(torch.uint8).any()) and not bool(state["default_scale"].any())


@pytest.mark.parametrize("fmt", FORMATS)
def test_types_of_rows_stay(fmt):
    """half(), double() and the like leave the codes and their scales what they are, and the buffers those that the map uses."""
    import ash

    n, width = 300, 12
    keys, x = keys_of(n, 3, 9), values(n, width, torch.float32, 9)
    m = ash.HashMap(3, width, n, DEV, value_formats=fmt)
    m.insert(keys[:200], x[:200])
    for change in (lambda: m.half(), lambda: m.double(), lambda: m.bfloat16(), lambda: m.float(),
                   lambda: torch.nn.ModuleList([m]).half(), lambda: torch.nn.ModuleList([m]).to(torch.float64)):
        change()
        assert m.default.dtype == ash.quant.FORMATS[fmt] and m.default_scale.dtype == torch.float32
        assert m.default is m.values["default"] and m.default_scale is m.values["default_scale"]
    m.insert(keys[200:], x[200:])
    codes, scale = plain(x, fmt)
    assert torch.equal(m.find(keys, return_values=True)[2], codes * scale[:, None])
    other = ash.HashMap(3, width, n, DEV, value_formats=fmt)
    other.load_state_dict(m.state_dict())
    assert torch.equal(other.find(keys, return_values=True)[2], codes * scale[:, None])
