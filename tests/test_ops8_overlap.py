"""Which outputs the 8-bit operators' binding takes beside their inputs: the input itself, or memory that shares no
element with it, such as other columns of the same buffer.  Checked on host tensors against a count of shared bytes."""
import random

import pytest
import torch

import lbrr


def bytes_of(t):
    rows, cols = t.shape
    at = (torch.arange(rows)[:, None] * t.stride(0) + torch.arange(cols)) * t.element_size() + t.data_ptr()
    return set((at.flatten()[:, None] + torch.arange(t.element_size())).flatten().tolist())


def accepted(t, other):
    """As the operators ask: the distance of a single row is any."""
    ld = lambda v: v.stride(0) if v.shape[0] > 1 else v.shape[1] + -v.shape[1] % 16
    try:
        lbrr._same_rows("out", t, ld(t), "resid", other, ld(other))
    except lbrr.LbrrError as e:
        assert e.code == lbrr.ERR_INVALID and "overlaps" in str(e)
        return False
    return True


def test_columns_beside_each_other():
    buf = torch.zeros(8, 512)
    left, right = buf[:, :256], buf[:, 256:]
    assert accepted(left, right) and accepted(right, left) and accepted(left, left)
    assert not accepted(buf[:, 1:257], left) and not accepted(left, buf[:, 255:511])
    assert accepted(buf[:4, :100], buf[4:, :100]) and not accepted(buf[:4, :100], buf[3:7, :100])


def test_another_distance_between_rows_is_refused():
    flat = torch.zeros(4096)
    a, b = flat.as_strided((8, 64), (256, 1), 0), flat.as_strided((8, 64), (128, 1), 64)
    assert not accepted(a, b) and not accepted(b, a)  # rows that could meet: not looked at one by one


@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.float16, torch.float16),
                                   (torch.float32, torch.float16), (torch.float16, torch.float32)])
def test_never_takes_shared_bytes(types):
    rng = random.Random(5)
    raw = torch.zeros(16384, dtype=torch.uint8)
    taken = 0
    for _ in range(4000):
        rows, cols = rng.randint(1, 6), rng.randint(1, 40)
        pitch = 4 * rng.randint(cols, 90)
        views = []
        for dt in types:
            size = torch.empty(0, dtype=dt).element_size()
            p = pitch if rng.random() < 0.8 else 4 * rng.randint(cols, 90)
            views.append(raw.view(dt).as_strided((rows, cols), (p // size, 1), rng.randint(0, 500)))
        t, other = views
        same = t.data_ptr() == other.data_ptr() and t.dtype is other.dtype and (rows == 1 or t.stride() == other.stride())
        shared = bool(bytes_of(t) & bytes_of(other))
        ok = accepted(t, other)
        assert ok if same else not (ok and shared)
        if not same and not shared and t.stride(0) * t.element_size() == other.stride(0) * other.element_size():
            assert ok
            taken += 1
    assert taken > 200
