"""DynamicQuantizeKernels.encode_rows: every row has the bits of DynamicQuantizeLinear on it alone (the oracle's), with
sentinels around every output."""
import numpy as np
import pytest

import og_oracle as oracle
import onegpu_cuda as og

pytestmark = pytest.mark.gpu


def check(device, dq, x, *, stride=0, off_x=0, off_y=0, off_s=0, off_z=0):
    """x: rows x columns, float32 or float16."""
    rows, columns = x.shape
    pitch = stride or columns
    store = np.full(off_x + max(rows - 1, 0) * pitch + columns, 1e4, x.dtype)  # never read between the rows
    for r in range(rows):
        store[off_x + r * pitch:off_x + r * pitch + columns] = x[r]
    y0 = np.full(off_y + rows * columns + 9, 0x3C, np.uint8)
    z0 = np.full(off_z + rows + 3, 0xEE, np.uint8)
    s0 = np.full(off_s + rows + 2, -5.0, np.float32)
    bx, by = device.create_buffer(x.dtype, store), device.create_buffer(np.uint8, y0)
    bs, bz = device.create_buffer(np.float32, s0), device.create_buffer(np.uint8, z0)
    enc = device.begin_commands()
    dq.encode_rows(enc, bx, off_x, rows, columns, stride, by, off_y, bs, off_s, bz, off_z)
    device.submit(enc)
    y, s, z = by.read(), bs.read(), bz.read()
    for b in (bx, by, bs, bz):
        b.dispose()
    for r in range(rows):
        wy, ws, wz = oracle.dynamic_quantize(x[r].astype(np.float32))
        y0[off_y + r * columns:off_y + (r + 1) * columns] = wy
        s0[off_s + r] = ws
        z0[off_z + r] = wz
    assert np.array_equal(s.view(np.uint32), s0.view(np.uint32)), (x.shape, x.dtype, s[off_s], s0[off_s])
    assert np.array_equal(z, z0), (x.shape, x.dtype)
    assert np.array_equal(y, y0), (x.shape, x.dtype, int(np.count_nonzero(y != y0)))


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("rows,columns", [(1, 1), (3, 2), (5, 7), (9, 31), (8, 32), (2, 33), (4, 255), (3, 256),
                                          (2, 1000), (7, 1024), (5, 1025), (3, 2056), (2, 4099), (1, 8192), (3, 16391),
                                          (2, 40001), (301, 129)])
def test_rows_are_bit_exact(device, kind, rows, columns):
    rng = np.random.default_rng(rows * 100003 + columns)
    with og.DynamicQuantizeKernels(device) as dq:
        x = (rng.standard_normal((rows, columns)) * rng.uniform(0.01, 30, (rows, 1))).astype(kind)
        check(device, dq, x)
        check(device, dq, x, off_x=1, off_y=3, off_s=1, off_z=2)
        check(device, dq, np.abs(x), stride=columns + 3, off_x=8, off_y=1)
        check(device, dq, -np.abs(x), stride=columns + 8, off_y=4)


@pytest.mark.parametrize("kind", [np.float32, np.float16])
def test_rows_of_every_distribution(device, kind):
    """The reference's input kinds (Int8Tests.cs:632-647), a row of each, and rows of special values."""
    with og.DynamicQuantizeKernels(device) as dq:
        for columns in (64, 777, 3000):
            rows = [oracle.dq_input(columns, 3, k) for k in range(7)]
            rng = np.random.default_rng(columns)
            base = rng.standard_normal(columns).astype(np.float32)
            special = []
            for value in (np.nan, np.inf, -np.inf, 65504.0, 1e-7, -0.0):
                r = base.copy()
                r[columns // 3] = value
                special.append(r)
            special += [np.full(columns, np.nan), np.full(columns, -np.inf), np.zeros(columns), np.full(columns, -0.0),
                        np.full(columns, 3.0), np.full(columns, -3.0), base * 1e-7]
            if kind == np.float32:
                special += [base * np.float32(1e-38), base * np.float32(3e37), np.full(columns, 1.4e-45)]
            with np.errstate(over="ignore"):
                check(device, dq, np.stack(rows + special).astype(np.float32).astype(kind))


@pytest.mark.parametrize("kind", [np.float32, np.float16])
def test_quotients_near_ties(device, kind):
    """Rows whose range is 255 steps of a power of two: every half-integer quotient is a tie."""
    with og.DynamicQuantizeKernels(device) as dq:
        for step in (1.0, 0.25, 2.0 ** -9):
            q = np.arange(-100, 155.5, 0.5)
            check(device, dq, np.tile((q * step).astype(kind), (3, 1)))


def test_no_rows(device):
    with og.DynamicQuantizeKernels(device) as dq:
        b = [device.create_buffer(k, 8) for k in (np.float32, np.uint8, np.float32, np.uint8)]
        enc = device.begin_commands()
        dq.encode_rows(enc, b[0], 0, 0, 8, 0, b[1], 0, b[2], 0, b[3], 0)
        assert enc.dispatch_count == 0
        device.submit(enc)
        for x in b:
            x.dispose()


def test_many_rows(device):
    """More rows than a launch's blocks hold at once, and codes that pass 2^31 bits apart."""
    rng = np.random.default_rng(2)
    with og.DynamicQuantizeKernels(device) as dq:
        check(device, dq, rng.standard_normal((70000, 40)).astype(np.float16))
        check(device, dq, rng.standard_normal((3000, 5003)).astype(np.float32))
