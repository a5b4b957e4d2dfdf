"""How paged_attention_kernel cuts a ragged batch over its workgroups, through the library's exports of the
arithmetic the kernel itself runs: every tile's positions are covered once, cuts fall where the kernel's
loads allow them, the parts of a tile belong to consecutive workgroups that the merge finds, and the
workgroups' shares are even. And the lane offsets of its direct-to-LDS loads."""
import ctypes as C

import numpy as np
import pytest

u32 = C.c_uint32


@pytest.fixture(scope="module")
def lib(hip):
    f = hip.LIB.ds5_index_pb_parts
    f.argtypes, f.restype = [u32, C.c_void_p, C.c_void_p, u32, u32, u32, C.c_int, u32, C.c_void_p], u32
    hip.LIB.ds5_index_pb_loads.argtypes = [u32, C.c_int, C.c_void_p]
    return hip.LIB


def parts(lib, new, before, group, hkv, grid, whole):
    n, b = np.array(new, np.uint32), np.array(before, np.uint32)
    most = 200000
    out = np.zeros((most, 10), np.uint32)
    k = lib.ds5_index_pb_parts(len(n), n.ctypes.data, b.ctypes.data, group, hkv, grid, whole, most, out.ctypes.data)
    assert k <= most
    return out[:k].astype(np.int64)


def check(lib, new, before, group, hkv, grid, whole):
    p = parts(lib, new, before, group, hkv, grid, whole)
    want = {}
    for b, (n, c) in enumerate(zip(new, before)):
        for i in range(-(-n * group // 128)):
            rows = min(n * group, 128 * (i + 1)) - 128 * i
            for h in range(hkv):
                want[h, b, i] = (128 * i, rows, c + (128 * i + rows - 1) // group + 1)
    seen = {}
    for w, h, b, i, k0, k1, kv, row0, rows, last in p.tolist():
        assert want[h, b, i] == (row0, rows, kv)
        assert 0 <= k0 <= k1 <= kv and (k0 < k1 or 0 < k0) and k0 % 64 == 0 and (k1 % 64 == 0 or k1 == kv)
        seen.setdefault((h, b, i), []).append((w, k0, k1, last))
    assert set(seen) == set(want)
    cont, heads = set(), set()
    for key, ps in seen.items():
        assert ps[0][1] == 0 and ps[-1][2] == want[key][2]
        assert all(a[2] == b[1] and a[0] + 1 == b[0] for a, b in zip(ps, ps[1:]))
        if len(ps) > 1:
            assert not whole and ps[0][3] == ps[-1][0], (key, ps)  # the merge's last workgroup
            assert ps[0][0] not in heads and not any(w in cont for w, *_ in ps[1:])
            heads.add(ps[0][0])
            cont |= {w for w, *_ in ps[1:]}
        else:
            assert ps[0][3] == ps[0][0]
    return p


BATCHES = [
    ([1], [0], 8, 4), ([1], [8191], 8, 4), ([1], [131071], 16, 1), ([2048], [0], 8, 4), ([203], [6000], 16, 4), ([16], [0], 8, 1),
    ([17], [3], 8, 1), ([1] * 32, list(range(511, 16383, 496))[:32], 8, 4), ([500, 100] + [1] * 22, [64] * 24, 8, 4),
    ([0, 3, 0, 1, 0], [40, 10, 9, 0, 7], 8, 2), ([300], [31], 3, 2), ([33], [77], 5, 4), ([64], [3000], 128, 1), ([7], [0], 200, 3),
    ([1] * 1024, [i % 60 for i in range(1024)], 4, 1), ([0] * 1000 + [1], [5] * 1000 + [20000], 8, 1), ([5000], [0], 1, 8),
    ([129, 128, 127, 1, 2], [63, 64, 65, 0, 1], 1, 8), ([40000], [90000], 16, 8),
]


@pytest.mark.parametrize("new,before,group,hkv", BATCHES)
def test_every_position_once(lib, new, before, group, hkv):
    for grid in (256, 255, 64, 7, 1):
        for whole in (0, 1):
            check(lib, new, before, group, hkv, grid, whole)


def test_random_batches(lib):
    g = np.random.default_rng(1)
    for _ in range(400):
        n = int(g.integers(1, 40))
        new = (g.integers(0, 2, n) * np.exp(g.uniform(0, 6, n))).astype(int).tolist()
        before = np.exp(g.uniform(0, 9, n)).astype(int).tolist()
        check(lib, new, before, int(g.choice([1, 2, 3, 5, 8, 16, 130])), int(g.integers(1, 9)), int(g.choice([256, 200, 31])), int(g.integers(0, 2)))


def test_nothing(lib):
    assert len(parts(lib, [0, 0], [5, 0], 8, 4, 256, 0)) == 0


@pytest.mark.parametrize("new,before,group,hkv", [([1], [32767], 16, 4), ([2048], [0], 8, 4), ([1] * 32, list(range(511, 16383, 496))[:32], 8, 4),
                                                  ([203], [6000], 16, 4), ([515], [0], 8, 4)])
def test_even_shares(lib, new, before, group, hkv):
    """No working workgroup's positions (and 64 for each of its parts) are more than a fifth above the mean, but
    for the two cuts' steps of 64."""
    p = check(lib, new, before, group, hkv, 256, 0)
    share = np.bincount(p[:, 0], weights=p[:, 5] - p[:, 4] + 64)
    assert share.max() <= 1.2 * share[share > 0].mean() + 128


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("v", [0, 1])
def test_loads_cover_a_group_once(lib, d, v):
    loads = 16 * 2 * d // 1024
    off = np.zeros(loads * 64, np.uint32)
    lib.ds5_index_pb_loads(d, v, off.ctypes.data)
    assert sorted(off.tolist()) == list(range(0, 16 * 2 * d, 16))
    lds = np.arange(loads * 64) * 16
    assert np.array_equal(off // (2 * d), lds // (2 * d))  # a chunk stays in its row
    # what the kernel reads back: chunk c of row r in slot c ^ swizzle(r), with the swizzle linear in xor
    slot, chunk, r = lds % (2 * d) // 16, off % (2 * d) // 16, lds // (2 * d)
    swz = {0: {128: r & 15, 64: (r >> 1) & 7}, 1: {128: 4 * (r & 3), 64: 4 * ((r >> 1) & 1)}}[v][d]
    assert np.array_equal(slot ^ chunk, swz)


@pytest.fixture
def estimate(lib):
    """Sets the error of the reciprocals' estimates, and takes it back."""
    lib.ds5_index_pb_estimate.argtypes, lib.ds5_index_pb_estimate.restype = [C.c_double], None
    yield lib.ds5_index_pb_estimate
    lib.ds5_index_pb_estimate(0.0)


@pytest.mark.parametrize("bits", [22, 21])
def test_plan_with_the_devices_reciprocals(lib, estimate, bits):
    """The device's reciprocals are 2^-44 off at most, from estimates 2^-22 off: cuts may fall elsewhere, and every
    position is still covered once, by parts that the merge finds."""
    exact, moved = [], 0
    g = np.random.default_rng(2)
    batches = [(*b, grid, whole) for b in BATCHES for grid in (256, 255, 64, 7) for whole in (0, 1)]
    for _ in range(300):
        n = int(g.integers(1, 40))
        new = (g.integers(0, 2, n) * np.exp(g.uniform(0, 6, n))).astype(int).tolist()
        before = np.exp(g.uniform(0, 9, n)).astype(int).tolist()
        batches.append((new, before, int(g.choice([1, 2, 3, 5, 8, 16, 130])), int(g.integers(1, 9)), int(g.choice([256, 200, 31])), int(g.integers(0, 2))))
    estimate(0.0)
    exact = [parts(lib, *b) for b in batches]
    estimate(2.0 ** -bits)
    for b, p in zip(batches, exact):
        q = check(lib, *b)
        moved += p.shape != q.shape or not np.array_equal(p, q)
    print(f"{moved} of {len(batches)} plans moved")


def test_the_estimates_error_reaches_the_plan(lib, estimate):
    """(With an error that no device has: the cuts fall elsewhere.)"""
    b = ([1] * 32, list(range(511, 16383, 496))[:32], 8, 4, 256, 0)
    exact = parts(lib, *b)
    estimate(2.0 ** -4)
    assert not np.array_equal(parts(lib, *b), exact)
