"""The 4-bit KV cache's kernels (tmg_kv4_*) against the numpy reference in 64
bits (kv4ref.py): codes and values exactly, the attention within the bound
derived there."""
import numpy as np
import pytest

import kv4ref as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def T():
    import tinyminigo_amd as T
    return T


@pytest.fixture(scope="module")
def H():
    from tinyminigo_amd import hip as H
    return H


class Cache:
    """n_seq slabs in device memory, every byte 0xFF (marked groups) at first,
    and what they should hold, in 64 bits."""

    def __init__(self, T, H, cap, nkv, hd, n_seq=1, gap=0):
        self.T, self.H, self.cap, self.nkv, self.hd, self.n_seq = T, H, cap, nkv, hd, n_seq
        self.size = T.kv4_bytes(cap, nkv, hd)
        self.stride = self.size + gap
        self.buf = H.DeviceBuffer(self.stride * n_seq)
        self.buf.fill_byte(0xFF)
        self.kv = T.Kv4(self.buf.addr, cap=cap, nkv=nkv, hd=hd, n_seq=n_seq, seq_stride=self.stride)
        self.want = np.full((n_seq, 2, nkv, cap, hd), np.nan)

    def expect(self, k, v, pos):
        """The rows k, v [n_seq][rows][nkv][hd] at each sequence's position."""
        for b, p in enumerate(pos):
            if 0 <= p <= self.cap - k.shape[1]:
                for i, x in enumerate((k, v)):
                    self.want[b, i, :, p:p + x.shape[1]] = R.stands_for(x[b]).transpose(1, 0, 2)

    def write(self, k, v, pos, dev=None, stride=0, stream=0):
        """Through tmg_kv4_write; positions on the device when dev is given."""
        width = self.nkv * self.hd
        kd, vd = rows_buffer(self.H, k, stride or width), rows_buffer(self.H, v, stride or width)
        at = {"pos_dev": dev.addr} if dev else {"pos": pos[0]}
        self.T.kv4_write(self.kv, kd.addr, vd.addr, k.shape[1], row_stride=stride, stream=stream, **at)
        self.H.synchronize()
        self.expect(k, v, pos)

    def fill(self, rng, upto, keys=None, values=None):
        """Random rows [0, upto) of every sequence."""
        k, v = rows(rng, self, upto), rows(rng, self, upto)
        if keys is not None:
            k = keys(k)
        if values is not None:
            v = values(v)
        self.write(k, v, [0] * self.n_seq)
        return k, v

    def held(self):
        raw = self.buf.to_array(np.uint8, self.stride * self.n_seq)
        return np.stack([R.unpack(raw[b * self.stride:b * self.stride + self.size], self.cap, self.nkv, self.hd)
                         for b in range(self.n_seq)])

    def check(self):
        np.testing.assert_array_equal(self.held(), self.want)


def rows(rng, c, n):
    x = rng.standard_normal((c.n_seq, n, c.nkv, c.hd)) * np.exp(0.7 * rng.standard_normal((c.n_seq, n, c.nkv, 1)))
    return x.astype(np.float32)


def rows_buffer(H, x, stride, fill=0.0):
    """Device rows of x [n_seq][rows][..] at the stride."""
    flat = x.reshape(x.shape[0] * x.shape[1], -1)
    out = np.full((flat.shape[0], stride), fill, np.float32)
    out[:, :flat.shape[1]] = flat
    return H.DeviceBuffer.from_array(out)


def ints(H, x):
    return H.DeviceBuffer.from_array(np.asarray(x, np.int32))


def attend(c, q, pos, dev=None, new=None, q_stride=0, out_stride=0, new_stride=0, scale=None, stream=0):
    """Through tmg_kv4_attn: [n_seq][rows][nq][hd], and what stands around the
    rows of the output stays as it was."""
    T, H = c.T, c.H
    n_seq, n, nq, hd = q.shape
    width = nq * hd
    qd = rows_buffer(H, q, q_stride or width)
    tail = 40
    out = H.DeviceBuffer.from_array(np.full(n_seq * n * (out_stride or width) + tail, 7.25, np.float32))
    ws_bytes = T.kv4_attn_workspace(c.kv, n, nq)
    ws = H.DeviceBuffer.from_array(np.concatenate([np.zeros(ws_bytes, np.uint8), np.full(64, 255, np.uint8)]))
    kd = vd = None
    if new is not None:
        kd, vd = (rows_buffer(H, x, new_stride or c.nkv * hd) for x in new)
    at = {"pos_dev": dev.addr} if dev else {"pos": pos[0]}
    T.kv4_attn(c.kv, qd.addr, out.addr, n, nq, k_dev=kd.addr if kd else 0, v_dev=vd.addr if vd else 0,
               q_stride=q_stride, out_stride=out_stride, row_stride=new_stride, scale=scale or 0.0, ws_dev=ws.addr,
               ws_bytes=ws_bytes, stream=stream, **at)
    H.synchronize()
    if new is not None:
        c.expect(new[0], new[1], pos)
    raw = out.to_array(np.float32, n_seq * n * (out_stride or width) + tail)
    assert (raw[-tail:] == 7.25).all()
    assert (ws.to_array(np.uint8, ws_bytes + 64)[-64:] == 255).all()
    body = raw[:-tail].reshape(n_seq * n, -1)
    assert (body[:, width:] == 7.25).all()
    return body[:, :width].reshape(q.shape)


def check_attn(c, got, q, pos, scale=None, only=None):
    for b, p in enumerate(pos):
        if only is not None and b not in only:
            continue
        if p < 0 or p + q.shape[1] > c.cap:
            assert (got[b] == 0).all()
            continue
        want, tol = R.attend(q[b], c.want[b, 0], c.want[b, 1], p, scale)
        np.testing.assert_array_equal(np.isnan(got[b]), np.isnan(want))
        err = np.abs(got[b] - want)
        with np.errstate(all="ignore"):
            worst = np.nanmax(err / tol) if np.isfinite(want).any() else 0.0
        assert worst <= 1.0, f"sequence {b}: {worst:.3g} times the bound"


# ---- rows written and read --------------------------------------------------------

HEADS = [(1, 16), (2, 16), (3, 32), (2, 64), (8, 128), (1, 256), (4, 256)]


@pytest.mark.parametrize("nkv,hd", HEADS)
@pytest.mark.parametrize("cap,pos,n", [(1, 0, 1), (7, 2, 5), (65, 0, 65), (300, 17, 100)])
def test_write_and_read(T, H, nkv, hd, cap, pos, n):
    rng = np.random.default_rng(cap * 1000 + nkv * 10 + hd)
    c = Cache(T, H, cap, nkv, hd)
    k, v = rows(rng, c, n), rows(rng, c, n)
    c.write(k, v, [pos])
    c.check()  # the rows, and nothing else
    width = nkv * hd
    kd, vd = (H.DeviceBuffer.from_array(np.full(n * width + 16, 3.5, np.float32)) for _ in range(2))
    T.kv4_read(c.kv, kd.addr, vd.addr, n, pos=pos)
    H.synchronize()
    for d, x in ((kd, k), (vd, v)):
        got = d.to_array(np.float32, n * width + 16)
        np.testing.assert_array_equal(got[:-16].reshape(1, n, nkv, hd), R.stands_for(x).astype(np.float32))
        assert (got[-16:] == 3.5).all()


def test_write_rounds_and_scales_by_the_definition(T, H):
    """Every threshold and its neighbours at many scales, both signs, maxima
    around 7 times a power of two, the ends of the scale's range, zeros,
    subnormals, infinities and NaN."""
    rng = np.random.default_rng(5)
    th = np.array([0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7], np.float32)
    near = np.concatenate([th, np.nextafter(th, np.float32(np.inf)), np.nextafter(th, np.float32(-np.inf))])
    out = []
    for e in [-149, -140, -126, -110, -103, -102, -101, -100, -99, -64, -20, -1, 0, 1, 7, 40, 100, 119, 122, 124, 125, 126]:
        for top in (3.5, 3.75, 4.0, 5.0, 6.0, 6.9999995, 7.0, 7.0000005, 7.5, 7.9999995):
            g = rng.choice(near, 32) * rng.choice([-1, 1], 32)
            g[rng.integers(32)] = top
            with np.errstate(all="ignore"):
                out.append(np.clip(g.astype(np.float64) * 2.0 ** e, -3.4028234e38, 3.4028234e38).astype(np.float32))
    for bad in (np.inf, -np.inf, np.nan):
        g = rng.standard_normal(32).astype(np.float32)
        g[rng.integers(32)] = bad
        out.append(g)
    out.append(np.zeros(32, np.float32))
    out.append(-np.zeros(32, np.float32))
    out += [np.zeros(32, np.float32)] * (-len(out) % 8)
    k = np.stack(out).reshape(1, -1, 2, 128)
    c = Cache(T, H, k.shape[1] + 1, 2, 128)
    c.write(k, k[:, ::-1].copy(), [1])
    c.check()


@pytest.mark.parametrize("hd", [16, 128])
def test_write_batch_by_device_positions(T, H, hd):
    """Idle slots, rows that would pass the capacity and the sequences' gaps
    stay as they were; strided rows."""
    rng = np.random.default_rng(hd)
    c = Cache(T, H, 40, 2, hd, n_seq=6, gap=48)
    pos = [3, -1, 36, 37, 0, -2147483648]
    k, v = rows(rng, c, 4), rows(rng, c, 4)
    c.write(k, v, pos, dev=ints(H, pos), stride=2 * hd + 12)
    c.check()
    raw = c.buf.to_array(np.uint8, c.stride * 6).reshape(6, -1)
    assert (raw[:, c.size:] == 255).all() and (raw[1] == 255).all() and (raw[3] == 255).all()
    # read: zeros for the sequences that take no part, gaps left
    stride = 2 * hd + 4
    kd = H.DeviceBuffer.from_array(np.full((24, stride), 9.0, np.float32))
    T.kv4_read(c.kv, kd.addr, 0, 4, pos_dev=ints(H, pos).addr, row_stride=stride)
    H.synchronize()
    got = kd.to_array(np.float32, 24 * stride).reshape(6, 4, stride)
    assert (got[..., 2 * hd:] == 9.0).all()
    want = R.stands_for(k).reshape(6, 4, -1)
    for b, p in enumerate(pos):
        np.testing.assert_array_equal(got[b, :, :2 * hd], want[b] if p in (3, 36, 0) else np.zeros((4, 2 * hd)))


# ---- attention ----------------------------------------------------------------------

@pytest.mark.parametrize("ctx", [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 257, 640, 1111])
def test_attn_single_token(T, H, ctx):
    rng = np.random.default_rng(ctx)
    c = Cache(T, H, 1200, 2, 128)
    c.fill(rng, ctx)
    q = rng.standard_normal((1, 1, 4, 128)).astype(np.float32)
    check_attn(c, attend(c, q, [ctx - 1]), q, [ctx - 1])


@pytest.mark.parametrize("hd", [16, 64, 128, 256])
@pytest.mark.parametrize("fill", [0xFD, 0xFE, 0x7F, None])
def test_attn_never_uses_unwritten_rows(T, H, hd, fill):
    """Whatever the memory held: any scale byte, any code."""
    rng = np.random.default_rng(hd)
    c = Cache(T, H, 300, 2, hd, n_seq=2)
    raw = rng.integers(0, 256, c.buf.nbytes, np.uint8) if fill is None else np.full(c.buf.nbytes, fill, np.uint8)
    for ctx, n in ((1, 1), (20, 3), (140, 1), (200, 40)):
        H.copy_device(c.buf, H.DeviceBuffer.from_array(raw), raw.size)
        one = T.Kv4(c.buf.addr, cap=300, nkv=2, hd=hd)
        for kv, seqs in ((one, 1), (c.kv, 2)):
            c.n_seq, kept = seqs, c.kv
            c.kv = kv
            c.want[:] = np.nan
            k, v = c.fill(rng, ctx)
            q = rng.standard_normal((seqs, n, 4, hd)).astype(np.float32)
            pos = [ctx - n] * seqs
            check_attn(c, attend(c, q, pos), q, pos)
            new = rows(rng, c, 1), rows(rng, c, 1)
            check_attn(c, attend(c, q[:, :1], [ctx] * seqs, new=new), q[:, :1], [ctx] * seqs)
            c.kv = kept


@pytest.mark.parametrize("nkv,hd", HEADS)
@pytest.mark.parametrize("group", [1, 2, 3, 4, 8, 20])
def test_attn_head_layouts(T, H, nkv, hd, group):
    rng = np.random.default_rng(nkv * 100 + hd + group)
    c = Cache(T, H, 300, nkv, hd)
    c.fill(rng, 300)
    for n in (1, 7):
        q = rng.standard_normal((1, n, nkv * group, hd)).astype(np.float32)
        pos = [int(rng.integers(0, 300 - n))]
        check_attn(c, attend(c, q, pos), q, pos)


@pytest.mark.parametrize("hd,group", [(16, 2), (64, 4), (128, 2), (128, 4), (128, 1), (256, 2)])
@pytest.mark.parametrize("n,pos", [(2, 0), (8, 5), (17, 0), (33, 31), (64, 64), (45, 300), (130, 0), (200, 77)])
def test_attn_pieces(T, H, hd, group, n, pos):
    rng = np.random.default_rng(n * 7 + hd + group)
    c = Cache(T, H, pos + n + 3, 2, hd)
    c.fill(rng, pos + n)
    q = rng.standard_normal((1, n, 2 * group, hd)).astype(np.float32)
    check_attn(c, attend(c, q, [pos]), q, [pos])


@pytest.mark.parametrize("n,pos", [(257, 0), (300, 1000)])
def test_attn_longer_pieces(T, H, n, pos):
    rng = np.random.default_rng(n)
    c = Cache(T, H, pos + n, 1, 128)
    c.fill(rng, pos + n)
    q = rng.standard_normal((1, n, 2, 128)).astype(np.float32)
    check_attn(c, attend(c, q, [pos]), q, [pos])


@pytest.mark.parametrize("hd,group,n", [(16, 2, 33), (32, 3, 45), (64, 4, 9), (64, 2, 100), (128, 2, 17), (128, 2, 100),
                                        (128, 4, 40), (128, 8, 16), (128, 1, 129), (256, 2, 20), (256, 4, 33)])
def test_attn_prompts_of_many_sequences(T, H, hd, group, n):
    """Enough tiles of columns for the prompts' kernel: first pieces and later
    ones, one column past a tile, idle slots, values and keys that are not
    finite, strided rows."""
    rng = np.random.default_rng(hd + group + n)
    c = Cache(T, H, n + 150, 4, hd, n_seq=128, gap=32)

    def spoil(k, at):
        k[5, at, 1, hd // 2] = np.nan
        k[7, at + 60, 0, 0] = np.inf
        return k
    c.fill(rng, n + 140, keys=lambda k: spoil(k, 61), values=lambda v: spoil(v, 63))
    pos = [int(x) for x in rng.integers(0, 140, 128)]
    pos[0], pos[1], pos[2], pos[3], pos[4], pos[5], pos[7] = 0, 150, -1, 151, 64, 40, 61
    q = rng.standard_normal((128, n, 4 * group, hd)).astype(np.float32)
    w = 4 * group * hd
    got = attend(c, q, pos, dev=ints(H, pos), q_stride=w + 4, out_stride=w + 12)
    check_attn(c, got, q, pos, only=(0, 1, 2, 3, 4, 5, 7, 8, 127))
    # appended first: the same rows as written by themselves
    new = rows(rng, c, n), rows(rng, c, n)
    got = attend(c, q, pos, dev=ints(H, pos), new=new)
    c.check()
    check_attn(c, got, q, pos, only=(0, 3, 9))


def test_attn_long_prompt(T, H):
    """One sequence of more than 2048 rows."""
    rng = np.random.default_rng(77)
    c = Cache(T, H, 2200, 8, 128)
    c.fill(rng, 2200)
    q = rng.standard_normal((1, 2100, 16, 128)).astype(np.float32)
    got = attend(c, q, [71])
    for t in (0, 1, 63, 64, 1000, 2047, 2099):
        check_attn(c, got[:, t:t + 1], q[:, t:t + 1], [71 + t])


def test_attn_longer_prompt(T, H):
    """Enough rows of one sequence for the prompts' kernel."""
    rng = np.random.default_rng(78)
    c = Cache(T, H, 3021, 8, 128)
    c.fill(rng, 3021)
    q = rng.standard_normal((1, 3000, 16, 128)).astype(np.float32)
    got = attend(c, q, [21])
    for t in (0, 1, 63, 64, 1000, 2047, 2999):
        check_attn(c, got[:, t:t + 1], q[:, t:t + 1], [21 + t])


@pytest.mark.parametrize("hd,group,n", [(32, 2, 17), (64, 4, 9), (128, 2, 32), (256, 3, 11)])
def test_attn_prompts_of_one_tile(T, H, hd, group, n):
    """More sequences, each of one tile of columns."""
    rng = np.random.default_rng(hd + group + n)
    c = Cache(T, H, n + 100, 4, hd, n_seq=180)
    c.fill(rng, n + 100)
    pos = [int(x) for x in rng.integers(0, 100, 180)]
    pos[0], pos[1], pos[2], pos[3] = 0, 100, -1, 101
    q = rng.standard_normal((180, n, 4 * group, hd)).astype(np.float32)
    check_attn(c, attend(c, q, pos, dev=ints(H, pos)), q, pos, only=(0, 1, 2, 3, 90, 179))


@pytest.mark.parametrize("n_seq,nkv,group,cap", [(2, 4, 2, 3000), (63, 2, 2, 1600), (64, 8, 1, 900), (65, 1, 4, 2500),
                                                 (130, 1, 2, 1500), (256, 2, 3, 700), (512, 1, 2, 700), (513, 1, 2, 600)])
def test_attn_of_many_ragged_sequences(T, H, n_seq, nkv, group, cap):
    """A few long sequences among short ones and idle slots, up to as many as
    share a launch's workgroups, and one more."""
    rng = np.random.default_rng(n_seq)
    c = Cache(T, H, cap, nkv, 16, n_seq=n_seq)
    c.fill(rng, cap)
    pos = rng.integers(0, 40, n_seq)
    pos[rng.integers(0, n_seq, max(2, n_seq // 4))] = rng.integers(cap // 2, cap, max(2, n_seq // 4))
    pos[rng.integers(0, n_seq, n_seq // 9)] = -1
    pos[0], pos[-1] = cap - 1, rng.integers(0, cap)
    pos = [int(p) for p in pos]
    q = rng.standard_normal((n_seq, 1, nkv * group, 16)).astype(np.float32)
    check_attn(c, attend(c, q, pos, dev=ints(H, pos)), q, pos)


@pytest.mark.parametrize("hd", [16, 32, 64, 128, 256])
def test_attn_prompts_with_values_of_all_sizes(T, H, hd):
    """Sequences of values around 1, growing by 2^60 within a block of keys and
    between blocks, shrinking, with zeros, and of 2^-60 only."""
    rng = np.random.default_rng(hd)
    c = Cache(T, H, 400, 4, hd, n_seq=128)
    size = np.zeros((128, 400))
    size[1] = np.repeat([-60, -30, 0, 5, 30, 60, 20, -20], 50)
    size[2] = rng.integers(-12, 13, 400)
    size[3] = rng.integers(-60, 61, 400)
    size[4] = -60
    size[5] = np.linspace(60, -60, 400)
    size[6] = np.where(np.arange(400) % 100 < 70, -40, 40)
    size[7] = np.where(np.arange(400) < 200, -110, 0)

    def sized(v):
        v = (v * np.exp2(size)[..., None, None]).astype(np.float32)
        v[8, 100:300] = 0.0
        v[9] = 0.0
        v[6, 150, 0, 0] = np.inf
        return v
    c.fill(rng, 400, values=sized)
    q = rng.standard_normal((128, 36, 8, hd)).astype(np.float32)
    pos = [364] * 128
    pos[1], pos[6] = 300, 130
    got = attend(c, q, pos, dev=ints(H, pos))
    check_attn(c, got, q, pos, only=range(12))


def test_attn_sharp_and_flat_softmax(T, H):
    """Scores of some hundreds, one dominant key, and equal keys."""
    rng = np.random.default_rng(9)
    c = Cache(T, H, 500, 2, 64)
    c.fill(rng, 500, keys=lambda k: (k * np.where(np.arange(500) % 250 < 125, 8.0, 0.0)[None, :, None, None]).astype(np.float32))
    q = (6 * rng.standard_normal((1, 3, 8, 64))).astype(np.float32)
    check_attn(c, attend(c, q, [497]), q, [497])
    check_attn(c, attend(c, q, [497], scale=1e-3), q, [497], scale=np.float64(np.float32(1e-3)))


@pytest.mark.parametrize("n", [1, 5])
@pytest.mark.parametrize("nkv,hd,group", [(2, 16, 2), (8, 128, 2), (2, 128, 4)])
def test_attn_batch_by_device_positions(T, H, n, nkv, hd, group):
    """Ragged positions, an idle slot in the middle and at the end, one past
    the capacity; strided rows of q and of the output."""
    rng = np.random.default_rng(n + hd)
    c = Cache(T, H, 700, nkv, hd, n_seq=7, gap=16)
    c.fill(rng, 700)
    pos = [0, 131, -1, 695, 699 if n == 1 else 700, 12, -5]
    q = rng.standard_normal((7, n, nkv * group, hd)).astype(np.float32)
    w = nkv * group * hd
    check_attn(c, attend(c, q, pos, dev=ints(H, pos), q_stride=w + 8, out_stride=w + 20), q, pos)


@pytest.mark.parametrize("n", [1, 6, 40])
@pytest.mark.parametrize("hd", [16, 32, 64, 128, 256])
def test_attn_appends_rows(T, H, n, hd):
    """New rows are written, and attended to, in the same call; a run of calls
    as a session makes them."""
    rng = np.random.default_rng(n + hd)
    c = Cache(T, H, 400, 2, hd, n_seq=3)
    at = [0, 64, 250]
    c.fill(rng, 250)
    for step in range(3):
        pos = [p + step * n for p in at]
        new = rows(rng, c, n), rows(rng, c, n)
        q = rng.standard_normal((3, n, 4, hd)).astype(np.float32)
        got = attend(c, q, pos, dev=ints(H, pos), new=new, new_stride=2 * hd + 4)
        c.check()
        check_attn(c, got, q, pos)


@pytest.mark.parametrize("n_seq", [1, 4])
@pytest.mark.parametrize("n,group", [(1, 2), (1, 3), (1, 20), (5, 2)])
@pytest.mark.parametrize("hd", [16, 32, 64, 128, 256])
def test_attn_appends_rows_to_shared_sequences(T, H, n_seq, n, group, hd):
    """Positions of which several workgroups take a part, and the step from one
    workgroup to several; marked groups of values and keys among them."""
    rng = np.random.default_rng(n + hd + group)
    c = Cache(T, H, 1500, 2, hd, n_seq=n_seq)

    def spoil(x, at):
        x[n_seq - 1, at, 1, hd // 2] = np.inf
        return x
    c.fill(rng, 1480, keys=lambda k: spoil(k, 1300), values=lambda v: spoil(v, 700))
    at = [1470, 510, -1, 1280][:n_seq]
    for step in range(4):
        pos = [p + step * n if p >= 0 else p for p in at]
        new = rows(rng, c, n), rows(rng, c, n)
        if step == 2:
            new[1][0, 0, 0, 3] = np.nan
        q = rng.standard_normal((n_seq, n, 2 * group, hd)).astype(np.float32)
        got = attend(c, q, pos, dev=ints(H, pos), new=new)
        c.check()
        check_attn(c, got, q, pos)


@pytest.mark.parametrize("n", [1, 40])
def test_attn_append_idle_slots_write_nothing(T, H, n):
    rng = np.random.default_rng(n)
    c = Cache(T, H, 200, 2, 128, n_seq=3)
    c.fill(rng, 150)
    pos = [150, -1, 201 - n]
    q = rng.standard_normal((3, n, 4, 128)).astype(np.float32)
    got = attend(c, q, pos, dev=ints(H, pos), new=(rows(rng, c, n), rows(rng, c, n)))
    c.check()
    check_attn(c, got, q, pos)


@pytest.mark.parametrize("hd", [16, 64, 128, 256])
@pytest.mark.parametrize("n,pos", [(1, 200), (9, 195), (60, 150), (140, 60)])
def test_attn_not_finite_values(T, H, hd, n, pos):
    """A group of values with an infinity or a NaN makes its 32 dimensions NaN
    for the rows that see it, and for no others."""
    rng = np.random.default_rng(hd + n)
    c = Cache(T, H, pos + n, 2, hd)

    def spoil(v):
        v[0, pos + n // 2, 0, hd - 1] = np.inf
        v[0, pos + n - 1, 1, 0] = np.nan
        return v
    c.fill(rng, pos + n, values=spoil)
    q = rng.standard_normal((1, n, 4, hd)).astype(np.float32)
    got = attend(c, q, [pos])
    check_attn(c, got, q, [pos])
    assert np.isnan(got).any() and (n == 1 or not np.isnan(got[0, 0]).any())


@pytest.mark.parametrize("hd", [16, 64, 128, 256])
@pytest.mark.parametrize("n,pos", [(1, 200), (9, 195), (60, 150), (140, 60)])
def test_attn_not_finite_keys(T, H, hd, n, pos):
    """A key with a NaN makes the rows that see it NaN, and no others."""
    rng = np.random.default_rng(hd + n)
    c = Cache(T, H, pos + n, 2, hd)

    def spoil(k):
        k[0, pos + n // 2, 0, 0] = np.nan
        return k
    c.fill(rng, pos + n, keys=spoil)
    q = rng.standard_normal((1, n, 4, hd)).astype(np.float32)
    got = attend(c, q, [pos])
    check_attn(c, got, q, [pos])
    assert np.isnan(got[0, n // 2:, :2]).all() and not np.isnan(got[0, :, 2:]).any()


def test_attn_all_keys_not_finite(T, H):
    """Runs of keys without a single finite score are not left out."""
    rng = np.random.default_rng(1)
    c = Cache(T, H, 1000, 1, 64)

    def spoil(k):
        k[0, 300:700] = np.nan
        return k
    c.fill(rng, 1000, keys=spoil)
    q = rng.standard_normal((1, 1, 2, 64)).astype(np.float32)
    for p in (299, 300, 999):
        got = attend(c, q, [p])
        assert np.isnan(got).all() == (p >= 300)
        check_attn(c, got, q, [p])


def test_attn_not_finite_queries(T, H):
    """A query row with an infinity or a NaN is NaN; its neighbours are not."""
    rng = np.random.default_rng(2)
    c = Cache(T, H, 300, 2, 128)
    c.fill(rng, 300)
    q = rng.standard_normal((1, 20, 4, 128)).astype(np.float32)
    q[0, 3, 1, 77] = np.nan
    q[0, 11, 2, 0] = np.inf
    got = attend(c, q, [280])
    bad = np.isnan(got).all(-1)[0]
    assert bad[3, 1] and bad[11, 2] and bad.sum() == 2
    q = np.nan_to_num(q, nan=0.0, posinf=0.0)
    again = attend(c, q, [280])
    assert (got[0][~bad] == again[0][~bad]).all()
    check_attn(c, again, q, [280])


def test_attn_large_and_small_magnitudes(T, H):
    """Values around 2^60 and 2^-60 and in one sequence; scores whose spread
    is past f32's exponential."""
    rng = np.random.default_rng(4)
    c = Cache(T, H, 260, 2, 128)
    c.fill(rng, 260, values=lambda v: (v * np.exp2(rng.integers(-60, 61, (1, 260, 1, 1)))).astype(np.float32),
           keys=lambda k: (k * np.exp2(rng.integers(-6, 4, (1, 260, 1, 1)))).astype(np.float32))
    q = rng.standard_normal((1, 2, 4, 128)).astype(np.float32)
    check_attn(c, attend(c, q, [258]), q, [258])


def test_host_memory_is_refused(T, H):
    """Before anything is launched."""
    from tinyminigo_amd._lib import TMG_E_INVALID
    host = np.zeros(T.kv4_bytes(64, 2, 64) + 16, np.uint8)
    kv = T.Kv4((host.ctypes.data + 15) // 16 * 16, cap=64, nkv=2, hd=64)
    dev = H.DeviceBuffer(1 << 16)
    for call in (lambda: T.kv4_write(kv, dev.addr, dev.addr, 1), lambda: T.kv4_read(kv, dev.addr, dev.addr, 1),
                 lambda: T.kv4_attn(kv, dev.addr, dev.addr + 4096, 1, 4)):
        with pytest.raises(T.TmgError) as e:
            call()
        assert e.value.code == TMG_E_INVALID


def test_attn_on_a_stream_and_in_graphs(T, H):
    """A decode step's append and attention captured by device position and
    replayed as the position advances, two graphs with one workspace in one
    stream; every replay against the eager result."""
    rng = np.random.default_rng(8)
    c, e = (Cache(T, H, 600, 2, 128, n_seq=2) for _ in range(2))
    k0, v0 = c.fill(rng, 300)
    e.write(k0, v0, [0, 0])
    width, nq = 2 * 128, 4
    s = H.Stream()
    kd, vd = H.DeviceBuffer(2 * width * 4), H.DeviceBuffer(2 * width * 4)
    qd = [H.DeviceBuffer(2 * nq * 128 * 4) for _ in range(2)]
    out = [H.DeviceBuffer(2 * nq * 128 * 4) for _ in range(2)]
    pd = ints(H, [0, 0])
    ws = H.DeviceBuffer(T.kv4_attn_workspace(c.kv, 1, nq))
    ws.fill_byte(0)

    def step(i):
        def go(st):
            T.kv4_attn(c.kv, qd[i].addr, out[i].addr, 1, nq, pos_dev=pd.addr, k_dev=kd.addr, v_dev=vd.addr,
                       ws_dev=ws.addr, ws_bytes=ws.nbytes, stream=st.addr)
        return go
    graphs = [H.Graph(s, step(i)) for i in range(2)]
    for n in range(4):
        pos = [300 + n, 17 + n]
        new = rows(rng, c, 1), rows(rng, c, 1)
        q = rng.standard_normal((2, 2, 1, nq, 128)).astype(np.float32)
        for d, x in [(kd, new[0]), (vd, new[1]), (qd[0], q[0]), (qd[1], q[1]), (pd, np.asarray(pos, np.int32))]:
            H.copy_device(d, H.DeviceBuffer.from_array(x), x.nbytes)
        for g in graphs:
            g.launch()
        s.synchronize()
        c.expect(new[0], new[1], pos)
        for i in range(2):
            got = out[i].to_array(np.float32, q[i].size).reshape(q[i].shape)
            eager = attend(e, q[i], pos, dev=ints(H, pos), new=new)
            np.testing.assert_array_equal(got, eager)
            check_attn(c, got, q[i], pos)
        c.check()


@pytest.mark.parametrize("n_seq", [1, 3])
def test_shared_sequences_in_graphs(T, H, n_seq):
    """Two graphs with one workspace whose sequences grow from one workgroup to
    several, an eager call between the replays."""
    rng = np.random.default_rng(80 + n_seq)
    c = Cache(T, H, 1600, 2, 128, n_seq=n_seq)
    c.fill(rng, 1600)
    nq, s = 4, H.Stream()
    size = n_seq * nq * 128
    qd, out = ([H.DeviceBuffer(size * 4) for _ in range(2)] for _ in range(2))
    pd = ints(H, [0] * n_seq)
    ws = H.DeviceBuffer(T.kv4_attn_workspace(c.kv, 1, nq))
    ws.fill_byte(0)

    def step(i):
        return lambda st: T.kv4_attn(c.kv, qd[i].addr, out[i].addr, 1, nq, pos_dev=pd.addr, ws_dev=ws.addr,
                                     ws_bytes=ws.nbytes, stream=st.addr)
    graphs = [H.Graph(s, step(i)) for i in range(2)]
    for first in (510, 511, 512, 1599, 700, 1100):
        pos = [first, 900, 20][:n_seq]
        q = rng.standard_normal((2, n_seq, 1, nq, 128)).astype(np.float32)
        for d, x in [(qd[0], q[0]), (qd[1], q[1]), (pd, np.asarray(pos, np.int32))]:
            H.copy_device(d, H.DeviceBuffer.from_array(x), x.nbytes)
        for g in graphs:
            g.launch()
        s.synchronize()
        for i in range(2):
            got = out[i].to_array(np.float32, size).reshape(q[i].shape)
            np.testing.assert_array_equal(got, attend(c, q[i], pos, dev=ints(H, pos)))
            check_attn(c, got, q[i], pos)


def test_attn_two_streams_at_once(T, H):
    """Calls with a workspace each overlap on two streams."""
    rng = np.random.default_rng(12)
    c = Cache(T, H, 3000, 2, 128)
    c.fill(rng, 3000)
    nq, streams = 4, [H.Stream(), H.Stream()]
    q = rng.standard_normal((8, 1, 1, nq, 128)).astype(np.float32)
    qd = [H.DeviceBuffer.from_array(x) for x in q]
    out = [H.DeviceBuffer(nq * 512) for _ in q]
    ws = [H.DeviceBuffer(T.kv4_attn_workspace(c.kv, 1, nq)) for _ in streams]
    for w in ws:
        w.fill_byte(0)
    for i in range(8):
        T.kv4_attn(c.kv, qd[i].addr, out[i].addr, 1, nq, pos=2990 + i, ws_dev=ws[i % 2].addr, ws_bytes=ws[i % 2].nbytes,
                   stream=streams[i % 2].addr)
    for s in streams:
        s.synchronize()
    for i in range(8):
        check_attn(c, out[i].to_array(np.float32, nq * 128).reshape(q[i].shape), q[i], [2990 + i])


def test_attn_is_the_same_every_time(T, H):
    rng = np.random.default_rng(13)
    c = Cache(T, H, 2000, 8, 128)
    c.fill(rng, 2000)
    for n in (1, 30):
        q = rng.standard_normal((1, n, 16, 128)).astype(np.float32)
        first = attend(c, q, [1900])
        for _ in range(5):
            np.testing.assert_array_equal(first, attend(c, q, [1900]))


def test_offsets_past_32_bits(T, H):
    """A cache of 2^22 + 64 positions, 4.6 GB: the same 2^16 rows over and
    over, so that the attention over all of them is the one over a copy."""
    rng = np.random.default_rng(21)
    nkv, hd, part, copies = 8, 128, 1 << 16, 64
    cap = part * copies + 64
    buf = H.DeviceBuffer(T.kv4_bytes(cap, nkv, hd))
    kv = T.Kv4(buf.addr, cap=cap, nkv=nkv, hd=hd)
    k, v = (rng.standard_normal((part, nkv, hd), dtype=np.float32) for _ in range(2))
    kd, vd = H.DeviceBuffer.from_array(k), H.DeviceBuffer.from_array(v)
    for i in range(copies):
        T.kv4_write(kv, kd.addr, vd.addr, part, pos=i * part)
    H.synchronize()
    for pos in (0, part * (copies - 1) + 5, part * copies - 3):
        back = H.DeviceBuffer(3 * nkv * hd * 4)
        T.kv4_read(kv, 0, back.addr, 3, pos=pos)
        H.synchronize()
        np.testing.assert_array_equal(back.to_array(np.float32, 3 * nkv * hd).reshape(3, nkv, hd),
                                      R.stands_for(v[np.arange(pos, pos + 3) % part]).astype(np.float32))
    q = rng.standard_normal((1, 1, 16, hd)).astype(np.float32)
    qd, out = H.DeviceBuffer.from_array(q), H.DeviceBuffer(16 * hd * 4)
    ws = H.DeviceBuffer(T.kv4_attn_workspace(kv, 1, 16))
    ws.fill_byte(0)
    T.kv4_attn(kv, qd.addr, out.addr, 1, 16, pos=part * copies - 1, ws_dev=ws.addr, ws_bytes=ws.nbytes)
    H.synchronize()
    got = out.to_array(np.float32, 16 * hd).reshape(16, hd)
    kk, vv = R.stands_for(k).transpose(1, 0, 2), R.stands_for(v).transpose(1, 0, 2)
    want, tol = R.attend(q[0], kk, vv, part - 1)
    # 64 times the weights: the bound's n / 8 grows by as much
    tol *= (4 + 2 * (16 + part * copies / 8)) / (4 + 2 * (16 + part / 8))
    assert (np.abs(got - want[0]) <= tol[0]).all()
    assert np.linalg.norm(got - want[0]) <= 1e-5 * np.linalg.norm(want[0])
