"""GPU tests of zmi_lora_direct (through the C ABI) against the definition in float64.

Tolerance, element by element, from the roundings that are allowed on the way (u = 2^-24, all sums in f32, any order):
  h:      K products of 16-bit values (exact in f32) and their sum: (K + 4) u * sum |x A|; then at least 16 bits of its
          value are kept: 2^-16 |h|;
  delta:  |scale| * (sum (error of h) |B| + (3 rank + 8) u sum |h B|)   (h may be split in up to three terms);
  dst:    the sum with base and the rounding to dst's type: half a step, eps / 2 relative to the value (and half the
          smallest subnormal)."""
import ctypes as C

import numpy as np
import pytest
import torch

from zendnn_amd import capi, lowoha
from tests import gpu_helpers as H

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


class Case:
    """Inputs of one call; every buffer is wider than what the call may touch, by sentinels."""

    def __init__(self, seed, T, K, N, rank, S, dt=BF, dst=None, mixed=True, pad=0, w_pad=0, none=0.15, ids=None, scales=True):
        g = torch.Generator(device=H.DEV)
        g.manual_seed(seed)
        rn = lambda *s: torch.randn(*s, generator=g, device=H.DEV)   # noqa: E731
        self.T, self.K, self.N, self.rank, self.S, self.dt, self.dst_dt = T, K, list(N), rank, S, dt, dst or dt
        R, cols = len(N) * rank, sum(N)
        self.x = rn(T, K + pad).to(dt)[:, :K]
        self.a = (rn(S, R, K + w_pad) / K ** 0.5).to(dt)[:, :, :K]
        self.b = [(rn(S, n, rank + w_pad) * 0.2).to(dt)[:, :, :rank] for n in N]
        if ids is None:
            ids = torch.randint(0, S, (T,), generator=g, device=H.DEV, dtype=torch.int32)
            ids[torch.rand(T, generator=g, device=H.DEV) < none] = -1
        self.ids = ids
        self.ranks = torch.randint(0, rank + 1, (S,), generator=g, device=H.DEV, dtype=torch.int32) if mixed else None
        if mixed:
            self.ranks[0] = rank
            for s in range(S):       # what a slot holds beyond its adapter's rank is not used, whatever it is
                r = int(self.ranks[s])
                for i in range(len(N)):
                    self.a[s, i * rank + r:(i + 1) * rank] = float("nan")
                    self.b[i][s, :, r:] = float("nan")
        self.scales = torch.rand(S, generator=g, device=H.DEV) * 2 - 0.5 if scales else None
        self.base = rn(T, cols + pad).to(self.dst_dt)[:, :cols]
        self.full = torch.full((T + 2, cols + 3 + pad), -7.0, dtype=self.dst_dt, device=H.DEV)
        self.dst = self.full[1:T + 1, 1 + (pad > 0):][:, :cols] if pad else self.full[1:T + 1, :cols]

    def want(self, base):
        """(exact result, tolerance) in float64."""
        y = base.double() if base is not None else torch.zeros(self.T, sum(self.N), dtype=torch.float64, device=H.DEV)
        tol = torch.zeros_like(y)
        for s in sorted({int(i) for i in self.ids.tolist() if 0 <= i < self.S}):
            rows = (self.ids == s).nonzero()[:, 0]
            r = min(max(int(self.ranks[s]), 0), self.rank) if self.ranks is not None else self.rank
            if not len(rows) or not r:
                continue
            x, c = self.x[rows].double(), 0
            scale = float(self.scales[s]) if self.scales is not None else 1.0
            for i, n in enumerate(self.N):
                a = self.a[s, i * self.rank:i * self.rank + r].double()
                b = self.b[i][s, :, :r].double()
                h = x @ a.t()
                eh = (self.K + 4) * U * (x.abs() @ a.abs().t()) + 2.0 ** -16 * h.abs()
                y[rows, c:c + n] += scale * (h @ b.t())
                tol[rows, c:c + n] = abs(scale) * (eh @ b.abs().t() + (3 * r + 8) * U * (h.abs() @ b.abs().t()))
                c += n
        f = torch.finfo(self.dst_dt)
        has = ((self.ids >= 0) & (self.ids < self.S))[:, None]
        tol = tol + torch.where(has, (f.eps / 2 + U) * (y.abs() + tol) + f.smallest_normal * f.eps / 2, torch.zeros_like(y))
        return y, tol

    def call(self, base, dst=None, workspace=None):
        return lowoha.lora_direct(self.x, self.ids, self.a, self.b if len(self.b) > 1 else self.b[0],
                                  self.dst if dst is None else dst, base, self.ranks, self.scales, workspace)

    def check(self, where="other"):
        self.full.fill_(-7.0)
        base = None
        if where == "other":
            base = self.base
        elif where == "dst":
            self.dst.copy_(self.base)
            base = self.dst
        y, tol = self.want(self.base if where != "zero" else None)
        assert self.call(base) == capi.SUCCESS, lowoha.last_error()
        assert lowoha.last_kernel().startswith("lora")
        self.compare(self.dst, y, tol)
        edge = self.full.clone()
        edge[1:self.T + 1, self.dst.storage_offset() % self.full.shape[1]:][:, :sum(self.N)] = -7.0
        assert (edge == -7.0).all(), "wrote outside dst"
        return self.dst

    @staticmethod
    def compare(got, y, tol):
        err = (got.double() - y).abs()
        bad = ~(err <= tol)
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float((err / tol).nan_to_num().max()))


SHAPES = [
    # T, K, N, rank, slots
    (1, 64, [64], 8, 1), (1, 4096, [4096], 16, 4), (1, 1, [1], 1, 1), (2, 2048, [512], 8, 2), (5, 128, [96], 16, 3),
    (16, 4096, [1024, 256, 256], 16, 16), (17, 520, [200], 32, 2), (33, 1024, [64, 64], 64, 40), (48, 4096, [640, 128], 64, 64),
    (64, 512, [130], 4, 3), (65, 512, [128], 16, 3), (100, 14336, [256], 16, 6), (130, 1000, [512], 128, 2),
    (200, 256, [256, 8, 24, 40], 24, 7), (257, 768, [1024], 256, 3), (300, 4096, [256], 8, 16), (513, 640, [320], 48, 1),
    (1000, 264, [72], 12, 300), (2049, 192, [136], 40, 5)]
ODD = [(1, 7, [3], 3, 2), (3, 77, [33], 5, 2), (31, 1001, [273], 12, 9), (70, 65, [65, 1, 3], 7, 4), (301, 333, [111], 9, 9),
       (129, 4099, [259], 33, 3), (40, 130, [66], 130, 3), (90, 63, [1], 1, 90)]


@pytest.mark.parametrize("T,K,N,rank,S", SHAPES + ODD)
@pytest.mark.parametrize("dt,dst", [(BF, BF), (HF, HF), (BF, F32)])
def test_random(T, K, N, rank, S, dt, dst):
    c = Case(T * 3 + K, T, K, N, rank, S, dt, dst)
    for where in ("other", "dst", "zero"):
        c.check(where)


@pytest.mark.parametrize("dt,dst", [(BF, HF), (HF, BF), (HF, F32)])
@pytest.mark.parametrize("T,K,N,rank,S", [(9, 512, [192], 16, 3), (150, 512, [192, 64], 32, 3), (77, 321, [99], 10, 3)])
def test_other_type_pairs(T, K, N, rank, S, dt, dst):
    c = Case(T, T, K, N, rank, S, dt, dst)
    c.check("other")
    c.check("dst")


@pytest.mark.parametrize("T,K,N,rank,S", [(1, 512, [256], 16, 2), (20, 512, [256, 64], 16, 3), (300, 512, [256], 64, 3), (300, 512, [252], 8, 3)])
@pytest.mark.parametrize("pad,w_pad", [(8, 0), (0, 8), (1, 0), (0, 1), (5, 3), (4, 4), (2, 2)])
def test_strides(T, K, N, rank, S, pad, w_pad):
    """Rows and weights inside wider buffers, with strides that keep and that break the alignment of vector accesses."""
    Case(T + pad, T, K, N, rank, S, BF, BF, pad=pad, w_pad=w_pad).check("other")
    Case(T + pad, T, K, N, rank, S, HF, F32, mixed=False, pad=pad, w_pad=w_pad, scales=False).check("dst")


@pytest.mark.parametrize("which", ["x", "a", "b", "base", "dst"])
@pytest.mark.parametrize("T", [1, 40, 200])
def test_addresses_that_are_not_aligned_for_vectors(which, T):
    c = Case(T, T, 512, [256], 16, 3)
    move = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device=H.DEV)[1:].view(t.shape).copy_(t)   # noqa: E731
    if which == "b":
        c.b = [move(c.b[0])]
    elif which == "dst":
        c.full = torch.full((c.full.numel() + 1,), -7.0, dtype=c.dst_dt, device=H.DEV)[1:].view(c.full.shape)
        c.dst = c.full[1:T + 1, :256]
        y, tol = c.want(c.base)
        assert c.call(c.base) == capi.SUCCESS
        return c.compare(c.dst, y, tol)
    else:
        setattr(c, which, move(getattr(c, which)))
    c.check("other")


@pytest.mark.parametrize("T", [1, 16, 64, 65, 500])
def test_slot_ids(T):
    """No adapter anywhere, one adapter everywhere, ids outside the slots, runs and interleaved ids."""
    i32 = dict(dtype=torch.int32, device=H.DEV)
    for ids in (torch.full((T,), -1, **i32), torch.full((T,), 2, **i32), torch.full((T,), 3, **i32),
                torch.tensor([-2 ** 31, 2 ** 31 - 1, 3, 0, -1, 65536] * T, **i32)[:T], torch.arange(T, **i32) % 3,
                torch.arange(T, **i32) * 3 // T, (torch.arange(T, **i32) % 17 == 16).int() * 2):
        c = Case(T, T, 512, [192], 16, 3, ids=ids, mixed=False)
        c.check("dst")
        c.check("other")
        c.check("zero")


def test_in_place_leaves_rows_without_an_adapter_alone():
    """Bit for bit, NaN payloads included."""
    for T in (8, 300):
        c = Case(1, T, 256, [128], 16, 3, none=0.5)
        bits = torch.randint(-2 ** 15, 2 ** 15, c.base.shape, device=H.DEV, dtype=torch.int16)
        none = c.ids < 0
        c.dst.copy_(c.base)
        c.dst.view(torch.int16)[none] = bits[none]
        assert c.call(c.dst) == capi.SUCCESS
        assert torch.equal(c.dst.view(torch.int16)[none], bits[none])


@pytest.mark.parametrize("T", [4, 48, 200])
def test_what_is_not_finite_stays_in_its_row(T):
    """NaN and infinite rows, slots that nobody uses, and stale workspace contents."""
    c = Case(5, T, 512, [192], 16, 4, mixed=False, ids=torch.arange(T, dtype=torch.int32, device=H.DEV) % 3)
    c.a[3] = float("nan")
    c.b[0][3] = float("inf")
    y, tol = c.want(c.base)
    c.x[1] = float("nan")
    c.x[2, 5] = float("inf")
    size = lowoha.lora_workspace_size(c.x, c.ids, c.a, c.b, c.dst)
    ws = torch.full((max(size, 16),), 0xff, dtype=torch.uint8, device=H.DEV)
    assert c.call(c.base, workspace=ws) == capi.SUCCESS
    keep = [t for t in range(T) if t not in (1, 2)]
    c.compare(c.dst[keep], y[keep], tol[keep])
    assert torch.isnan(c.dst[1]).all() and not torch.isfinite(c.dst[2]).any()


def test_values_near_the_limits_of_f16():
    """h beyond what f16 holds, products that come back into range, and results that round to infinity."""
    for T in (3, 100):
        c = Case(11, T, 512, [128], 16, 2, HF, HF, mixed=False, none=0.0)
        c.x.mul_(200.0)
        c.a.mul_(300.0)
        c.b[0].mul_(2.0 ** -12)
        c.check("other")
        c = Case(12, T, 512, [128], 16, 2, HF, HF, mixed=False, none=0.0)
        c.x.mul_(2.0 ** -9)
        c.a.mul_(2.0 ** -8)
        c.check("zero")
        c = Case(13, T, 64, [64], 8, 1, HF, HF, mixed=False, none=0.0, scales=False)
        c.x.fill_(100.0)
        c.a.fill_(100.0)
        c.b[0].fill_(100.0)
        assert c.call(None) == capi.SUCCESS
        assert (c.dst == float("inf")).all()


def test_repeated_calls_and_batch_mates_do_not_change_the_bits():
    c = Case(21, 180, 2048, [512], 32, 4)
    c.check("other")
    first = c.dst.clone()
    for _ in range(3):
        assert c.call(c.base) == capi.SUCCESS
        assert torch.equal(c.dst, first)


def test_empty_batch():
    c = Case(1, 4, 64, [32], 8, 2)
    z = lambda t: t[:0]   # noqa: E731
    assert lowoha.lora_direct(z(c.x), z(c.ids), c.a, c.b[0], z(c.dst), z(c.base)) == capi.SUCCESS
    assert (c.full == -7.0).all()


@pytest.mark.parametrize("T", [1, 24, 700])
def test_captured_graphs_with_their_own_workspaces(T):
    """Two graphs of different sizes replayed in turn, beside eager calls that use the thread's own scratch."""
    lib, s = capi.load(), torch.cuda.Stream()
    cases = [Case(30 + k, T + 3 * k, 1024, [320, 64], 16, 3, mixed=k == 1) for k in range(2)]
    graphs = []
    try:
        lib.zmi_set_stream(s.cuda_stream)
        for c in cases:
            size = lowoha.lora_workspace_size(c.x, c.ids, c.a, c.b, c.dst)
            ws = torch.empty(max(size, 16), dtype=torch.uint8, device=H.DEV)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                assert c.call(c.base, workspace=ws) == capi.SUCCESS, lowoha.last_error()
                refused = c.call(c.base)
                err = lowoha.last_error()
            assert refused == capi.SUCCESS if size == 0 else (refused == capi.FAILURE and "capture" in err)
            graphs.append((g, ws))
    finally:
        lib.zmi_set_stream(None)
    for k in range(4):
        for c, (g, ws) in zip(cases, graphs):
            c.x.copy_(torch.randn(c.x.shape, device=H.DEV))
            c.ids.copy_(torch.randint(-1, 3, c.ids.shape, device=H.DEV))
            c.dst.fill_(0.0)
            ws.fill_(0xff)
            g.replay()
            torch.cuda.synchronize()
            y, tol = c.want(c.base)
            c.compare(c.dst, y, tol)
            graph_bits = c.dst.clone()
            assert c.call(c.base) == capi.SUCCESS
            torch.cuda.synchronize()
            assert torch.equal(c.dst, graph_bits)


def test_two_streams_of_one_thread():
    lib = capi.load()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    cases = [Case(40 + k, 300, 4096, [1024], 32, 4) for k in range(2)]
    torch.cuda.synchronize()
    try:
        for _ in range(3):
            for c, s in zip(cases, streams):
                lib.zmi_set_stream(s.cuda_stream)
                assert c.call(c.base) == capi.SUCCESS
    finally:
        lib.zmi_set_stream(None)
    torch.cuda.synchronize()
    for c in cases:
        c.compare(c.dst, *c.want(c.base))


def test_offsets_beyond_31_bits():
    """Slots, rows of x and rows of dst more than 2^31 elements apart."""
    far = (1 << 31) + 4096
    for T in (2, 66):
        c = Case(50, T, 256, [128], 16, 2, none=0.0)
        a = torch.empty(far + 16 * 256, dtype=BF, device=H.DEV).as_strided((2, 16, 256), (far, 256, 1)).copy_(c.a)
        b = torch.empty(far + 128 * 16, dtype=BF, device=H.DEV).as_strided((2, 128, 16), (far, 16, 1)).copy_(c.b[0])
        c.a, c.b = a, [b]
        c.check("other")
    del a, b
    c = Case(51, 3, 256, [128], 16, 2, none=0.0)
    c.x = torch.empty(2 * far + 256, dtype=BF, device=H.DEV).as_strided((3, 256), (far, 1)).copy_(c.x)
    c.base = torch.empty(2 * far + 128, dtype=BF, device=H.DEV).as_strided((3, 128), (far, 1)).copy_(c.base)
    y, tol = c.want(c.base)
    assert c.call(c.base, dst=c.base) == capi.SUCCESS, lowoha.last_error()
    c.compare(c.base, y, tol)


def test_ranks_outside_their_range_are_clamped():
    c = Case(60, 70, 256, [64], 8, 3, mixed=False)
    c.ranks = torch.tensor([-5, 1000, 3], dtype=torch.int32, device=H.DEV)
    c.check("other")


def test_workspace_that_is_too_small_is_refused():
    c = Case(61, 100, 4096, [64], 8, 3)
    size = lowoha.lora_workspace_size(c.x, c.ids, c.a, c.b, c.dst)
    ws = torch.empty(size, dtype=torch.uint8, device=H.DEV)
    assert c.call(c.base, workspace=ws) == capi.SUCCESS
    assert c.call(c.base, workspace=ws[:size - 1]) == capi.FAILURE and "workspace" in lowoha.last_error()


def test_wrappers_refuse_what_they_cannot_describe():
    c = Case(62, 4, 64, [32], 8, 2)
    for kw in (dict(x=c.x[:, ::2]), dict(a=c.a[:, :4]), dict(b=c.b[0][:1]), dict(dst=c.dst.t()), dict(base=c.base[:, :8]),
               dict(slot_ids=c.ids.long()), dict(slot_ids=c.ids[:2]), dict(scales=c.scales.double()), dict(b=c.b[0].half()),
               dict(ranks=c.ids[:1]), dict(base=c.base.float())):
        args = dict(x=c.x, slot_ids=c.ids, a=c.a, b=c.b[0], dst=c.dst) | kw
        with pytest.raises(ValueError):
            lowoha.lora_direct(**args)


@pytest.mark.parametrize("T,K,N,rank,S", [(129, 256, [96], 8, 17), (512, 320, [72, 40], 16, 16), (513, 320, [72, 40], 16, 16), (512, 320, [72], 33, 2),
                                          (500, 64, [16], 8, 4096), (5000, 72, [24], 8, 4095), (9001, 128, [40], 16, 7), (20000, 64, [16], 4, 1500),
                                          (33000, 64, [8], 8, 2), (4097, 4096, [64], 8, 3), (3000, 1024, [64], 200, 6), (700, 2048, [128, 64, 64], 256, 2)])
def test_plans(T, K, N, rank, S):
    """Batches on both sides of the borders between the ways of sorting rows: few and many rows, slots and ranks."""
    c = Case(T + S, T, K, N, rank, S, mixed=S < 100)
    c.check("other")
    c.check("dst")
    first = c.call(c.base, dst=c.dst) == capi.SUCCESS and c.dst.clone()
    assert c.call(c.base) == capi.SUCCESS and torch.equal(first, c.dst)


def test_sorted_batches_and_long_runs():
    """Rows of a request next to each other, and one request that fills the batch."""
    for T in (300, 3000):
        i32 = dict(dtype=torch.int32, device=H.DEV)
        for ids in ((torch.arange(T, **i32) * 5 // T), torch.zeros(T, **i32), torch.arange(T, **i32).flip(0) * 6 // T - 1):
            Case(T, T, 1024, [264], 32, 5, ids=ids.contiguous()).check("dst")


@pytest.mark.parametrize("T", [20, 300])
@pytest.mark.parametrize("dt,small,large", [(HF, 2.0 ** -24, 2.0 ** 10), (BF, 2.0 ** -131, 2.0 ** 120)])
def test_subnormal_operands_count(dt, small, large, T):
    """Subnormal x (and A, and B) against large ones: the products are ordinary values."""
    g = torch.Generator(device=H.DEV)
    g.manual_seed(T)
    whole = lambda *s: torch.randint(-7, 8, s, generator=g, device=H.DEV).double()   # noqa: E731
    for which in ("x", "a", "b"):
        c = Case(70, T, 256, [64], 16, 3, dt, F32, mixed=False)
        c.x = (whole(T, 256) * (small if which == "x" else large if which == "a" else 1.0)).to(dt)
        c.a = (whole(3, 16, 256) * (small if which == "a" else large if which == "x" else 1.0)).to(dt)
        c.b = [(whole(3, 64, 16) * (small if which == "b" else 1.0)).to(dt)]
        if which == "b":
            c.scales = torch.full((3,), 2.0 ** 20, device=H.DEV)
        c.check("zero")


def test_two_threads_at_once():
    """Each thread with its own stream (and so its own scratch), small and planned calls in turn."""
    import threading
    lib = capi.load()
    cases = [[Case(80 + k, T, 1024, [320], 32, 4) for T in (24, 700)] for k in range(2)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    failed = []

    def work(mine, s):
        try:
            lib.zmi_set_stream(s.cuda_stream)
            for _ in range(8):
                for c in mine:
                    if c.call(c.base) != capi.SUCCESS:
                        failed.append(lowoha.last_error())
        finally:
            lib.zmi_set_stream(None)

    threads = [threading.Thread(target=work, args=a) for a in zip(cases, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for mine in cases:
        for c in mine:
            c.compare(c.dst, *c.want(c.base))


@pytest.mark.parametrize("dt,pad", [(BF, 0), (HF, 0), (HF, 5)])
@pytest.mark.parametrize("T,K,N,rank", [(322, 320, [72], 128), (2100, 328, [64], 128), (4200, 520, [64], 128), (2200, 264, [40], 64),
                                        (33000, 72, [8], 64), (20000, 264, [16], 32), (33000, 264, [8], 32), (1200, 264, [520, 8], 64)])
def test_tile_shapes(T, K, N, rank, dt, pad):
    """Every height of a shrink tile with every number of rank tiles."""
    Case(T + rank, T, K, N, rank, 2, dt, mixed=False, pad=pad, w_pad=pad).check("other")


@pytest.mark.parametrize("rank", [5, 32, 33, 64])
@pytest.mark.parametrize("dst", [HF, BF])
def test_f16_columns_of_a_lane(rank, dst):
    """Eight columns a lane up to rank 32, four beyond: slices that end inside a wavefront's columns, all in eights."""
    Case(rank, 600, 264, [520, 8, 136], rank, 3, HF, dst).check("dst")
