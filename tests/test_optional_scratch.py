"""Scratch that a product can do without is not asked for in a way that fails the
call."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_copied_rows_while_the_program_captures_a_graph(rt, oracle):
    """Rows of 1019 and 1020 bytes are copied to an aligned pitch first.  With a
    capture open on a stream of the program's own, an ordinary allocation is
    refused; before the rows were copied these products made none."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(5)
    cases = []
    for M, K, N in ((900, 1019, 640), (660, 1020, 474)):
        a, b = rng.integers(0, 256, (M, K), dtype=np.uint8), rng.integers(-127, 128, (K, N), dtype=np.int8)
        zps = np.array([131], np.uint8), np.array([7], np.int8)
        cases.append((a, b, zps, [rt.DeviceArray.from_numpy(v) for v in (a, b) + zps], rt.DeviceArray((M, N), np.int32)))

    def run(rows=None):
        for a, b, _, (da, db, az, bz), out in cases:
            if rows:
                da = rt.DeviceArray.view_of(da, 0, (rows, a.shape[1]))
                out = rt.DeviceArray.view_of(out, 0, (rows, b.shape[1]))
            rt.MatMulInteger(da, db, az, bz, out=out)
            assert rows or "any K" not in rt.last_gemm_kernel(), rt.last_gemm_kernel()

    run()  # (a kernel is loaded when it is first launched, which a capture refuses too)
    rt.synchronize()
    rt.clear_cache()  # the thread's pool of GPU memory
    for c in cases:
        rt.mark_constant(c[3][1])
    run(rows=2)  # packs the weights
    rt.synchronize()
    x = torch.ones(1024, device="cuda")
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        y = x * 3.0
        run()
    rt.synchronize()
    for _ in range(3):
        x.add_(1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, x * 3.0)
    for a, b, (az, bz), on_gpu, out in cases:
        assert np.array_equal(out.numpy(), oracle.matmul_integer(a, b, az, bz)), a.shape
        rt.unmark_constant(on_gpu[1])


def _block_operands(rt, seed, M, K, N):
    """e4m3 operands of 1, 2 .. with their scales, and the product in 64 bits."""
    rng = np.random.default_rng(seed)
    a, b = (rng.choice(np.uint8([0x00, 0x30, 0x38, 0x40, 0xB8]), s) for s in ((M, K), (N, K)))
    kb = -(-K // 128)
    sa, sb = (rng.choice(np.float32([0.5, 1, 2]), s) for s in ((M, kb), (-(-N // 128), kb)))
    x, w = (rt.to_float32(t.view(rt.float8_e4m3fn)).astype(np.float64) for t in (a, b))
    x *= np.repeat(sa, 128, 1)[:, :K]
    w *= np.repeat(np.repeat(sb, 128, 0)[:N], 128, 1)[:, :K]
    return [t.view(rt.float8_e4m3fn) if t.dtype == np.uint8 else t for t in (a, sa, b, sb)], x @ w.T


# (few bits, so that sums are exact: 4095 terms of +-0.25 .. 4, scales 0.25 .. 4)
BLOCK_PRODUCTS = [(900, 1019, 640, "any K"), (70, 4096, 1024, "K in parts"), (100, 4095, 500, "both"), (130, 768, 768, "neither")]


def test_block_products_while_the_program_captures_a_graph(rt):
    """Copies of rows of 1019 bytes and sums of parts of K are scratch that these
    products can do without."""
    torch = pytest.importorskip("torch")
    cases = []
    for i, (M, K, N, _) in enumerate(BLOCK_PRODUCTS):
        given, want = _block_operands(rt, i, M, K, N)
        cases.append(([rt.DeviceArray.from_numpy(t) for t in given], want, rt.DeviceArray((M, N), np.float32)))

    def run():
        for given, _, out in cases:
            rt.MatMulBlocks(*given, out=out)

    run()
    rt.synchronize()
    rt.clear_cache()
    x = torch.ones(1024, device="cuda")
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        y = x * 3.0
        run()
    rt.synchronize()
    for _ in range(3):
        x.add_(1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, x * 3.0)
    for _, want, out in cases:
        assert np.array_equal(out.numpy(), want.astype(np.float32))


class _BlockGemm(ctypes.Structure):
    """om::BlockGemm (llm_kernels.h)."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("a", "a_scale", "b", "b_scale", "bias", "y")] + \
               [(n, ctypes.c_int64) for n in ("M", "N", "K", "bias_len")] + \
               [(n, ctypes.c_int) for n in ("kind", "activation")] + [(n, ctypes.c_void_p) for n in ("rows", "parts")]


@pytest.mark.parametrize("M,K,N,wants", BLOCK_PRODUCTS + [
    (33, 129, 1001, "any K"), (1000, 16, 40, "neither"),
    (70, 33001, 40, "both"),          # more scales than LDS has room for
    (2 ** 21 + 37, 17, 1, "any K")])  # more rows than one launch takes
def test_block_products_without_room_for_scratch(rt, M, K, N, wants):
    """The launch as the runtime makes it where there is no memory for the copies, the
    sums, or either."""
    torch = pytest.importorskip("torch")
    lib = rt.load()
    row_bytes = getattr(lib, "_ZN2om20block_gemm_row_bytesERKNS_9BlockGemmE")
    part_bytes = getattr(lib, "_ZN2om21block_gemm_part_bytesERKNS_9BlockGemmE")
    launch = getattr(lib, "_ZN2om17launch_block_gemmEP12ihipStream_tRKNS_9BlockGemmE")
    row_bytes.restype = part_bytes.restype = ctypes.c_size_t
    launch.argtypes = [ctypes.c_void_p, ctypes.POINTER(_BlockGemm)]
    given, want = _block_operands(rt, M, M, K, N)
    bias = np.arange(N, dtype=np.float32)
    on_gpu = [rt.DeviceArray.from_numpy(t) for t in given + [bias]]
    g = _BlockGemm(*[t.ptr for t in on_gpu], None, M, N, K, N, 0, 0, None, None)
    rows = row_bytes(ctypes.byref(g))
    assert (rows > 0) == (K % 16 != 0)
    assert rows == 0 or part_bytes(ctypes.byref(g)) == 0
    room = torch.empty(rows + 16, dtype=torch.uint8, device="cuda")
    for g.rows in {None, room.data_ptr() if rows else None}:
        parts = part_bytes(ctypes.byref(g))
        assert g.rows or not rows or not parts
        if g.rows or not rows:
            assert (parts > 0) == (wants in ("K in parts", "both"))
        sums = torch.empty(parts + 16, dtype=torch.uint8, device="cuda")
        for g.parts in {None, sums.data_ptr() if parts else None}:
            out = rt.DeviceArray.from_numpy(np.full((M, N), np.nan, np.float32))
            g.y = out.ptr
            assert launch(None, ctypes.byref(g)) == 0
            torch.cuda.synchronize()
            assert np.array_equal(out.numpy(), (want + bias).astype(np.float32)), (g.rows, g.parts)
            assert ("many rows" in rt.last_gemm_kernel()) == (rows > 0 and not g.rows), rt.last_gemm_kernel()
            assert ("parts" in rt.last_gemm_kernel()) == bool(g.parts)
