"""Arguments that the 8-bit cache's calls refuse before anything is launched,
beside those of test_cpu_kv8.py. None needs a GPU."""
import pytest

import fekv
from fekv import _lib
from test_cpu_kv8 import gather_args


@pytest.mark.parametrize("cs", [8, 24, 40, 17])
def test_gather_refuses_slots_without_a_scale_of_their_own(cs):
    """One scale row per 16 slots: a pool's last slots would read past them."""
    assert fekv.load().fe_kv8_gather(*gather_args(cs=cs)) == _lib.FE_ERR_INVALID_ARGUMENT
    assert b"cache_slots" in fekv.load().fe_last_error()


@pytest.mark.parametrize("out_rows,num_pages,status", [
    (-1, 1, _lib.FE_ERR_INVALID_ARGUMENT), (4, -1, _lib.FE_ERR_INVALID_ARGUMENT)])
def test_gather_refuses_negative_sizes(out_rows, num_pages, status):
    codes, exps, out, kv, pages, *rest = gather_args()
    assert fekv.load().fe_kv8_gather_within(codes, exps, out, out_rows, kv, pages, num_pages,
                                            *rest) == status


# ---------------------------------------------------------------------------
# tensors that are not on the current device
# ---------------------------------------------------------------------------

torch = pytest.importorskip("torch")


class Placed(torch.Tensor):
    """A CPU tensor that says it is on CUDA device `where`."""

    is_cuda = True

    def get_device(self):
        return self.where


def placed(t, where):
    t = t.as_subclass(Placed)
    t.where = where
    return t


class Calls:
    """Stands in for the library: every call succeeds and is counted."""

    def __init__(self):
        self.count = 0

    def __getattr__(self, name):
        def call(*args):
            self.count += 1
            return 0

        return call


@pytest.fixture
def lib(monkeypatch):
    from fekv import ops

    calls = Calls()
    monkeypatch.setattr(ops._lib, "load", lambda: calls)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 0, raising=False)
    return calls


def pool(where):
    return fekv.Kv8Pool(placed(torch.zeros(48, 2, 128, dtype=torch.float8_e4m3fn), where),
                        placed(torch.zeros(3, 2, dtype=torch.uint8), where))


def append_call(**at):
    where = lambda name: at.get(name, 0)  # noqa: E731
    t = lambda name, *shape, dtype=torch.bfloat16: placed(  # noqa: E731
        torch.zeros(*shape, dtype=dtype), where(name))
    fekv.append_kv8(t("q", 3, 4, 128), t("k", 3, 2, 128), t("v", 3, 2, 128), pool(where("kpool")),
                    pool(where("vpool")), t("slots", 3, dtype=torch.int64),
                    t("pos", 3, dtype=torch.int64), t("cache", 8, 64, dtype=torch.float32),
                    q_out=t("q_out", 3, 4, 128))


def gather_call(**at):
    t = lambda name, *v: placed(torch.tensor(v, dtype=torch.int32), at.get(name, 0))  # noqa: E731
    out = placed(torch.zeros(16, 2, 128, dtype=torch.bfloat16), at.get("out", 0))
    fekv.gather_kv8(pool(at.get("pool", 0)), out, t("kv", 0, 1), t("pages", 1), t("last", 5),
                    t("offset", 0), 5, 16)


def copy_call(**at):
    t = lambda name: placed(torch.zeros(1, dtype=torch.int32), at.get(name, 0))  # noqa: E731
    fekv.copy_blocks_kv8([pool(0), pool(at.get("kpool", 0))], [pool(at.get("vpool", 0)), pool(0)],
                         t("src"), t("dst"), t("ntok"), 16)


def bare_plan(index=0):
    plan = fekv.Kv8Plan.__new__(fekv.Kv8Plan)
    plan.lib, plan.handle, plan.rows = fekv.ops._lib.load(), None, 3
    plan.hq, plan.dim, plan.pool_shape, plan.dtype = 4, 128, (48, 2, 128), torch.bfloat16
    plan.index = index
    return plan


def attention_call(**at):
    plan = bare_plan(at.get("plan", 0))
    t = lambda name: placed(torch.zeros(3, 4, 128, dtype=torch.bfloat16), at.get(name, 0))  # noqa: E731
    plan.attention(t("q"), pool(at.get("kpool", 0)), pool(at.get("vpool", 0)), t("out"))


@pytest.mark.parametrize("call,names", [
    (append_call, "q k v kpool vpool slots pos cache q_out"),
    (gather_call, "pool out kv pages last offset"),
    (copy_call, "kpool vpool src dst ntok"),
    (attention_call, "plan q kpool vpool out")])
def test_what_is_on_another_device_is_refused(lib, call, names):
    call()  # all on the current device
    count = lib.count
    for name in names.split():
        for where in (1, -1):
            with pytest.raises(ValueError, match="current device|contiguous"):
                call(**{name: where})
    assert lib.count == count  # nothing was launched


# ---------------------------------------------------------------------------
# metadata shorter than a prepare reads
# ---------------------------------------------------------------------------

META = dict(qo=(0, 2, 3, 3), kv=(0, 2, 3, 4), pages=(5, 1, 2, 7), last=(16, 3, 1))


def host_prepare(batch=None, **kw):
    m = {**META, **kw}
    bare_plan(m.pop("plan", 0)).prepare(m["qo"], m["kv"], m["pages"], m["last"], batch, stream=0)


def device_prepare(batch=3, where=None, plan=0, **kw):
    m = {n: placed(torch.tensor(v, dtype=torch.int32), int(n == where))
         for n, v in {**META, **kw}.items()}
    bare_plan(plan).prepare_device(m["qo"], m["kv"], m["pages"], m["last"], batch, 3, stream=0)


def step_prepare(plan=0, where=None, slots=None):
    t = {n: placed(torch.zeros(*shape, dtype=dt), int(n == where))
         for n, shape, dt in (("tables", (3, 4), torch.int32), ("starts", (3,), torch.int32),
                              ("slots", (6,), torch.int64), ("positions", (6,), torch.int64))}
    bare_plan(plan).step_prepare_device(t["tables"], t["starts"], 2,
                                        t["slots"] if slots is None else slots, t["positions"],
                                        stream=0)


@pytest.mark.parametrize("prepare,wrong", [
    (host_prepare, dict(qo=(0, 2, 3))), (host_prepare, dict(last=(16, 3))),
    (host_prepare, dict(pages=(5, 1, 2))), (host_prepare, dict(batch=4)),
    (host_prepare, dict(batch=-1)), (host_prepare, dict(plan=1)),
    (device_prepare, dict(qo=(0, 2, 3))), (device_prepare, dict(kv=(0, 2, 3))),
    (device_prepare, dict(last=(16, 3))), (device_prepare, dict(batch=4)),
    (device_prepare, dict(batch=-1)), (device_prepare, dict(plan=1)),
    *((device_prepare, dict(where=n)) for n in META),
    *((step_prepare, dict(where=n)) for n in ("tables", "starts", "slots", "positions")),
    (step_prepare, dict(plan=1)),
    (step_prepare, dict(slots=placed(torch.zeros(1, dtype=torch.int64), 0))),
    (step_prepare, "strided")])
def test_prepares_refuse_what_they_would_read_or_write_past(lib, prepare, wrong):
    if wrong == "strided":
        wrong = dict(slots=placed(torch.zeros(1, dtype=torch.int64).expand(6), 0))
    prepare()
    count = lib.count
    with pytest.raises(ValueError):
        prepare(**wrong)
    assert lib.count == count


def test_a_prepare_of_part_of_the_metadata_is_taken(lib):
    host_prepare(batch=2)
    device_prepare(batch=2)
    host_prepare(pages=(5, 1, 2, 7, 9))
    assert lib.count == 3
