"""What the entry points of libgq_hip.so would launch, without a GPU: `launches(calls)` runs them in a process of their own on a
stand-in for the HIP runtime (launch_recorder.c)."""
import ctypes
import json
import os
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
PACKAGE = os.path.join(os.path.dirname(HERE), "popxl-addons_amd")


class _Record(ctypes.Structure):
    _fields_ = [("launch", ctypes.c_int32), ("device", ctypes.c_int32), ("grid", ctypes.c_uint32 * 3), ("block", ctypes.c_uint32 * 3),
                ("lds", ctypes.c_uint64), ("kernel", ctypes.c_char * 160)]


def launches(calls):
    """calls: [(device, entry point, arguments)]; an argument is a number or [structure of _gq_hip, *its fields] (passed by address).
    Result: for each call {"code": its return value, "records": [what it launched or set, in order]}.  Addresses are never read."""
    with tempfile.TemporaryDirectory() as folder:
        recorder = os.path.join(folder, "recorder.so")
        subprocess.run(["gcc", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-o", recorder, os.path.join(HERE, "launch_recorder.c")], check=True)
        done = subprocess.run([sys.executable, os.path.abspath(__file__), recorder], input=json.dumps(calls), capture_output=True, text=True,
                              timeout=100)
    assert done.returncode == 0, done.stderr
    return json.loads(done.stdout)


def _main(recorder):
    stand_in = ctypes.CDLL(recorder, mode=ctypes.RTLD_GLOBAL)
    stand_in.recorder_record.restype = ctypes.POINTER(_Record)
    sys.path.insert(0, PACKAGE)
    from popxl_addons import _gq_hip

    lib, results = _gq_hip.load(), []
    for device, name, arguments in json.load(sys.stdin):
        stand_in.recorder_clear()
        stand_in.recorder_device(device)
        given = [ctypes.byref(getattr(_gq_hip, a[0])(*a[1:])) if isinstance(a, list) else a for a in arguments]
        code = getattr(lib, name)(*given)
        records = [stand_in.recorder_record(i).contents for i in range(stand_in.recorder_count())]
        results.append({"code": code, "records": [dict(launch=bool(r.launch), device=r.device, grid=list(r.grid), block=list(r.block), lds=r.lds,
                                                       kernel=r.kernel.decode()) for r in records]})
    print(json.dumps(results))


if __name__ == "__main__":
    _main(sys.argv[1])
