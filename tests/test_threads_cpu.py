"""What ranks that run as threads (tests/fake_dist.py) share on the host."""
import os
import sys
import threading

import numpy as np


def test_threads_read_one_archive(golden_dir):
    g = np.load(os.path.join(golden_dir, "teacher_sage_int2_p4.npz"))
    want = {n: g[n] for n in g.files}
    errors = []

    def read_all():
        try:
            for n in g.files * 2:
                np.testing.assert_array_equal(g[n], want[n])
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    before = sys.getswitchinterval()
    sys.setswitchinterval(1e-5)
    try:
        threads = [threading.Thread(target=read_all) for _ in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(before)
    assert not errors, errors[0]
