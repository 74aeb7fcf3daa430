"""What yuuka_memcpy_h2d has written is there for the next launch on any stream, also one that does not wait for the default one."""
import numpy as np
import pytest

from yuuka_b200 import cuda

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nbytes", [4, 60_000, 66_000, 300_000, 1_300_000, 9_000_000])
def test_an_upload_is_there_for_the_next_launch(nbytes):
    dev = cuda.Device(0)
    stream, a, b = dev.stream(), dev.alloc(nbytes), dev.alloc(nbytes)
    words = nbytes // 4
    for i in range(300):
        x = np.full(words, i + 1, np.int32)
        a.write(x)
        cuda.check(cuda.lib().yuuka_buffer_copy(stream.h, b.h, 0, a.h, 0, words * 4, None))
        stream.synchronize()
        got = b.read(np.int32, words)
        late = np.flatnonzero(got != i + 1)
        assert late.size == 0, (i, late.size, late[:3], got[late[:3]])
    for q in (a, b):
        q.free()
    stream.destroy()
    dev.close()
