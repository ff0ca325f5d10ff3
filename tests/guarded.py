"""Device buffers between guard words, for tests that check what a call writes and what it leaves alone."""
import numpy as np
import torch

GUARD = 64


class Guarded:
    """``data`` (a numpy array) in device memory, ``shift`` elements past a 16-byte boundary, with GUARD elements of a
    pattern on either side."""

    def __init__(self, data, device, shift=0):
        data = np.ascontiguousarray(data)
        self.shape, self.n, self.at = data.shape, data.size, GUARD + shift
        pattern = np.full(self.n + 2 * GUARD + shift, 77, data.dtype)
        pattern[self.at:self.at + self.n] = data.reshape(-1)
        self.buffer = torch.from_numpy(pattern).to(device)
        self.flat = self.buffer[self.at:self.at + self.n]

    @property
    def pointer(self):
        return self.flat.data_ptr()

    def numpy(self):
        """The contents, after a look at the guards."""
        everything = self.buffer.cpu().numpy()
        assert (everything[:self.at] == 77).all() and (everything[self.at + self.n:] == 77).all(), "written out of bounds"
        return everything[self.at:self.at + self.n].reshape(self.shape)


def pointer(t):
    return None if t is None else t.pointer
