//! A served token's events over packed 4-bit weights and a paged key-value
//! cache.  None has a reference counterpart; `include/emel_hip.h` holds their
//! formulas, layouts and guards, and each returns the library's status.

use crate::device::HipError;
use crate::ffi;
use crate::kernel::{HipEvent, HipKernel};
use crate::view::{DeviceView, DeviceViewMut};

/// The packed format of a product's weights.
#[derive(Clone, Copy, Debug, Eq, PartialEq)]
pub enum PackedFormat {
    /// Blocks of 32 values.
    Q4_0,
    /// Blocks of 256 values.
    Q4K,
}

/// `dst[r, c] = sum over k of W[r, k] x[k, c]`, W packed rows of `format`.
#[derive(Debug)]
pub struct OpMulMatQ4<'a> {
    format: PackedFormat,
    weights: DeviceView<'a>,
    x: DeviceView<'a>,
    dst: DeviceViewMut<'a>,
}

impl<'a> OpMulMatQ4<'a> {
    /// Creates the event; validation occurs when it is dispatched.
    #[must_use]
    pub const fn new(format: PackedFormat, weights: DeviceView<'a>, x: DeviceView<'a>, dst: DeviceViewMut<'a>) -> Self {
        Self { format, weights, x, dst }
    }
}

impl HipEvent for OpMulMatQ4<'_> {
    type Output = Result<(), HipError>;

    fn dispatch(self, kernel: &mut HipKernel) -> Self::Output {
        let (w, x, y) = (self.weights.as_ffi(), self.x.as_ffi(), self.dst.as_ffi());
        // SAFETY: live device views, checked by the library.
        HipError::check(kernel.call(|s| unsafe {
            match self.format {
                PackedFormat::Q4_0 => ffi::emel_op_mul_mat_q4_0(w, x, y, s),
                PackedFormat::Q4K => ffi::emel_op_mul_mat_q4_k(w, x, y, s),
            }
        }))
    }
}

/// Writes new tokens' keys and values into their slots of the page pools.
#[derive(Debug)]
pub struct OpPagedKvAppend<'a> {
    k: DeviceView<'a>,
    v: DeviceView<'a>,
    slots: DeviceView<'a>,
    k_pages: DeviceViewMut<'a>,
    v_pages: DeviceViewMut<'a>,
}

impl<'a> OpPagedKvAppend<'a> {
    /// Creates the event; validation occurs when it is dispatched.
    #[must_use]
    pub const fn new(
        k: DeviceView<'a>,
        v: DeviceView<'a>,
        slots: DeviceView<'a>,
        k_pages: DeviceViewMut<'a>,
        v_pages: DeviceViewMut<'a>,
    ) -> Self {
        Self { k, v, slots, k_pages, v_pages }
    }
}

impl HipEvent for OpPagedKvAppend<'_> {
    type Output = Result<(), HipError>;

    fn dispatch(self, kernel: &mut HipKernel) -> Self::Output {
        let (k, v, t) = (self.k.as_ffi(), self.v.as_ffi(), self.slots.as_ffi());
        let (kp, vp) = (self.k_pages.as_ffi(), self.v_pages.as_ffi());
        // SAFETY: live device views, checked by the library; the kernel skips
        // slots outside the pools.
        HipError::check(kernel.call(|s| unsafe { ffi::emel_op_paged_kv_append(k, v, t, kp, vp, s) }))
    }
}

/// Attention of one new token per sequence over its cached pages.
#[derive(Debug)]
pub struct OpPagedAttention<'a> {
    q: DeviceView<'a>,
    k_pages: DeviceView<'a>,
    v_pages: DeviceView<'a>,
    page_table: DeviceView<'a>,
    lengths: DeviceView<'a>,
    scale: f32,
    window: u64,
    soft_cap: f32,
    dst: DeviceViewMut<'a>,
}

impl<'a> OpPagedAttention<'a> {
    /// Every position, scores as they are; validation occurs when it is
    /// dispatched.
    #[must_use]
    pub const fn new(
        q: DeviceView<'a>,
        k_pages: DeviceView<'a>,
        v_pages: DeviceView<'a>,
        page_table: DeviceView<'a>,
        lengths: DeviceView<'a>,
        scale: f32,
        dst: DeviceViewMut<'a>,
    ) -> Self {
        Self { q, k_pages, v_pages, page_table, lengths, scale, window: 0, soft_cap: 0.0, dst }
    }

    /// Only the last `window` positions (0: every position).
    #[must_use]
    pub const fn with_window(mut self, window: u64) -> Self {
        self.window = window;
        self
    }

    /// Scores capped at `soft_cap` by its tanh (0: as they are).
    #[must_use]
    pub const fn with_soft_cap(mut self, soft_cap: f32) -> Self {
        self.soft_cap = soft_cap;
        self
    }
}

impl HipEvent for OpPagedAttention<'_> {
    type Output = Result<(), HipError>;

    fn dispatch(self, kernel: &mut HipKernel) -> Self::Output {
        let (q, kp, vp) = (self.q.as_ffi(), self.k_pages.as_ffi(), self.v_pages.as_ffi());
        let (t, n, y) = (self.page_table.as_ffi(), self.lengths.as_ffi(), self.dst.as_ffi());
        let (scale, window, cap) = (self.scale, self.window, self.soft_cap);
        // SAFETY: live device views, checked by the library; the kernel reads
        // no page outside the pools.
        HipError::check(kernel.call(|s| unsafe { ffi::emel_op_paged_attention(q, kp, vp, t, n, scale, window, cap, y, s) }))
    }
}

/// Penalties, biases and a token mask on rows of logits.
#[derive(Debug)]
pub struct OpLogitsAdjust<'a> {
    logits: DeviceView<'a>,
    adjusted: DeviceViewMut<'a>,
    history: Option<DeviceView<'a>>,
    history_len: Option<DeviceView<'a>>,
    repeat: Option<DeviceView<'a>>,
    frequency: Option<DeviceView<'a>>,
    presence: Option<DeviceView<'a>>,
    biases: Option<(DeviceView<'a>, DeviceView<'a>)>,
    allowed: Option<DeviceView<'a>>,
}

impl<'a> OpLogitsAdjust<'a> {
    /// A copy of the logits; the parts below add to it.  Validation occurs
    /// when it is dispatched.
    #[must_use]
    pub const fn new(logits: DeviceView<'a>, adjusted: DeviceViewMut<'a>) -> Self {
        Self {
            logits,
            adjusted,
            history: None,
            history_len: None,
            repeat: None,
            frequency: None,
            presence: None,
            biases: None,
            allowed: None,
        }
    }

    /// The ids each row has seen, and how many of them count.
    #[must_use]
    pub const fn with_history(mut self, ids: DeviceView<'a>, len: Option<DeviceView<'a>>) -> Self {
        self.history = Some(ids);
        self.history_len = len;
        self
    }

    /// The penalties of seen tokens, a value per row each.
    #[must_use]
    pub const fn with_penalties(
        mut self,
        repeat: Option<DeviceView<'a>>,
        frequency: Option<DeviceView<'a>>,
        presence: Option<DeviceView<'a>>,
    ) -> Self {
        self.repeat = repeat;
        self.frequency = frequency;
        self.presence = presence;
        self
    }

    /// What is added to the tokens of `ids`.
    #[must_use]
    pub const fn with_biases(mut self, ids: DeviceView<'a>, values: DeviceView<'a>) -> Self {
        self.biases = Some((ids, values));
        self
    }

    /// A bit per token, clear where it may not be taken.
    #[must_use]
    pub const fn with_mask(mut self, allowed: DeviceView<'a>) -> Self {
        self.allowed = Some(allowed);
        self
    }
}

fn raw(view: Option<&DeviceView<'_>>) -> *const ffi::EmelTensorView {
    view.map_or(core::ptr::null(), |v| core::ptr::from_ref(v.as_ffi()))
}

impl HipEvent for OpLogitsAdjust<'_> {
    type Output = Result<(), HipError>;

    fn dispatch(self, kernel: &mut HipKernel) -> Self::Output {
        let request = ffi::EmelLogitsAdjustRequest {
            logits: self.logits.as_ffi(),
            adjusted: self.adjusted.as_ffi(),
            history: raw(self.history.as_ref()),
            history_len: raw(self.history_len.as_ref()),
            repeat: raw(self.repeat.as_ref()),
            frequency: raw(self.frequency.as_ref()),
            presence: raw(self.presence.as_ref()),
            bias_ids: raw(self.biases.as_ref().map(|b| &b.0)),
            bias: raw(self.biases.as_ref().map(|b| &b.1)),
            allowed: raw(self.allowed.as_ref()),
            reserved: 0,
        };
        // SAFETY: the request's views live until the call returns and describe
        // live device memory, checked by the library.
        HipError::check(kernel.call(|s| unsafe { ffi::emel_logits_adjust(&raw const request, s) }))
    }
}
