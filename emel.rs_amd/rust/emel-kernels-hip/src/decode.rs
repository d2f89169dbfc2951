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

/// Queries, and keys where given, turned by their positions on one to four
/// axes.
#[derive(Debug)]
pub struct OpRope<'a> {
    q: DeviceView<'a>,
    q_out: DeviceViewMut<'a>,
    k: Option<(DeviceView<'a>, DeviceViewMut<'a>)>,
    positions: DeviceView<'a>,
    factors: Option<DeviceView<'a>>,
    sections: [u32; 4],
    flags: u32,
    base: f32,
    scale: f32,
    magnitude: f32,
}

impl<'a> OpRope<'a> {
    /// Pairs of values half the turned ones apart, `sections` of them for each
    /// axis, with frequencies from `base`; validation occurs when it is
    /// dispatched.
    #[must_use]
    pub const fn new(q: DeviceView<'a>, q_out: DeviceViewMut<'a>, positions: DeviceView<'a>, sections: [u32; 4], base: f32) -> Self {
        Self { q, q_out, k: None, positions, factors: None, sections, flags: 0, base, scale: 1.0, magnitude: 1.0 }
    }

    /// The tokens' keys, turned with them.
    #[must_use]
    pub const fn with_keys(mut self, k: DeviceView<'a>, k_out: DeviceViewMut<'a>) -> Self {
        self.k = Some((k, k_out));
        self
    }

    /// What each pair's frequency is divided by.
    #[must_use]
    pub const fn with_factors(mut self, factors: DeviceView<'a>) -> Self {
        self.factors = Some(factors);
        self
    }

    /// What positions, and the results, are multiplied by.
    #[must_use]
    pub const fn with_scale(mut self, scale: f32, magnitude: f32) -> Self {
        self.scale = scale;
        self.magnitude = magnitude;
        self
    }

    /// `ffi::EMEL_ROPE_ADJACENT` and its neighbours.
    #[must_use]
    pub const fn with_flags(mut self, flags: u32) -> Self {
        self.flags = flags;
        self
    }
}

impl HipEvent for OpRope<'_> {
    type Output = Result<(), HipError>;

    fn dispatch(self, kernel: &mut HipKernel) -> Self::Output {
        let request = ffi::EmelRopeRequest {
            q: self.q.as_ffi(),
            q_out: self.q_out.as_ffi(),
            k: raw(self.k.as_ref().map(|k| &k.0)),
            k_out: self.k.as_ref().map_or(core::ptr::null(), |k| core::ptr::from_ref(k.1.as_ffi())),
            positions: self.positions.as_ffi(),
            factors: raw(self.factors.as_ref()),
            sections: self.sections,
            flags: self.flags,
            base: self.base,
            scale: self.scale,
            magnitude: self.magnitude,
        };
        // SAFETY: the request's views live until the call returns and describe
        // live device memory, checked by the library.
        HipError::check(kernel.call(|s| unsafe { ffi::emel_op_rope(&raw const request, s) }))
    }
}

/// Writes new tokens' keys and values into their slots of the page pools, as
/// halves or packed rows.
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

/// Keys and values of the slots named, read back from the page pools as f32.
#[derive(Debug)]
pub struct OpPagedKvRead<'a> {
    k_pages: DeviceView<'a>,
    v_pages: DeviceView<'a>,
    slots: DeviceView<'a>,
    k: DeviceViewMut<'a>,
    v: DeviceViewMut<'a>,
}

impl<'a> OpPagedKvRead<'a> {
    /// Creates the event; validation occurs when it is dispatched.
    #[must_use]
    pub const fn new(
        k_pages: DeviceView<'a>,
        v_pages: DeviceView<'a>,
        slots: DeviceView<'a>,
        k: DeviceViewMut<'a>,
        v: DeviceViewMut<'a>,
    ) -> Self {
        Self { k_pages, v_pages, slots, k, v }
    }
}

impl HipEvent for OpPagedKvRead<'_> {
    type Output = Result<(), HipError>;

    fn dispatch(self, kernel: &mut HipKernel) -> Self::Output {
        let (kp, vp, t) = (self.k_pages.as_ffi(), self.v_pages.as_ffi(), self.slots.as_ffi());
        let (k, v) = (self.k.as_ffi(), self.v.as_ffi());
        // SAFETY: live device views, checked by the library; the kernel skips
        // slots outside the pools.
        HipError::check(kernel.call(|s| unsafe { ffi::emel_op_paged_kv_read(kp, vp, t, k, v, s) }))
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
