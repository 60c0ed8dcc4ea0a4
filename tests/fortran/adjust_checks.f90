! adjust_checks.f90 -- steps that draw from adjusted logits (fg_paged_step_adjust of
! include/fgpt.h) on an 8-bit paged cache, from Fortran; test code, built by build()
! next to this file.
!
!   refusals   a null handle and an incomplete history are refused (needs no device).
!   banned     the prompt IDS_FILE on an int8 cache, then NGEN greedy steps, each id
!              banned (a bias of -infinity) once it has come up, every even id by a
!              mask. OUT_FILE gets a line of NGEN ids.
!
! Usage:
!   adjust_checks refusals
!   adjust_checks banned WDIR L D H KH HD V IDS_FILE NGEN OUT_FILE
program adjust_checks
  use, intrinsic :: iso_c_binding
  use, intrinsic :: ieee_arithmetic
  use, intrinsic :: iso_fortran_env, only: error_unit
  use fgpt_c
  use fgpt_util
  implicit none

  character(len=512) :: mode

  if (command_argument_count() < 1) call usage()
  call get_command_argument(1, mode)
  select case (trim(mode))
  case ('refusals')
    call run_refusals()
  case ('banned')
    call run_banned()
  case default
    call usage()
  end select

contains

  subroutine usage()
    write (error_unit, '(A)') 'usage: adjust_checks refusals'
    write (error_unit, '(A)') '       adjust_checks banned WDIR L D H KH HD V IDS NGEN OUT'
    stop 2
  end subroutine usage

  subroutine ok(what, rc)
    character(*), intent(in) :: what
    integer(c_int32_t), intent(in) :: rc
    if (rc /= FG_OK) call stop_rc(what, rc)
  end subroutine ok

  subroutine run_refusals()
    type(c_ptr) :: nul, pc
    type(fg_adjust_cfg), target :: adjust
    integer(c_int32_t) :: one(1)
    nul = c_null_ptr
    one = 1
    if (fg_paged_step_adjust(nul, nul, 1, one, one, one, c_loc(adjust), nul, nul, nul) /= FG_EARG) stop 1
    if (fg_paged_create(nul, 4, 16, 1, FG_KV_I8 + FG_KV_PREFIX, 0, 0, pc) /= FG_EARG) stop 1
    write (*, '(A)') 'refusals: ok'
  end subroutine run_refusals

  subroutine run_banned()
    character(len=512) :: wdir, ids_file, out_file
    type(fg_dims) :: dims
    type(fg_adjust_cfg), target :: adjust
    type(c_ptr) :: m, pc
    integer :: n, ngen, i, u
    integer(c_int), allocatable :: ids(:)
    integer(c_int), allocatable, target :: out(:)
    integer(c_int32_t), allocatable, target :: mask(:)
    integer(c_int32_t), target :: next(1), starts(2)
    real(c_float), allocatable, target :: ban(:)
    real(c_float), allocatable :: cos_b(:), sin_b(:)

    if (command_argument_count() < 11) call usage()
    wdir = sarg(2)
    dims = fg_dims(iarg(3), iarg(4), iarg(5), iarg(6), iarg(7), iarg(8), 1.0e-5_c_float)
    ids_file = sarg(9); ngen = iarg(10); out_file = sarg(11)
    call read_ids(trim(ids_file), ids, n)
    allocate (out(ngen), ban(ngen), mask((dims%vocab_size + 31)/32))
    call ok('load', fg_model_load(dims, trim(wdir)//c_null_char, m))
    call rope_tables(n + ngen, dims%head_dim, cos_b, sin_b)
    call ok('rope', fg_set_rope(m, 0, n + ngen, cos_b, sin_b))
    call ok('create', fg_paged_create(m, (n + ngen)/16 + 2, 16, 1, FG_KV_I8, 0, 0, pc))

    mask = int(z'AAAAAAAA', c_int32_t)   ! odd ids alone
    ban = -ieee_value(1.0_c_float, ieee_positive_inf)
    adjust%mask = c_loc(mask)
    adjust%n_mask = 1
    adjust%bias_start = c_loc(starts)
    adjust%bias_id = c_loc(out)
    adjust%bias = c_loc(ban)
    starts(1) = 0
    do i = 1, ngen
      starts(2) = i - 1
      adjust%n_bias = i - 1
      if (i == 1) then
        call ok('prompt', fg_paged_step_adjust(m, pc, 1, [0], [n], ids, c_loc(adjust), c_null_ptr, &
            c_null_ptr, c_loc(next)))
      else
        call ok('step', fg_paged_step_adjust(m, pc, 1, [0], [1], out(i - 1:i - 1), c_loc(adjust), &
            c_null_ptr, c_null_ptr, c_loc(next)))
      end if
      out(i) = next(1)
    end do
    call ok('destroy', fg_paged_destroy(pc))
    call ok('destroy', fg_model_destroy(m))
    open (newunit=u, file=trim(out_file), status='replace', action='write')
    write (u, '(*(I0,1X))') out
    close (u)
  end subroutine run_banned
end program adjust_checks
